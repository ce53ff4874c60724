// Split-KV decode attention over a 4-bit KV cache (row format: kv4.cuh).
//
//   out[b, h] = softmax_j(scale * q . k_j) v_j,   k_j = s c_j + m (per group),
// one query per sequence, keys j < L_b = seq_lens[b].
//
// Bound: HBM.  A key of one KV head is D + 16 bytes (144 at D = 128, against 512
// in 16 bits) for 4 D G FLOPs.  On CUDA cores the unpacking and the FMAs would
// cost about 4 instructions a value, more than the issue slots that HBM's rate
// leaves (3.2 lane operations a value), so both products run on tensor cores
// (mma.sync m16n8k16; 8 columns = the query heads that share the KV head, and
// a single query token cannot fill a tcgen05 tile) and the codes enter them
// without being converted: a 4-bit code in the low bits of an fp16 word is the
// subnormal number c * 2^-24, exactly, so one AND makes an operand.  The codes
// of the upper half of the dims sit 4 bits higher and count 16-fold; q (for
// K) and the final factor (for V) undo that with powers of two.
//   scores  S^T[key, head] = s0 * acc0 + s1 * acc1 + m0 * sum(q0) + m1 * sum(q1)
//           with acc_g the fp32 accumulator of group g's dims;
//   output  O^T[dim, head] of group g += codes^T (P s_g), and one number per
//           head and group, sum_j P_j m_g[j], is added to every dim at the end.
// With up to 4 heads on a KV head (NH = 1) the 8 columns hold each head's two
// groups instead of 8 heads: a lane has one head's scores, half the exponentials,
// and the lower nibbles need no mask, since whole bytes times q0 less the upper
// nibbles times q0 are the lower nibbles times q0.  With 5 to 8 (NH = 2) a lane has
// two heads; more take several CTAs.  Long caches take V's sums more finely (sums_finely).
// q enters as fp16 scaled per head by a power of two so that its largest value
// is about 2^14: a bf16 or fp16 q (below 2^114) then loses nothing but what lies
// 2^-38 below that value.  P s_g enters as fp16 (rounded to 2^-11, finer than the
// bf16 that P is usually held in); the running reference M of the softmax is that of
// P s, each key's score with the exponent of its own V scale, so that the largest P s
// stays near 2^5 whatever the scales are.  What is 2^-19 of it loses a bit a halving:
// another key's share, which then does not show beside the largest, or the other half
// of the dims where its scales are that much smaller.  Sums, maxima and statistics are
// fp32.
//
// Each warp walks its own 32-key tiles through a ring of shared-memory stages
// filled by cp.async, with no barrier between warps until the end; the warps
// merge through shared memory, the splits in a cluster (merges_in_cluster), through
// the workspace and a second kernel, or not at all where one split covers the cache.
//
// Measured, D = 128, bf16 (us; of the cache's bytes at 6397 GB/s): 64 sequences of
// 1000 keys, 32 heads, 47 (99%); 32 of 1 to 4096 keys 57.7 (86%: the short ones leave
// SMs idle at the end); 3 of 60,000 keys, 64 heads on 8, 40.9 (79%: 500 instructions
// a warp's tile of 32 keys, 60% of the issue slots); one of 1000 keys 5.5.  What took
// 32 sequences of 4096 there from 83: ldmatrix and movmatrix in place of shuffles, the
// mask-free operands, splits of equal length by the rule at split_keys.
#include <algorithm>
#include <atomic>

#include "kv4.cuh"

LPC_DECLARE_STATUS(g_kv4_attn_status)

unsigned int lpc_status_kv4_attention(bool clear) {
  unsigned int v = 0;
  cudaMemcpyFromSymbol(&v, g_kv4_attn_status, sizeof(v));
  if (clear && v) {
    unsigned int z = 0;
    cudaMemcpyToSymbol(g_kv4_attn_status, &z, sizeof(z));
  }
  return v;
}

namespace {

using lpc::Num;
using lpc::cp16;
using lpc::cp8;
using lpc::cp_commit;
using lpc::cp_wait;

constexpr int TK = 32;        // keys per warp tile
constexpr int NST = 3;          // stages per warp
constexpr int HB = 8;         // query heads per CTA (columns of the products)
constexpr int UNIT = 128;     // shortest split: one tile per warp; workspace granularity
constexpr int CLUSTER = 4;    // splits that a cluster merges
constexpr float LOG2E = 1.4426950408889634f;
// The reference M is set RISE below the largest P s and moved when a key
// exceeds it by LIFT: fp16 holds 2^(LIFT + 1), and a tile that stays below
// costs one vote instead of a rescaling of the accumulators.
constexpr float RISE = 5.f, LIFT = 13.f;

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The same, zeros instead of the source's bytes when not `ok`.
__device__ __forceinline__ void cp16z(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp8z(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(ok ? 8 : 0)
               : "memory");
}

__device__ __forceinline__ float ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same with a zero accumulator going in.
__device__ __forceinline__ void mma_f16_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                              uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// Four (two) 8x8 matrices of 16-bit units, transposed: rows are keys, and the
// lane (r, t) gets unit r of keys 2t and 2t + 1.
__device__ __forceinline__ void ldm4(uint32_t (&v)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldm2(uint32_t (&v)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0,%1}, [%2];"
               : "=r"(v[0]), "=r"(v[1])
               : "r"(addr)
               : "memory");
}

// Transpose of an 8x8 matrix of 16-bit values spread over the warp.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
  return d;
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}

template <typename T>
__device__ __forceinline__ void unpack_sm(uint32_t w, float& s, float& m);
template <>
__device__ __forceinline__ void unpack_sm<__nv_bfloat16>(uint32_t w, float& s, float& m) {
  s = lpc::bf16lo(w);
  m = lpc::bf16hi(w);
}
template <>
__device__ __forceinline__ void unpack_sm<__half>(uint32_t w, float& s, float& m) {
  const float2 f = __half22float2(*reinterpret_cast<__half2*>(&w));
  s = f.x;
  m = f.y;
}

// What a key adds to its score for the reference M: the exponent of the larger of its two
// V scales, as an integer that orders as it (non-finite numbers, which must not move the
// other keys' reference, turn negative).
// In bf16 at least 40 below the exponent of its minima, so that P m stays in fp32 too;
// the codes of a key that this decides count less than 2^-40 of its minimum.
template <typename T>
__device__ __forceinline__ uint32_t scale_bits(uint2 row) {
  constexpr bool HALF = std::is_same<T, __half>::value;
  constexpr uint32_t UP = HALF ? 0x04000400u : 0x00800080u;
  const uint32_t v = __vimax3_s16x2((row.x & 0x7FFF7FFFu) + UP, (row.y & 0x7FFF7FFFu) + UP, 0u);
  if constexpr (HALF) return v & 0xFFFFu;
  return (uint32_t)max((int)(v & 0xFFFFu), (int)(v >> 16) - (40 << 7));
}
template <typename T>
__device__ __forceinline__ float scale_exponent(uint32_t bits) {
  if constexpr (std::is_same<T, __half>::value) return (float)((int)(bits >> 10) - 16);
  // below 2^-60 the scales no longer move the reference: the sum of the P
  // themselves, up to 2^60 times larger than P s, has to stay in fp32
  return fmaxf((float)((int)(bits >> 7) - 128), -60.f);
}

template <int D, int W>
struct Layout {
  static constexpr int CB = D / 2;                 // code bytes of a row
  static constexpr int CODES = TK * CB;            // of a tile, K or V
  static constexpr int SCALES = TK * 8;
  static constexpr int STAGE = 2 * CODES + 2 * SCALES;
  static constexpr int RED = HB * (D + 2) * 4;     // merge buffer of a warp, or of the CTA
  // where piece p of key's V row is stored
  __device__ static __forceinline__ int place(int key, int p) {
    return D == 128 ? p ^ ((key >> 1) & 3) : D == 64 ? p ^ ((key >> 2) & 1) : p;
  }
  static constexpr int SMEM = W * NST * STAGE > (W + 1) * RED ? W * NST * STAGE : (W + 1) * RED;
};

template <typename T, int D, int NH, int W, bool FINE>
__global__ void __launch_bounds__(W * 32, W == 4 ? 4 : 1)
    kv4_split_kernel(const T* __restrict__ q, const uint8_t* __restrict__ kcodes,
                     const uint8_t* __restrict__ kscales, const uint8_t* __restrict__ vcodes,
                     const uint8_t* __restrict__ vscales, const int32_t* __restrict__ seq_lens,
                     T* __restrict__ out, float* __restrict__ part_o, float* __restrict__ part_ml,
                     int H, int G, int head_blocks, int max_splits, int chunk, int cluster,
                     float scale_log2, lpc::Kv4Rows rows) {
  using L = Layout<D, W>;
  constexpr int CB = L::CB;
  constexpr int KW = D / 32;              // K words of a lane and key
  constexpr int VM = D / 32;              // V products per group: 16 dims each
  constexpr int NI = VM == 1 ? 1 : 2;     // of them from one ldmatrix
  extern __shared__ __align__(16) uint8_t smem[];

  lpc::pdl_trigger();
  lpc::pdl_wait();
  const int split = blockIdx.x;
  const int kvh = blockIdx.y / head_blocks;
  const int hb = blockIdx.y - kvh * head_blocks;
  const int64_t b = blockIdx.z;
  const int heads = min(HB, G - hb * HB);             // query heads of this CTA
  const int64_t h0 = (int64_t)kvh * G + hb * HB;      // the first of them
  int64_t row0, head_rows, cap;
  const bool inside = rows.locate(b, &row0, &head_rows, &cap);
  int len = lpc::ld_dep(seq_lens + b);
  if (!inside || len > cap) {
    if (split == 0 && threadIdx.x == 0) atomicOr(&g_kv4_attn_status, LPC_DEV_ERR_BOUNDS);
    len = inside ? (int)cap : 0;
  }
  const int nsplits = len > 0 ? (len + chunk - 1) / chunk : 0;
  if (split >= nsplits) {
    if (W == 16 && len > 0 && cluster && nsplits > 1) {  // the others read no sums of this CTA, but wait for it
      lpc::cluster_sync();
      lpc::cluster_sync();
    }
    if (len <= 0 && split == 0)  // an empty context attends to nothing
      for (int i = threadIdx.x; i < heads * D; i += blockDim.x)
        out[(b * H + h0) * D + i] = Num<T>::from_f(0.f);
    return;
  }
  const int start = split * chunk;
  const int end = min(start + chunk, len);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = lane >> 2, t = lane & 3;

  const int64_t head_row = row0 + kvh * head_rows;
  const uint8_t* kc = kcodes + head_row * CB;
  const uint8_t* vc = vcodes + head_row * CB;
  const uint8_t* ks = kscales + head_row * 8;
  const uint8_t* vs = vscales + head_row * 8;
  uint8_t* ring = smem + warp * (NST * L::STAGE);

  // stage at ring offset `to` <- this warp's next tile; rows past `end` become zeros
  const uint8_t* fk = kc + (int64_t)(start + warp * TK) * CB + lane * 16;
  const uint8_t* fv = vc + (int64_t)(start + warp * TK) * CB + lane * 16;
  const uint8_t* fks = ks + (int64_t)(start + warp * TK + lane) * 8;
  const uint8_t* fvs = vs + (int64_t)(start + warp * TK + lane) * 8;
  int fleft = end - (start + warp * TK);  // keys from the next tile's first on
  const uint32_t ring_u = lpc::smem_u32(ring);
  const uint32_t fdst = ring_u + lane * 16, fdst_s = fdst - lane * 8;
  // V's 16-byte pieces are stored with their place in the row mixed with the
  // key, so that one piece of 8 keys -- what ldmatrix reads -- lies in 32 banks
  const uint32_t fdst_v = ring_u + L::CODES + (lane * 16 / CB) * CB + L::place(lane * 16 / CB, lane * 16 % CB / 16) * 16;
  auto fetch = [&](int to) {
    if (fleft >= TK) {
#pragma unroll
      for (int c = 0; c < L::CODES / 512; ++c) {
        cp16(fdst + to + c * 512, fk + c * 512);
        cp16(fdst_v + to + c * 512, fv + c * 512);
      }
      cp8(fdst_s + to + 2 * L::CODES, fks);
      cp8(fdst_s + to + 2 * L::CODES + L::SCALES, fvs);
    } else if (fleft > 0) {
#pragma unroll
      for (int c = 0; c < L::CODES / 512; ++c) {
        const bool ok = (c * 512 + lane * 16) / CB < fleft;
        cp16z(fdst + to + c * 512, ok ? fk + c * 512 : kc, ok);
        cp16z(fdst_v + to + c * 512, ok ? fv + c * 512 : vc, ok);
      }
      const bool ok = lane < fleft;
      cp8z(fdst_s + to + 2 * L::CODES, ok ? fks : ks, ok);
      cp8z(fdst_s + to + 2 * L::CODES + L::SCALES, ok ? fvs : vs, ok);
    }
    cp_commit();
    fleft -= W * TK;
    fk += W * TK * CB;
    fv += W * TK * CB;
    fks += W * TK * 8;
    fvs += W * TK * 8;
  };
#pragma unroll
  for (int i = 0; i < NST - 1; ++i) fetch(i * L::STAGE);

  // q as the products' column operand: column c is head c, or, where at most 4
  // heads share the KV head (NH = 1), head c / 2 of the even columns, so that
  // each lane has one head's scores.  Lane (r, t) holds column r's dims of words
  // t*KW .. t*KW + KW - 1: word w covers dims 4w..4w+3 of each group.
  const int qh = NH == 1 ? r >> 1 : r;
  const bool has_q = qh < heads;
  uint32_t qb[KW][2][2];
  float qs0 = 0.f, qs1 = 0.f, amax = 0.f;
  float qv[KW][8];
  {
    const T* qp = q + (b * H + h0 + (has_q ? qh : 0)) * D + 4 * KW * t;
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      uint32_t w[2 * KW];  // 4 KW dims
      if constexpr (KW == 1) {
        const uint2 v = lpc::ld_dep8(qp + g * (D / 2));
        w[0] = v.x;
        w[1] = v.y;
      } else {
#pragma unroll
        for (int i = 0; i < KW / 2; ++i) {
          const uint4 v = lpc::ld_dep16(qp + g * (D / 2) + 8 * i);
          w[4 * i] = v.x;
          w[4 * i + 1] = v.y;
          w[4 * i + 2] = v.z;
          w[4 * i + 3] = v.w;
        }
      }
#pragma unroll
      for (int i = 0; i < 2 * KW; ++i) {
        float lo, hi;
        unpack_sm<T>(w[i], lo, hi);
        if (!has_q) lo = hi = 0.f;
        qv[i / 2][g * 4 + 2 * (i & 1)] = lo;
        qv[i / 2][g * 4 + 2 * (i & 1) + 1] = hi;
        amax = fmaxf(amax, fmaxf(fabsf(lo), fabsf(hi)));
        if (g == 0) qs0 += lo + hi; else qs1 += lo + hi;
      }
    }
  }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    qs0 += __shfl_xor_sync(0xffffffffu, qs0, o);
    qs1 += __shfl_xor_sync(0xffffffffu, qs1, o);
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  }
  int e = 0;
  if (amax > 0.f && amax < INFINITY) e = 14 - ((int)(__float_as_uint(amax) >> 23) - 127);
  e = max(-100, min(100, e));
  const float up = __uint_as_float((uint32_t)(127 + e) << 23);
  // NH = 1: operands of the bytes (q0 | 0) and of their upper nibbles (-q0 | q1 / 16),
  // for the even | odd columns; NH = 2: of the lower nibbles (q0) and the upper (q1 / 16)
#pragma unroll
  for (int w = 0; w < KW; ++w)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t q0 = pack_half2(qv[w][i] * up, qv[w][i + 2] * up);
      const uint32_t q1 = pack_half2(qv[w][4 + i] * (up * 0.0625f), qv[w][6 + i] * (up * 0.0625f));
      if constexpr (NH == 1) {
        qb[w][0][i] = r & 1 ? 0u : q0;
        qb[w][1][i] = r & 1 ? q1 : q0 ^ 0x80008000u;
      } else {
        qb[w][0][i] = q0;
        qb[w][1][i] = q1;
      }
    }
  // what this lane needs of its score columns: head t, or heads 2t and 2t + 1
  float cs[NH], z0[NH], z1[NH], M[NH], l[NH], a0s[NH], a1s[NH];
#pragma unroll
  for (int n = 0; n < NH; ++n) {
    const int from = (2 * t + n) * 4;
    const int eh = __shfl_sync(0xffffffffu, e, from);
    cs[n] = __uint_as_float((uint32_t)(127 + 24 - eh) << 23) * scale_log2;
    z0[n] = __shfl_sync(0xffffffffu, qs0, from) * scale_log2;
    z1[n] = __shfl_sync(0xffffffffu, qs1, from) * scale_log2;
    M[n] = -INFINITY;
    l[n] = a0s[n] = a1s[n] = 0.f;
  }
  constexpr int AG = NH;  // NH = 1: columns 2t and 2t + 1 are the groups of head t
  float acc[AG][VM][4];
#pragma unroll
  for (int g = 0; g < AG; ++g)
#pragma unroll
    for (int i = 0; i < VM; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[g][i][j] = 0.f;

  constexpr uint32_t LOW = 0x000F000Fu, HIGH = 0x00F000F0u, BYTES = 0x00FF00FFu;
  const uint32_t even = r & 1 ? 0u : 0xFFFFFFFFu;
  // this lane's row of the V matrices: lanes 0-7 keys 0-7 and 8-15 keys 8-15 of
  // the first piece, 16-31 the same of the second
  const uint32_t vsrc = (lane & 15) * CB + (D == 32 ? 0 : L::place(lane & 7, lane >> 4) * 16);
  int at = 0, to = (NST - 1) * L::STAGE;  // ring offsets of this tile and of the next fetch
  for (int left = end - (start + warp * TK); left > 0; left -= W * TK) {
    __syncwarp();  // every lane has read the stage that is filled next
    fetch(to);
    cp_wait<NST - 1>();
    __syncwarp();
    const uint8_t* sk = ring + at;
    const uint32_t sv = ring_u + at + L::CODES;
    const uint8_t* sks = sk + 2 * L::CODES;
    const uint8_t* svs = sks + L::SCALES;
    at = at == (NST - 1) * L::STAGE ? 0 : at + L::STAGE;
    to = to == (NST - 1) * L::STAGE ? 0 : to + L::STAGE;

    // scores of keys 16u + r and 16u + r + 8
    float x[2][2][NH];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      uint32_t wa[KW], wb[KW];
      const uint8_t* pa = sk + (16 * u + r) * CB + t * (KW * 4);
      const uint8_t* pb = pa + 8 * CB;
      if constexpr (KW == 4) {
        const uint4 a = *reinterpret_cast<const uint4*>(pa), c = *reinterpret_cast<const uint4*>(pb);
        wa[0] = a.x; wa[1] = a.y; wa[2] = a.z; wa[3] = a.w;
        wb[0] = c.x; wb[1] = c.y; wb[2] = c.z; wb[3] = c.w;
      } else if constexpr (KW == 2) {
        const uint2 a = *reinterpret_cast<const uint2*>(pa), c = *reinterpret_cast<const uint2*>(pb);
        wa[0] = a.x; wa[1] = a.y;
        wb[0] = c.x; wb[1] = c.y;
      } else {
        wa[0] = *reinterpret_cast<const uint32_t*>(pa);
        wb[0] = *reinterpret_cast<const uint32_t*>(pb);
      }
      float c0[4], c1[4];
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        if constexpr (NH == 1) {
          const uint32_t a0 = wa[w] & BYTES, b0 = wb[w] & BYTES;
          const uint32_t a1 = __byte_perm(wa[w], 0u, 0x4341), b1 = __byte_perm(wb[w], 0u, 0x4341);
          if (w == 0) mma_f16_first(c0, a0, b0, a1, b1, qb[w][0][0], qb[w][0][1]);
          else mma_f16(c0, a0, b0, a1, b1, qb[w][0][0], qb[w][0][1]);
          mma_f16(c0, a0 & HIGH, b0 & HIGH, a1 & HIGH, b1 & HIGH, qb[w][1][0], qb[w][1][1]);
        } else {
          const uint32_t a8 = wa[w] >> 8, b8 = wb[w] >> 8;
          if (w == 0) {
            mma_f16_first(c0, wa[w] & LOW, wb[w] & LOW, a8 & LOW, b8 & LOW, qb[w][0][0], qb[w][0][1]);
            mma_f16_first(c1, wa[w] & HIGH, wb[w] & HIGH, a8 & HIGH, b8 & HIGH, qb[w][1][0],
                          qb[w][1][1]);
          } else {
            mma_f16(c0, wa[w] & LOW, wb[w] & LOW, a8 & LOW, b8 & LOW, qb[w][0][0], qb[w][0][1]);
            mma_f16(c1, wa[w] & HIGH, wb[w] & HIGH, a8 & HIGH, b8 & HIGH, qb[w][1][0], qb[w][1][1]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint2 w = *reinterpret_cast<const uint2*>(sks + (16 * u + r + 8 * i) * 8);
        float s0, m0, s1, m1;
        unpack_sm<T>(w.x, s0, m0);
        unpack_sm<T>(w.y, s1, m1);
#pragma unroll
        for (int n = 0; n < NH; ++n) {
          const float sc = NH == 1 ? fmaf(s1, c0[2 * i + 1], s0 * c0[2 * i])
                                   : fmaf(s1, c1[2 * i + n], s0 * c0[2 * i + n]);
          x[u][i][n] = fmaf(sc, cs[n], fmaf(m1, z1[n], m0 * z0[n]));
        }
      }
    }
    if (left < TK) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (16 * u + 8 * i + r >= left)
#pragma unroll
            for (int n = 0; n < NH; ++n) x[u][i][n] = -INFINITY;
    }
    // the reference M, moved only when a key rises far above it
    const uint32_t bits = scale_bits<T>(*reinterpret_cast<const uint2*>(svs + lane * 8));
    const float most = scale_exponent<T>(__reduce_max_sync(0xffffffffu, bits));
    bool rise = false;  // for all that the highest score and the largest scale say
#pragma unroll
    for (int n = 0; n < NH; ++n)
      rise |= fmaxf(fmaxf(x[0][0][n], x[0][1][n]), fmaxf(x[1][0][n], x[1][1][n])) + most > M[n] + LIFT;
    if (__any_sync(0xffffffffu, rise)) {
      const float mine = scale_exponent<T>(bits);
      float v[NH];
#pragma unroll
      for (int n = 0; n < NH; ++n) v[n] = -INFINITY;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float e = __shfl_sync(0xffffffffu, mine, 16 * u + 8 * i + r);
#pragma unroll
          for (int n = 0; n < NH; ++n) v[n] = fmaxf(v[n], x[u][i][n] + e);
        }
#pragma unroll
      for (int n = 0; n < NH; ++n) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) v[n] = fmaxf(v[n], __shfl_xor_sync(0xffffffffu, v[n], o));
        const float next = fmaxf(fmaxf(M[n], v[n] - RISE), -3.4e38f);
        const float f = fast_exp2(M[n] - next);
        M[n] = next;
        l[n] *= f;
        a0s[n] *= f;
        a1s[n] *= f;
#pragma unroll
        for (int g = 0; g < AG; ++g)
#pragma unroll
          for (int i = 0; i < VM; ++i) {
            acc[g][i][n] *= f;
            acc[g][i][2 + n] *= f;
            if constexpr (NH == 1) {
              acc[g][i][1] *= f;
              acc[g][i][3] *= f;
            }
          }
      }
    }
    // weights, then the output products
    uint32_t pb[2][2][2];  // [u][group][keys 0-7 / 8-15]
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint2 w = *reinterpret_cast<const uint2*>(svs + (16 * u + r + 8 * i) * 8);
        float s0, m0, s1, m1;
        unpack_sm<T>(w.x, s0, m0);
        unpack_sm<T>(w.y, s1, m1);
        float p[2] = {0.f, 0.f};
#pragma unroll
        for (int n = 0; n < NH; ++n) {
          p[n] = fast_exp2(x[u][i][n] - M[n]);
          l[n] += p[n];
          a0s[n] = fmaf(p[n], m0, a0s[n]);
          a1s[n] = fmaf(p[n], m1, a1s[n]);
        }
        if constexpr (std::is_same<T, __half>::value) {
          // an fp16 output shows the rounding of P s to fp16, which the products
          // take times a code; with 8 times it taken out, times a code - 8
#pragma unroll
          for (int n = 0; n < NH; ++n) {
            const float e0 = p[n] * s0, e1 = p[n] * s1;
            a0s[n] = fmaf(8.f, e0 - __half2float(__float2half_rn(e0)), a0s[n]);
            a1s[n] = fmaf(8.f, e1 - __half2float(__float2half_rn(e1)), a1s[n]);
          }
        }
        if constexpr (NH == 1 && FINE) {
          // columns 2t and 2t + 1 carry head t's groups: the lower nibbles times (P s0 | 0)
          // and the upper ones times (0 | P s1)
          const uint32_t both = transpose8(pack_half2(p[0] * s0, p[0] * s1));
          pb[u][0][i] = both & even;
          pb[u][1][i] = both & ~even;
        } else if constexpr (NH == 1) {
          // the same, the bytes times (P s0 | 0) and their upper nibbles times
          // (-P s0 | P s1), which leave the lower nibbles in one
          pb[u][1][i] = transpose8(pack_half2(-p[0] * s0, p[0] * s1));
          pb[u][0][i] = (pb[u][1][i] ^ 0x80008000u) & even;
        } else {
          pb[u][0][i] = transpose8(pack_half2(p[0] * s0, p[1] * s0));
          pb[u][1][i] = transpose8(pack_half2(p[0] * s1, p[1] * s1));
        }
      }
      // codes of keys 16u .. 16u + 15, 16 dims (8 units) of each group at a time
      if constexpr (!FINE)
#pragma unroll
        for (int j = 0; j < VM; j += NI) {
          uint32_t v[4];
          const uint32_t src = sv + 16 * u * CB + (j == 0 ? vsrc : vsrc ^ 32u);
          if constexpr (VM == 1) ldm2(v, src);
          else ldm4(v, src);
#pragma unroll
          for (int i = 0; i < NI; ++i) {
            const uint32_t lo = v[2 * i], hi = v[2 * i + 1];
            if constexpr (NH == 1) {
              const uint32_t l0 = lo & BYTES, h0 = hi & BYTES;
              const uint32_t l1 = __byte_perm(lo, 0u, 0x4341), h1 = __byte_perm(hi, 0u, 0x4341);
              mma_f16(acc[0][j + i], l0, l1, h0, h1, pb[u][0][0], pb[u][0][1]);
              mma_f16(acc[0][j + i], l0 & HIGH, l1 & HIGH, h0 & HIGH, h1 & HIGH, pb[u][1][0], pb[u][1][1]);
            } else {
              const uint32_t lo8 = lo >> 8, hi8 = hi >> 8;
              mma_f16(acc[0][j + i], lo & LOW, lo8 & LOW, hi & LOW, hi8 & LOW, pb[u][0][0], pb[u][0][1]);
              mma_f16(acc[AG - 1][j + i], lo & HIGH, lo8 & HIGH, hi & HIGH, hi8 & HIGH, pb[u][1][0],
                      pb[u][1][1]);
            }
          }
        }
    }
    if constexpr (FINE)
#pragma unroll
      for (int j = 0; j < VM; j += NI) {
        float part[AG][NI][4];  // of this tile
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          uint32_t v[4];
          const uint32_t src = sv + 16 * u * CB + (j == 0 ? vsrc : vsrc ^ 32u);
          if constexpr (VM == 1) ldm2(v, src);
          else ldm4(v, src);
#pragma unroll
          for (int i = 0; i < NI; ++i) {
            const uint32_t lo = v[2 * i], hi = v[2 * i + 1];
            const uint32_t l0 = (lo << 4) & HIGH, l1 = (lo >> 4) & HIGH, h0 = (hi << 4) & HIGH,
                           h1 = (hi >> 4) & HIGH;
            if (u == 0) mma_f16_first(part[0][i], l0, l1, h0, h1, pb[0][0][0], pb[0][0][1]);
            else mma_f16(part[0][i], l0, l1, h0, h1, pb[1][0][0], pb[1][0][1]);
            const uint32_t l8 = (lo >> 8) & HIGH, h8 = (hi >> 8) & HIGH;
            if (u == 0 && AG == 2)
              mma_f16_first(part[1 % AG][i], lo & HIGH, l8, hi & HIGH, h8, pb[0][1][0], pb[0][1][1]);
            else
              mma_f16(part[AG - 1][i], lo & HIGH, l8, hi & HIGH, h8, pb[u][1][0], pb[u][1][1]);
          }
        }
#pragma unroll
        for (int g = 0; g < AG; ++g)
#pragma unroll
          for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int n = 0; n < 4; ++n) acc[g][j + i][n] += part[g][i][n];
      }
  }
  cp_wait<0>();
  // a head's sums over the 8 lanes that hold its keys
#pragma unroll
  for (int n = 0; n < NH; ++n)
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
      l[n] += __shfl_xor_sync(0xffffffffu, l[n], o);
      a0s[n] += __shfl_xor_sync(0xffffffffu, a0s[n], o);
      a1s[n] += __shfl_xor_sync(0xffffffffu, a1s[n], o);
    }
  __syncthreads();  // the rings become the merge buffer: [W][HB][D + 2]
  float* red = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int n = 0; n < NH; ++n) {
    const int h = NH == 1 ? t : 2 * t + n;
    if (h >= heads) continue;
    float* p = red + (warp * HB + h) * (D + 2);
#pragma unroll
    for (int i = 0; i < VM; ++i) {
      // rows r and r + 8 of product i are the two dims of unit 8i + r
      const int d = 2 * (8 * i + r);
      constexpr int g1 = AG - 1;
      const int n1 = NH == 1 ? 1 : n;
      constexpr float ONE = FINE ? 1048576.f : 16777216.f;
      p[d] = fmaf(acc[0][i][n], ONE, a0s[n]);
      p[d + 1] = fmaf(acc[0][i][2 + n], ONE, a0s[n]);
      p[d + D / 2] = fmaf(acc[g1][i][n1], 1048576.f, a1s[n]);
      p[d + D / 2 + 1] = fmaf(acc[g1][i][2 + n1], 1048576.f, a1s[n]);
    }
    if (r == 0) {
      p[D] = M[n];
      p[D + 1] = l[n];
    }
  }
  __syncthreads();
  for (int idx = threadIdx.x; idx < heads * D; idx += W * 32) {
    const int h = idx / D, d = idx - h * D;
    float Mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < W; ++w) Mx = fmaxf(Mx, red[(w * HB + h) * (D + 2) + D]);
    const float Mu = Mx == -INFINITY ? 0.f : Mx;
    float O = 0.f, Ls = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float* p = red + (w * HB + h) * (D + 2);
      const float f = fast_exp2(p[D] - Mu);
      O = fmaf(f, p[d], O);
      Ls = fmaf(f, p[D + 1], Ls);
    }
    const int64_t bh = b * H + h0 + h;
    if (nsplits == 1) {
      out[bh * D + d] = Num<T>::from_f(Ls == 0.f ? 0.f : O / Ls);
    } else if (W == 16 && cluster) {
      float* p = red + (W * HB + h) * (D + 2);
      p[d] = O;
      if (d == 0) {
        p[D] = Mx;
        p[D + 1] = Ls;
      }
    } else {
      const int64_t pi = bh * max_splits + split;
      part_o[pi * D + d] = O;
      if (d == 0) {
        part_ml[2 * pi] = Mx;
        part_ml[2 * pi + 1] = Ls;
      }
    }
  }
  if (W == 4 || !cluster || nsplits == 1) return;
  // the splits of this cluster: each CTA adds its share of the outputs over all
  // of them through distributed shared memory, in split order
  lpc::cluster_sync();
  const int share = (heads * D + nsplits - 1) / nsplits;
  for (int i = threadIdx.x; i < share; i += W * 32) {
    const int idx = split * share + i;
    if (idx >= heads * D) break;
    const int h = idx / D, d = idx - h * D;
    const uint32_t at_h = lpc::smem_u32(red + (W * HB + h) * (D + 2));
    float Mx = -INFINITY, mv[CLUSTER], lv[CLUSTER], ov[CLUSTER];
#pragma unroll
    for (int s = 0; s < CLUSTER; ++s)
      if (s < nsplits) {
        const uint32_t p = lpc::mapa_shared(at_h, s);
        mv[s] = ld_cluster(p + D * 4);
        lv[s] = ld_cluster(p + D * 4 + 4);
        ov[s] = ld_cluster(p + d * 4);
      }
#pragma unroll
    for (int s = 0; s < CLUSTER; ++s)
      if (s < nsplits) Mx = fmaxf(Mx, mv[s]);
    const float Mu = Mx == -INFINITY ? 0.f : Mx;
    float O = 0.f, Ls = 0.f;
#pragma unroll
    for (int s = 0; s < CLUSTER; ++s)
      if (s < nsplits) {
        const float f = fast_exp2(mv[s] - Mu);
        O = fmaf(f, ov[s], O);
        Ls = fmaf(f, lv[s], Ls);
      }
    out[(b * H + h0 + h) * D + d] = Num<T>::from_f(Ls == 0.f ? 0.f : O / Ls);
  }
  lpc::cluster_sync();  // no CTA leaves while its sums are read
}

// One CTA per (sequence, head).  Warp w adds the splits w, w + CWARPS, ..., the
// warps' sums meet in shared memory: the order is fixed.  The kernel is a chain of
// latencies, so the length and the first AHEAD splits a warp are asked for at once,
// before it is known how many the sequence has (the others' numbers are not used):
// one of 131,000 keys 31.6 us against 33.4, 8 of 8,000 19.2 against 20.3.
constexpr int CWARPS = 8;
template <typename T, int D>
__global__ void __launch_bounds__(CWARPS * 32)
    kv4_combine_kernel(const float* part_o, const float* part_ml,
                       const int32_t* __restrict__ seq_lens, T* out, int H,
                       int max_splits, int chunk, lpc::Kv4Rows rows) {
  lpc::pdl_trigger();
  lpc::pdl_wait();
  constexpr int DPL = D / 32, AHEAD = 4;
  __shared__ float so[CWARPS][D + 2];
  const int64_t bh = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t b = bh / H;
  const float2* ml = reinterpret_cast<const float2*>(part_ml) + bh * max_splits;
  const float* po = part_o + bh * max_splits * D + lane * DPL;
  const float first_m = lane < max_splits ? ml[lane].x : 0.f;
  float pre[AHEAD][DPL];
  float2 pre_ml[AHEAD];
#pragma unroll
  for (int k = 0; k < AHEAD; ++k) {
    const int s = warp + k * CWARPS;
    pre_ml[k] = make_float2(0.f, 0.f);
    if (s < max_splits) pre_ml[k] = ml[s];
#pragma unroll
    for (int i = 0; i < DPL; ++i) pre[k][i] = s < max_splits ? po[(int64_t)s * D + i] : 0.f;
  }
  int64_t row0, head_rows, cap;
  const bool inside = rows.locate(b, &row0, &head_rows, &cap);
  int len = lpc::ld_dep(seq_lens + b);
  if (len > cap) len = (int)cap;
  const int ns = inside && len > 0 ? (len + chunk - 1) / chunk : 0;
  if (ns <= 1) return;  // written by the split kernel
  float mx = lane < ns ? first_m : -INFINITY;
  for (int s = lane + 32; s < ns; s += 32) mx = fmaxf(mx, ml[s].x);
#pragma unroll
  for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  const float Mu = mx == -INFINITY ? 0.f : mx;
  float O[DPL], Ls = 0.f;
#pragma unroll
  for (int i = 0; i < DPL; ++i) O[i] = 0.f;
#pragma unroll
  for (int k = 0; k < AHEAD; ++k)
    if (warp + k * CWARPS < ns) {
      const float f = fast_exp2(pre_ml[k].x - Mu);
#pragma unroll
      for (int i = 0; i < DPL; ++i) O[i] = fmaf(f, pre[k][i], O[i]);
      Ls = fmaf(f, pre_ml[k].y, Ls);
    }
#pragma unroll 4
  for (int s = warp + AHEAD * CWARPS; s < ns; s += CWARPS) {
    const float2 v = ml[s];
    const float f = fast_exp2(v.x - Mu);
#pragma unroll
    for (int i = 0; i < DPL; ++i) O[i] = fmaf(f, po[(int64_t)s * D + i], O[i]);
    Ls = fmaf(f, v.y, Ls);
  }
#pragma unroll
  for (int i = 0; i < DPL; ++i) so[warp][lane * DPL + i] = O[i];
  if (lane == 0) so[warp][D] = Ls;
  __syncthreads();
  for (int d = threadIdx.x; d < D; d += CWARPS * 32) {
    float o = 0.f, l = 0.f;
#pragma unroll
    for (int w = 0; w < CWARPS; ++w) {
      o += so[w][d];
      l += so[w][D];
    }
    out[bh * D + d] = Num<T>::from_f(l == 0.f ? 0.f : o / l);
  }
}

// A cluster of up to 4 CTAs of 16 warps merges its splits in distributed shared
// memory: 1000 keys of 32 KV heads 5.9 us against 6.7 with the second kernel, 8
// sequences of 8,000 keys 19.4 against 21.3.  128 CTAs in such clusters fit 16
// SMs of each of the GPU's 8 parts at once; 144 in clusters of 6 did not (74 us
// against 41 for three sequences of 60,000).
bool merges_in_cluster(int64_t pairs, int64_t splits) {
  return splits > 1 && splits <= CLUSTER && pairs * splits <= 128;
}

template <typename T, int D, int NH, int W, bool FINE>
int launch(const lpc_kv4* kv, const void* q, const int32_t* lens, void* out, float* po, float* pml,
           int64_t batch, int heads, int max_splits, int chunk, float scale_log2, cudaStream_t s) {
  using L = Layout<D, W>;
  static std::atomic<uint64_t> mask{0};
  int rc = lpc::once_per_device_smem((const void*)kv4_split_kernel<T, D, NH, W, FINE>, L::SMEM, mask);
  if (rc) return rc;
  const int G = heads / kv->kv_heads;
  const int blocks = (G + HB - 1) / HB;
  const int grid_splits = (int)((kv->max_seq_len + chunk - 1) / chunk);
  const lpc::Kv4Rows rows = lpc::kv4_rows(kv);
  const int cluster = W == 16 && merges_in_cluster(batch * kv->kv_heads * blocks, grid_splits);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = lpc::use_pdl() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)grid_splits;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid_splits, (unsigned)(kv->kv_heads * blocks), (unsigned)batch);
  cfg.blockDim = dim3(W * 32);
  cfg.dynamicSmemBytes = L::SMEM;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = cluster ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, kv4_split_kernel<T, D, NH, W, FINE>, (const T*)q,
                         (const uint8_t*)kv->key_codes, (const uint8_t*)kv->key_scales,
                         (const uint8_t*)kv->value_codes, (const uint8_t*)kv->value_scales, lens,
                         (T*)out, po, pml, heads, G, blocks, max_splits, chunk, cluster, scale_log2,
                         rows) != cudaSuccess)
    return lpc::check_launch("decode_attention_int4 (split)");
  if ((rc = lpc::check_launch("decode_attention_int4 (split)"))) return rc;
  if (grid_splits == 1 || cluster) return LPC_OK;
  cfg.numAttrs = 1;
  cfg.gridDim = dim3((unsigned)(batch * heads));
  cfg.blockDim = dim3(CWARPS * 32);
  cfg.dynamicSmemBytes = 0;
  if (cudaLaunchKernelEx(&cfg, kv4_combine_kernel<T, D>, (const float*)po, (const float*)pml, lens,
                         (T*)out, heads, max_splits, chunk, rows) != cudaSuccess)
    return lpc::check_launch("decode_attention_int4 (combine)");
  return lpc::check_launch("decode_attention_int4 (combine)");
}

// Whether V's sums are taken finely (FINE of the split kernel).  The tensor core does not
// normalise subnormal operands and cuts what it adds: a code in the lowest four bits of its
// half keeps 10 bits less of its product than fp32, and the accumulator cuts again as it
// grows, always towards zero.  The sums come out 3 to 6e-6 of their codes' part too
// small, which an output, the difference of the codes' and the minima's parts, shows once
// many keys average to little.  FINE: codes in bits 4 to 7, and sums that start at zero
// with each tile of 32 keys and are added in fp32.  Relative error plain / FINE (fp32 with
// outputs rounded once): fp16 of 4096 keys 2.6 / 2.5e-4 (2.0e-4), 32,768 3.4 / 2.8,
// 131,072 5.1 / 2.6; bf16 of 131,072 1.84 / 1.83e-3 (1.73), 4,000,000 3.4 / 1.8.  It costs
// 8%: fp16, 32 sequences of 1 to 4096 keys 59.7 / 64.6 us, 3 of 60,000 42.1 / 45.4.
bool sums_finely(const lpc_kv4* kv) {
  return kv->max_seq_len > (kv->dtype == LPC_DTYPE_F16 ? 1 << 13 : 1 << 18);
}

template <typename T, int D>
int launch_nw(const lpc_kv4* kv, const void* q, const int32_t* lens, void* out, float* po,
              float* pml, int64_t batch, int heads, int max_splits, int chunk, float scale_log2,
              bool wide, cudaStream_t s) {
#define LPC_KV4_NW(NH, W)                                                                         \
  return sums_finely(kv) ? launch<T, D, NH, W, true>(kv, q, lens, out, po, pml, batch, heads,     \
                                                     max_splits, chunk, scale_log2, s)            \
                         : launch<T, D, NH, W, false>(kv, q, lens, out, po, pml, batch, heads,    \
                                                      max_splits, chunk, scale_log2, s)
  if (heads / kv->kv_heads <= 4) {
    if (wide) LPC_KV4_NW(1, 16);
    LPC_KV4_NW(1, 4);
  }
  if (wide) LPC_KV4_NW(2, 16);
  LPC_KV4_NW(2, 4);
#undef LPC_KV4_NW
}

constexpr int64_t MAX_BATCH = 65535;
constexpr int64_t MAX_SEQ = 65535LL * UNIT;
constexpr int MAX_HEADS = 65535;

// Split length (a multiple of UNIT) and CTA width of a launch, by the least
// estimated time, in keys of one of the 592 four-warp CTAs that run at once (about 67
// keys a microsecond at D = 128).  A CTA costs its keys and an overhead (q, the
// pipeline's start, the merge); splits that no cluster merges cost the second
// kernel, and each a little there.
//   * 4 warps, four CTAs an SM: any number of rounds of CTAs, which overlap.  Up
//     to four rounds count as whole rounds.  Among lengths within an eighth of the
//     least the shortest is taken: sequences are rarely all of the full length,
//     and short splits even them out (32 sequences of 1 to 4096 keys: 59 us with
//     splits of 1024, 63 with 4096).
//   * 16 warps, one CTA an SM, one round: a quarter of the splits for the same
//     keys a warp.  Measured 16 / 4 warps, us: 1000 keys of 32 heads 5.9 / 7.6,
//     300 keys of 4 x 32 heads 4.5 / 7.1, three sequences of 60,000 (64 heads on
//     8) 41 / 46, one of 131,000 (32 on 8) 33 / 37 (then with a slower second kernel).
//     They fill their SMs: where it costs at most an eighth more keys a CTA, SMs are
//     left free for the second kernel's CTAs to wait on (one of 32,000 keys, 32 on 8:
//     13.6 us in 16 splits, 14.8 in 18).
constexpr int64_t SLOTS_PER_SM = 4;
constexpr int64_t JOIN_PER_SM = 6;  // CTAs of the second kernel that an SM holds
int split_keys(const lpc_kv4* kv, int64_t batch, int heads, bool* wide) {
  const int64_t G = heads / kv->kv_heads, blocks = (G + HB - 1) / HB;
  const int64_t pairs = batch * kv->kv_heads * blocks, cap = kv->max_seq_len;
  const int64_t sms = lpc::current_device_sms(), slots = SLOTS_PER_SM * sms;
  const int64_t overhead = G <= 4 ? 200 : 400;
  auto joined = [](int64_t splits) { return splits > 1 ? 200 + 4 * splits : 0; };
  auto units = [](int64_t keys) { return (keys + UNIT - 1) / UNIT * UNIT; };
  auto estimate = [&](int64_t chunk) {
    const int64_t splits = (cap + chunk - 1) / chunk, ctas = pairs * splits, each = chunk + overhead;
    const int64_t t = ctas <= 4 * slots ? (ctas + slots - 1) / slots * each
                                        : (ctas * each + each * slots / 2) / slots;
    return t + joined(splits);
  };
  // 1 to 12 splits, and what fills 1 to 8 rounds
  constexpr int CAND = 20;
  int64_t chunks[CAND], costs[CAND], least = INT64_MAX;
  int count = 0;
  for (int i = 0; i < CAND; ++i) {
    const int64_t n = i < 12 ? i + 1 : (i - 11) * slots / pairs;
    if (n < 1 || (n > 1 && n * pairs > 8 * slots)) continue;
    const int64_t chunk = units((cap + n - 1) / n);
    chunks[count] = chunk;
    costs[count] = estimate(chunk);
    least = std::min(least, costs[count++]);
  }
  int64_t best = INT64_MAX;
  for (int i = 0; i < count; ++i)
    if (costs[i] <= least + least / 8) best = std::min(best, chunks[i]);
  *wide = false;
  if (pairs <= sms) {
    auto even = [&](int64_t n) { return units((cap + n - 1) / n); };
    int64_t chunk = even(sms / pairs);
    if (!merges_in_cluster(pairs, (cap + chunk - 1) / chunk)) {
      const int64_t n = (sms - (batch * heads + JOIN_PER_SM - 1) / JOIN_PER_SM) / pairs;
      if (n >= 1 && even(n) <= chunk + chunk / 8) chunk = even(n);
    }
    const int64_t splits = (cap + chunk - 1) / chunk;
    const int64_t t = chunk / 4 + 220 + (merges_in_cluster(pairs, splits) ? 80 : joined(splits));
    if (t < least) {
      *wide = true;
      return (int)chunk;
    }
  }
  return (int)best;
}

bool sizes_ok(const lpc_kv4* kv, int64_t batch, int heads) {
  return batch >= 0 && batch <= MAX_BATCH && heads > 0 && heads <= MAX_HEADS &&
         heads % kv->kv_heads == 0 && kv->max_seq_len <= MAX_SEQ && batch * heads <= 0x7fffffffLL;
}

}  // namespace

namespace {

struct Plan {
  int chunk, splits;
  bool wide, joined;  // 16-warp CTAs; splits merged by the second kernel
};
Plan make_plan(const lpc_kv4* kv, int64_t batch, int heads) {
  Plan p;
  p.chunk = split_keys(kv, batch, heads, &p.wide);
  p.splits = (int)((kv->max_seq_len + p.chunk - 1) / p.chunk);
  const int64_t pairs = batch * kv->kv_heads * ((heads / kv->kv_heads + HB - 1) / HB);
  p.joined = p.splits > 1 && !(p.wide && merges_in_cluster(pairs, p.splits));
  return p;
}
int64_t plan_bytes(const Plan& p, const lpc_kv4* kv, int64_t batch, int heads) {
  return p.joined ? batch * heads * p.splits * (int64_t)(kv->head_dim + 2) * 4 : 0;
}

}  // namespace

extern "C" int64_t lpc_decode_attention_int4_workspace_bytes(const lpc_kv4* kv, int64_t batch,
                                                             int heads) {
  if (lpc::kv4_check(kv, "decode_attention_int4") || !sizes_ok(kv, batch, heads) || batch == 0)
    return 0;
  return plan_bytes(make_plan(kv, batch, heads), kv, batch, heads);
}

extern "C" int lpc_decode_attention_int4_kernels(const lpc_kv4* kv, int64_t batch, int heads) {
  if (lpc::kv4_check(kv, "decode_attention_int4") || !sizes_ok(kv, batch, heads) || batch == 0)
    return 0;
  return make_plan(kv, batch, heads).joined ? 2 : 1;
}

extern "C" int lpc_decode_attention_int4(const lpc_kv4* kv, const void* q, const int32_t* seq_lens,
                                         void* out, void* workspace, int64_t workspace_bytes,
                                         int64_t batch, int heads, float sm_scale, void* stream) {
  using namespace lpc;
  int rc = kv4_check(kv, "decode_attention_int4");
  if (rc) return rc;
  if (!sizes_ok(kv, batch, heads) || (kv->max_batch > 0 && batch > kv->max_batch)) {
    set_error("decode_attention_int4: invalid sizes (batch=%lld heads=%d kv_heads=%d "
              "max_batch=%lld max_seq_len=%lld)", (long long)batch, heads, kv->kv_heads,
              (long long)kv->max_batch, (long long)kv->max_seq_len);
    return LPC_ERR_INVALID;
  }
  if (batch == 0) return LPC_OK;
  if (!q || !seq_lens || !out || !aligned16(q) || !aligned16(out)) {
    set_error("decode_attention_int4: q, seq_lens and out must be given, q and out 16-byte aligned");
    return LPC_ERR_INVALID;
  }
  const Plan plan = make_plan(kv, batch, heads);
  const int chunk = plan.chunk;
  const int64_t splits = plan.splits, need = plan_bytes(plan, kv, batch, heads);
  const bool wide = plan.wide;
  if (need && (!workspace || workspace_bytes < need || !aligned16(workspace))) {
    set_error("decode_attention_int4: workspace of %lld bytes required, got %lld", (long long)need,
              (long long)workspace_bytes);
    return LPC_ERR_INVALID;
  }
  if ((int64_t)kv->kv_heads * ((heads / kv->kv_heads + HB - 1) / HB) > 65535) {
    set_error("decode_attention_int4: too many heads");
    return LPC_ERR_UNSUPPORTED;
  }
  float* po = static_cast<float*>(workspace);
  float* pml = po ? po + batch * heads * splits * kv->head_dim : nullptr;
  const float sl2 = sm_scale * LOG2E;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
#define LPC_KV4(T, DD) \
  return launch_nw<T, DD>(kv, q, seq_lens, out, po, pml, batch, heads, (int)splits, chunk, sl2, wide, s)
  if (kv->dtype == LPC_DTYPE_BF16) {
    if (kv->head_dim == 128) LPC_KV4(__nv_bfloat16, 128);
    if (kv->head_dim == 64) LPC_KV4(__nv_bfloat16, 64);
    LPC_KV4(__nv_bfloat16, 32);
  }
  if (kv->head_dim == 128) LPC_KV4(__half, 128);
  if (kv->head_dim == 64) LPC_KV4(__half, 64);
  LPC_KV4(__half, 32);
#undef LPC_KV4
}
