// RoPE + append into a 4-bit KV cache, and its read-back (row format: kv4.cuh).
//
// Append: qkv [B, S, (H + 2 Hkv) D] -> q rotated into q_out [B, H, S, D]; k
// rotated and rounded to the data type as the 16-bit append does, v as given,
// both held as
//   m = min of the group,  s = T(fl(fl(max - min) / 15)),
//   c = rint(clamp(fl(fl(x - m) * fl(1 / s)), 0, 15)),
// every operation one fp32 rounding, so that the same bytes come out of any
// correct evaluation.  m is exact in T.  A scale below 2^-126 (whose inverse
// fp32 does not hold) becomes 0 and its codes 0; a group with a non-finite
// value, or with a range whose scale T does not hold, holds s = m = NaN: it
// reads as NaN and not as some finite number.
//
// Bound: HBM.  A thread owns 8 rotation pairs of one (token, head): two 16-byte
// loads, and for k and v one 8-byte store of codes; the D / 16 threads of a
// row find min and max of its two groups, both packed in a word, in 2 * log2(D / 16)
// shuffles.  Measured, D = 128, bf16: four prompts of 2048 tokens, 32 heads on 8,
// 32.8 us (its bytes at 6397 GB/s 27.7; the append into a 16-bit cache 41.9), 32
// decode tokens of 32 heads 2.1 us (16-bit 2.5).  The read-back of 2 x 16,000 rows
// of 32 heads: 109 us, 96% of the rate, mostly its 16-bit output.
#include <algorithm>

#include "kv4.cuh"

LPC_DECLARE_STATUS(g_kv4_append_status)

unsigned int lpc_status_kv4_append(bool clear) {
  unsigned int v = 0;
  cudaMemcpyFromSymbol(&v, g_kv4_append_status, sizeof(v));
  if (clear && v) {
    unsigned int z = 0;
    cudaMemcpyToSymbol(g_kv4_append_status, &z, sizeof(z));
  }
  return v;
}

namespace lpc {

int kv4_check(const lpc_kv4* kv, const char* what) {
  if (!kv || !kv->key_codes || !kv->key_scales || !kv->value_codes || !kv->value_scales) {
    set_error("%s: null cache pointer", what);
    return LPC_ERR_INVALID;
  }
  if (kv->dtype != LPC_DTYPE_BF16 && kv->dtype != LPC_DTYPE_F16) {
    set_error("%s: only bf16 and fp16 are supported", what);
    return LPC_ERR_UNSUPPORTED;
  }
  if (kv->head_dim != 32 && kv->head_dim != 64 && kv->head_dim != 128) {
    set_error("%s: head_dim must be 32, 64 or 128, got %d", what, kv->head_dim);
    return LPC_ERR_UNSUPPORTED;
  }
  if (kv->kv_heads <= 0 || kv->kv_heads > 65535 || kv->max_seq_len <= 0 ||
      kv->max_seq_len > 0x7fffffffLL ||
      (kv->seq_base ? (!kv->seq_cap || kv->total_rows <= 0) : kv->max_batch <= 0)) {
    set_error("%s: invalid cache sizes (kv_heads=%d max_seq_len=%lld max_batch=%lld "
              "total_rows=%lld)", what, kv->kv_heads, (long long)kv->max_seq_len,
              (long long)kv->max_batch, (long long)kv->total_rows);
    return LPC_ERR_INVALID;
  }
  if (!aligned16(kv->key_codes) || !aligned16(kv->value_codes) ||
      (reinterpret_cast<uintptr_t>(kv->key_scales) & 7u) ||
      (reinterpret_cast<uintptr_t>(kv->value_scales) & 7u)) {
    set_error("%s: codes must be 16-byte and scales 8-byte aligned", what);
    return LPC_ERR_INVALID;
  }
  return LPC_OK;
}

}  // namespace lpc

namespace {

using lpc::Num;

// Pairs of T as they lie in a 32-bit word; a NaN wins.
template <typename T>
struct Pair;
template <>
struct Pair<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t min(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
  }
  static __device__ __forceinline__ uint32_t max(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
  }
  static __device__ __forceinline__ float lo(uint32_t w) { return lpc::bf16lo(w); }
  static __device__ __forceinline__ float hi(uint32_t w) { return lpc::bf16hi(w); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
};
template <>
struct Pair<__half> {
  static __device__ __forceinline__ uint32_t min(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
  }
  static __device__ __forceinline__ uint32_t max(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
  }
  static __device__ __forceinline__ float lo(uint32_t w) {
    return __half2float(__ushort_as_half((unsigned short)w));
  }
  static __device__ __forceinline__ float hi(uint32_t w) {
    return __half2float(__ushort_as_half((unsigned short)(w >> 16)));
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
};

template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  return make_uint4(Pair<T>::pack(f[0], f[1]), Pair<T>::pack(f[2], f[3]), Pair<T>::pack(f[4], f[5]),
                    Pair<T>::pack(f[6], f[7]));
}

// 8 table entries: as they lie (16 bits), or fp32.
template <typename TT>
struct Entries {
  uint32_t w[sizeof(TT) * 2];
  __device__ __forceinline__ void load(const TT* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(TT) / 2; ++i) {
      const uint4 v = lpc::ld_dep16(p + 4 * i);
      w[4 * i] = v.x;
      w[4 * i + 1] = v.y;
      w[4 * i + 2] = v.z;
      w[4 * i + 3] = v.w;
    }
  }
  __device__ __forceinline__ float at(int i) const {
    if constexpr (sizeof(TT) == 4) return __uint_as_float(w[i]);
    else return i & 1 ? Pair<TT>::hi(w[i / 2]) : Pair<TT>::lo(w[i / 2]);
  }
};

// a * b + c * d (c * d subtracted where MINUS), each operation rounded once.
// Products of two 16-bit numbers are exact in fp32, so that the sum may be an FMA.
template <bool EXACT, bool MINUS>
__device__ __forceinline__ float rot(float a, float b, float c, float d) {
  const float p = __fmul_rn(c, d);
  if constexpr (EXACT) return __fmaf_rn(a, b, MINUS ? -p : p);
  else return MINUS ? __fsub_rn(__fmul_rn(a, b), p) : __fadd_rn(__fmul_rn(a, b), p);
}

// d / 15, correctly rounded: division by a constant as the product with its rounded
// inverse, corrected once by the remainder d - 15 q, which an FMA gives exactly (Markstein's
// scheme).  Checked against the division for every significand; d below 2^-100, where the
// remainder loses bits, takes the division.
__device__ __forceinline__ float over15(float d) {
  if (d < 0x1p-100f) return __fdiv_rn(d, 15.f);
  const float inv = 1.f / 15.f;
  const float q = __fmul_rn(d, inv);
  return __fmaf_rn(__fmaf_rn(-15.f, q, d), inv, q);
}

// Scale (as T) of a group and the factor that turns x - min into a code; NaN
// and 0 where the group has no finite scale.
template <typename T>
__device__ __forceinline__ void group_numbers(float lo, float hi, T& s, float& inv) {
  s = Num<T>::from_f(over15(__fsub_rn(hi, lo)));
  const float sf = Num<T>::to_f(s);
  inv = 0.f;
  if (!(sf < INFINITY)) s = Num<T>::from_f(__int_as_float(0x7fffffff));
  else if (sf < 1.17549435e-38f) s = Num<T>::from_f(0.f);
  else inv = __frcp_rn(sf);
}

// rint(clamp((x - lo) * inv)) in the low bits of an fp32 number: adding 1.5 * 2^23
// rounds to an integer, halves to even.  x >= lo, so that only the upper end clamps.
__device__ __forceinline__ uint32_t code_bits(float x, float lo, float inv) {
  const float t = __fmul_rn(__fsub_rn(x, lo), inv);
  return __float_as_uint(__fadd_rn(fminf(t, 15.f), 12582912.f));
}

constexpr int THREADS = 256;

// One CTA: one token, K * (threads / chunks) of its heads; thread t owns chunk
// t % chunks of head t / chunks + k * hpb, as in the 16-bit append.
template <typename T, typename TT, int D, int K>
__global__ void __launch_bounds__(THREADS, sizeof(TT) == 2 ? 4 : 3) kv4_append_kernel(
    const T* qkv, const int64_t* positions, const TT* cosb, const TT* sinb, int64_t table_rows,
    T* q_out, uint8_t* kcodes, uint8_t* kscales, uint8_t* vcodes, uint8_t* vscales, int64_t seq,
    int H, lpc::Kv4Rows rows) {
  constexpr int C = D / 16;  // threads of a row
  constexpr bool EXACT = sizeof(TT) == 2;
  using P = Pair<T>;
  lpc::pdl_trigger();
  lpc::pdl_wait();
  const int Hkv = rows.kv_heads;
  const int all = H + 2 * Hkv;
  const int hpb = (int)blockDim.x / C;
  const int64_t tok = blockIdx.x;
  const int c = (int)threadIdx.x % C;
  const int hh0 = (int)threadIdx.x / C + (int)blockIdx.y * K * hpb;
  const int d = c * 8;
  const T* src = qkv + (tok * all + hh0) * D + d;
  uint4 x0[K], x1[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    x0[k] = x1[k] = make_uint4(0u, 0u, 0u, 0u);
    if (hh0 + k * hpb < all) {
      x0[k] = lpc::ld_dep16(src + k * hpb * D);
      x1[k] = lpc::ld_dep16(src + k * hpb * D + D / 2);
    }
  }
  const int64_t pos = lpc::ld_dep(positions + tok);
  const int64_t b = tok / seq;
  T* qdst = q_out + ((b * H + hh0) * seq + (tok - b * seq)) * D + d;
  int64_t row0 = 0, head_rows = 0, cap = 0;
  const bool inside = rows.locate(b, &row0, &head_rows, &cap);
  if (pos < 0 || !inside || pos >= cap || pos >= table_rows) {  // the same for the whole CTA
    if (pos >= 0 && threadIdx.x == 0) atomicOr(&g_kv4_append_status, LPC_DEV_ERR_BOUNDS);
    // a skipped token leaves the cache as it is; its q rows become zero
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (hh0 + k * hpb < H) {
        T* dst = qdst + (int64_t)k * hpb * seq * D;
        *reinterpret_cast<uint4*>(dst) = make_uint4(0u, 0u, 0u, 0u);
        *reinterpret_cast<uint4*>(dst + D / 2) = make_uint4(0u, 0u, 0u, 0u);
      }
    return;
  }
  Entries<TT> c0, s0, c1, s1;
  if (hh0 < H + Hkv) {  // the thread's first head is its lowest; v heads are not rotated
    const TT* cr = cosb + pos * D + d;
    const TT* sr = sinb + pos * D + d;
    c0.load(cr);
    s0.load(sr);
    c1.load(cr + D / 2);
    s1.load(sr + D / 2);
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int hh = hh0 + k * hpb;
    uint32_t a0[4] = {x0[k].x, x0[k].y, x0[k].z, x0[k].w};
    uint32_t a1[4] = {x1[k].x, x1[k].y, x1[k].z, x1[k].w};
    if (hh < H + Hkv) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float o0[2], o1[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float f0 = j ? P::hi(a0[i]) : P::lo(a0[i]), f1 = j ? P::hi(a1[i]) : P::lo(a1[i]);
          const int e = 2 * i + j;
          o0[j] = rot<EXACT, true>(f0, c0.at(e), f1, s0.at(e));
          o1[j] = rot<EXACT, false>(f1, c1.at(e), f0, s1.at(e));
        }
        a0[i] = P::pack(o0[0], o0[1]);  // the values that the 16-bit cache would hold
        a1[i] = P::pack(o1[0], o1[1]);
      }
      if (hh < H) {
        T* dst = qdst + (int64_t)k * hpb * seq * D;
        *reinterpret_cast<uint4*>(dst) = make_uint4(a0[0], a0[1], a0[2], a0[3]);
        *reinterpret_cast<uint4*>(dst + D / 2) = make_uint4(a1[0], a1[1], a1[2], a1[3]);
      }
    }
    if (!__any_sync(0xffffffffu, hh >= H && hh < all)) continue;
    // min and max of both groups, group 0 in the low half of the words
    const uint32_t m0 = P::min(P::min(a0[0], a0[1]), P::min(a0[2], a0[3]));
    const uint32_t m1 = P::min(P::min(a1[0], a1[1]), P::min(a1[2], a1[3]));
    const uint32_t M0 = P::max(P::max(a0[0], a0[1]), P::max(a0[2], a0[3]));
    const uint32_t M1 = P::max(P::max(a1[0], a1[1]), P::max(a1[2], a1[3]));
    uint32_t mn = P::min(__byte_perm(m0, m1, 0x5410), __byte_perm(m0, m1, 0x7632));
    uint32_t mx = P::max(__byte_perm(M0, M1, 0x5410), __byte_perm(M0, M1, 0x7632));
#pragma unroll
    for (int o = 1; o < C; o <<= 1) {
      mn = P::min(mn, __shfl_xor_sync(0xffffffffu, mn, o));
      mx = P::max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    }
    if (hh < H || hh >= all) continue;
    const float lo0 = P::lo(mn), lo1 = P::hi(mn);
    __align__(8) T sc[4];
    float i0, i1;
    group_numbers<T>(lo0, P::lo(mx), sc[0], i0);
    group_numbers<T>(lo1, P::hi(mx), sc[2], i1);
    const bool bad0 = sc[0] != sc[0], bad1 = sc[2] != sc[2];
    sc[1] = bad0 ? sc[0] : Num<T>::from_f(lo0);
    sc[3] = bad1 ? sc[2] : Num<T>::from_f(lo1);
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t byte[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t f0 = a0[2 * i + j / 2], f1 = a1[2 * i + j / 2];
        // the low bits of b1 * 16 + b0: the constant's share of them is 0
        byte[j] = code_bits(j & 1 ? P::hi(f1) : P::lo(f1), lo1, i1) * 16u +
                  code_bits(j & 1 ? P::hi(f0) : P::lo(f0), lo0, i0);
      }
      w[i] = __byte_perm(__byte_perm(byte[0], byte[1], 0x0040), __byte_perm(byte[2], byte[3], 0x0040),
                         0x5410);
      // fminf took a NaN for 15: a group without a scale has codes 0
      if (bad0) w[i] &= 0xF0F0F0F0u;
      if (bad1) w[i] &= 0x0F0F0F0Fu;
    }
    const bool key = hh < H + Hkv;
    const int64_t row = row0 + pos + (int64_t)(hh - H - (key ? 0 : Hkv)) * head_rows;
    *reinterpret_cast<uint2*>((key ? kcodes : vcodes) + row * (D / 2) + d) = make_uint2(w[0], w[1]);
    if (c == 0)
      *reinterpret_cast<uint2*>((key ? kscales : vscales) + row * 8) =
          *reinterpret_cast<const uint2*>(sc);
  }
}

// K and V of (b, head, positions[b, s]) as T: thread = 8 code bytes of one row,
// of K and of V; rows run along s, so both sides are contiguous where the
// positions are.
template <typename T, int D>
__global__ void __launch_bounds__(THREADS) kv4_read_kernel(
    const uint8_t* __restrict__ kcodes, const uint8_t* __restrict__ kscales,
    const uint8_t* __restrict__ vcodes, const uint8_t* __restrict__ vscales,
    const int64_t* __restrict__ positions, T* __restrict__ k_out, T* __restrict__ v_out,
    int64_t seq, lpc::Kv4Rows rows) {
  constexpr int C = D / 16;
  lpc::pdl_trigger();
  lpc::pdl_wait();
  const int64_t s = (int64_t)blockIdx.x * (THREADS / C) + threadIdx.x / C;
  if (s >= seq) return;
  const int c = threadIdx.x % C;
  const int h = blockIdx.y;
  const int64_t b = blockIdx.z;
  const int64_t pos = lpc::ld_dep(positions + b * seq + s);
  int64_t row0, head_rows, cap;
  const bool inside = rows.locate(b, &row0, &head_rows, &cap);
  const int64_t o = ((b * rows.kv_heads + h) * seq + s) * D + c * 8;
  if (pos < 0 || !inside || pos >= cap) {
    if (pos >= 0) atomicOr(&g_kv4_append_status, LPC_DEV_ERR_BOUNDS);
    const uint4 z = make_uint4(0u, 0u, 0u, 0u);
    *reinterpret_cast<uint4*>(k_out + o) = z;
    *reinterpret_cast<uint4*>(k_out + o + D / 2) = z;
    *reinterpret_cast<uint4*>(v_out + o) = z;
    *reinterpret_cast<uint4*>(v_out + o + D / 2) = z;
    return;
  }
  const int64_t row = row0 + (int64_t)h * head_rows + pos;
  const uint2 cw[2] = {lpc::ld_dep8(kcodes + row * (D / 2) + c * 8),
                       lpc::ld_dep8(vcodes + row * (D / 2) + c * 8)};
  const uint2 sw[2] = {lpc::ld_dep8(kscales + row * 8),
                       lpc::ld_dep8(vscales + row * 8)};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const T* sm = reinterpret_cast<const T*>(&sw[i]);
    const float s0 = Num<T>::to_f(sm[0]), m0 = Num<T>::to_f(sm[1]);
    const float s1 = Num<T>::to_f(sm[2]), m1 = Num<T>::to_f(sm[3]);
    float lo[8], hi[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t byte = (j < 4 ? cw[i].x : cw[i].y) >> (8 * (j & 3));
      lo[j] = fmaf((float)(byte & 15u), s0, m0);
      hi[j] = fmaf((float)((byte >> 4) & 15u), s1, m1);
    }
    T* dst = (i ? v_out : k_out) + o;
    *reinterpret_cast<uint4*>(dst) = pack8<T>(lo);
    *reinterpret_cast<uint4*>(dst + D / 2) = pack8<T>(hi);
  }
}

struct Launch {
  cudaLaunchAttribute attr[1];
  cudaLaunchConfig_t cfg = {};
  Launch(dim3 grid, int threads, cudaStream_t s) {
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = lpc::use_pdl() ? 1 : 0;
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
  }
};

template <typename T, typename TT, int D>
int append(const lpc_kv4* kv, const void* qkv, const int64_t* pos, const void* cosb,
           const void* sinb, int64_t table_rows, void* q_out, int64_t batch, int64_t seq, int H,
           cudaStream_t s) {
  constexpr int C = D / 16;
  const int all = H + 2 * kv->kv_heads;
  // two heads a thread, one where that would leave SMs without a CTA; CTAs of equal
  // size (whole warps), no thread without a head but in the last one
  const int chunks = all * C;
  const int K = chunks > THREADS && batch * seq * ((chunks + 2 * THREADS - 1) / (2 * THREADS)) >=
                                        2 * lpc::current_device_sms() ? 2 : 1;
  const int ctas = (chunks + K * THREADS - 1) / (K * THREADS);
  const int threads = std::min(THREADS, ((chunks + K * ctas - 1) / (K * ctas) + 31) / 32 * 32);
  Launch l(dim3((unsigned)(batch * seq), (unsigned)((chunks + K * threads - 1) / (K * threads))),
           threads, s);
  const lpc::Kv4Rows rows = lpc::kv4_rows(kv);
#define LPC_APPEND(KK)                                                                          \
  cudaLaunchKernelEx(&l.cfg, kv4_append_kernel<T, TT, D, KK>, (const T*)qkv, pos,               \
                     (const TT*)cosb, (const TT*)sinb, table_rows, (T*)q_out,                   \
                     (uint8_t*)kv->key_codes, (uint8_t*)kv->key_scales,                         \
                     (uint8_t*)kv->value_codes, (uint8_t*)kv->value_scales, seq, H, rows)
  if (K == 1) LPC_APPEND(1); else LPC_APPEND(2);
#undef LPC_APPEND
  return lpc::check_launch("rope_kv_append_int4");
}

template <typename T, int D>
int read(const lpc_kv4* kv, const int64_t* pos, void* k_out, void* v_out, int64_t batch,
         int64_t seq, cudaStream_t s) {
  constexpr int RPB = THREADS / (D / 16);
  Launch l(dim3((unsigned)((seq + RPB - 1) / RPB), (unsigned)kv->kv_heads, (unsigned)batch),
           THREADS, s);
  cudaLaunchKernelEx(&l.cfg, kv4_read_kernel<T, D>, (const uint8_t*)kv->key_codes,
                     (const uint8_t*)kv->key_scales, (const uint8_t*)kv->value_codes,
                     (const uint8_t*)kv->value_scales, pos, (T*)k_out, (T*)v_out, seq,
                     lpc::kv4_rows(kv));
  return lpc::check_launch("kv_read_int4");
}

}  // namespace

extern "C" int lpc_rope_kv_append_int4(const lpc_kv4* kv, const void* qkv,
                                       const int64_t* positions, const void* cos, const void* sin,
                                       int64_t table_rows, void* q_out, int64_t batch, int64_t seq,
                                       int num_heads, int table_dtype, void* stream) {
  using namespace lpc;
  int rc = kv4_check(kv, "rope_kv_append_int4");
  if (rc) return rc;
  if (batch < 0 || seq < 0 || num_heads <= 0 || num_heads > 65535 || table_rows <= 0 ||
      batch > 0x7fffffffLL || seq > 0x7fffffffLL || batch * seq > 0x7fffffffLL ||
      (kv->max_batch > 0 && batch > kv->max_batch)) {
    set_error("rope_kv_append_int4: invalid sizes (batch=%lld seq=%lld heads=%d max_batch=%lld)",
              (long long)batch, (long long)seq, num_heads, (long long)kv->max_batch);
    return LPC_ERR_INVALID;
  }
  if (batch == 0 || seq == 0) return LPC_OK;
  if (!qkv || !positions || !cos || !sin || !q_out || !aligned16(qkv) || !aligned16(cos) ||
      !aligned16(sin) || !aligned16(q_out)) {
    set_error("rope_kv_append_int4: tensors must be given and 16-byte aligned");
    return LPC_ERR_INVALID;
  }
  if (table_dtype != kv->dtype && table_dtype != LPC_DTYPE_F32) {
    set_error("rope_kv_append_int4: table dtype must match activations or be fp32");
    return LPC_ERR_UNSUPPORTED;
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool wide = table_dtype == LPC_DTYPE_F32;
#define LPC_A(T, DD)                                                                              \
  return wide ? append<T, float, DD>(kv, qkv, positions, cos, sin, table_rows, q_out, batch, seq, \
                                     num_heads, s)                                                \
              : append<T, T, DD>(kv, qkv, positions, cos, sin, table_rows, q_out, batch, seq,     \
                                 num_heads, s)
  if (kv->dtype == LPC_DTYPE_BF16) {
    if (kv->head_dim == 128) LPC_A(__nv_bfloat16, 128);
    if (kv->head_dim == 64) LPC_A(__nv_bfloat16, 64);
    LPC_A(__nv_bfloat16, 32);
  }
  if (kv->head_dim == 128) LPC_A(__half, 128);
  if (kv->head_dim == 64) LPC_A(__half, 64);
  LPC_A(__half, 32);
#undef LPC_A
}

extern "C" int lpc_kv_read_int4(const lpc_kv4* kv, const int64_t* positions, void* k_out,
                                void* v_out, int64_t batch, int64_t seq, void* stream) {
  using namespace lpc;
  int rc = kv4_check(kv, "kv_read_int4");
  if (rc) return rc;
  if (batch < 0 || batch > 65535 || seq < 0 || seq > 0x7fffffffLL ||
      (kv->max_batch > 0 && batch > kv->max_batch)) {
    set_error("kv_read_int4: invalid sizes (batch=%lld seq=%lld max_batch=%lld)", (long long)batch,
              (long long)seq, (long long)kv->max_batch);
    return LPC_ERR_INVALID;
  }
  if (batch == 0 || seq == 0) return LPC_OK;
  if (!positions || !k_out || !v_out || !aligned16(k_out) || !aligned16(v_out)) {
    set_error("kv_read_int4: tensors must be given and 16-byte aligned");
    return LPC_ERR_INVALID;
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
#define LPC_R(T, DD) return read<T, DD>(kv, positions, k_out, v_out, batch, seq, s)
  if (kv->dtype == LPC_DTYPE_BF16) {
    if (kv->head_dim == 128) LPC_R(__nv_bfloat16, 128);
    if (kv->head_dim == 64) LPC_R(__nv_bfloat16, 64);
    LPC_R(__nv_bfloat16, 32);
  }
  if (kv->head_dim == 128) LPC_R(__half, 128);
  if (kv->head_dim == 64) LPC_R(__half, 64);
  LPC_R(__half, 32);
#undef LPC_R
}
