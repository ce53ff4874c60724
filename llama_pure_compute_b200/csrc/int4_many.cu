// Products with 4-bit weights, up to 64 tokens, where int4_linear.cu's pick() finds
// neither of its own kernels cheaper: tcgen05, weights as the M operand.
//
// mma.sync needs one instruction for 16 rows x 8 tokens x 16 columns: from 16
// tokens on its issue rate, not HBM, is the limit (32 tokens, 22,016 x 4096: 41
// us).  Here a CTA takes 128 weight rows and all tokens; 64 columns at a time
//   * a warpgroup turns codes into fp16 weights in registers, a thread its own
//     row (one logic instruction makes two codes the halves 1024 + c, or 64 + c from
//     the upper nibbles; a packed subtraction leaves c, and the packed FMA with
//     (s 2^e, m 2^e) gives (s c + m) 2^e with one rounding), and stores them to tensor
//     memory: the A operand never touches shared memory, whose bandwidth a 16 KB tile
//     per 4 KB of codes would exceed.  Without the subtraction, codes as the subnormals
//     c * 2^-24, it was 2 to 6% faster, but s had to carry the 2^24, which left the
//     weights the lowest of fp16's exponents: groups 2^-8 of their row's largest lost bits;
//   * x, fp16 (bf16 rows are converted first, scaled by a power of two each, by a
//     small kernel), comes by TMA as the B operand;
//   * one thread issues tcgen05.mma with the fp32 sums in tensor memory.
// A step is a chain of waits and dependent instructions of over 800 cycles (without the
// subtraction 810: unpacking 310, the wait for the tile 175, the store 110), far more than
// its share of HBM's time (175), so the CTAs are small, four an SM, and their chains
// overlap: about 350 a step. The tensor pipe takes 256 of them, 64 a product whatever the
// tokens.
// Measured, bf16, groups of 128: 22,016 x 4096 at 16 / 32 / 64 tokens 21.3 / 22.9 / 24.7
// us (stream 7.5), 4096 x 4096 at 64 14.6, 128,256 x 4096 at 32 86.8 (44).  Two
// warpgroups a CTA and clusters of 16 were slower.
// A weight is rounded to fp16: off by at most 2^-11 of itself, or 2^-39 of its row's
// largest |m| + 15 |s| where that is more.  The roundings are independent.  Measured,
// normal x and w, k = 4096, relative: with bf16 numbers 2.2e-5, which the outputs (1.7e-3)
// do not show; with fp16 numbers 2.0e-4, beside the outputs' own 2.1e-4 2.9e-4 in all
// (SwiGLU, two products, 3.5e-4), as a 16-bit copy of the weight would give.  e is a power
// per weight row (int4.cuh), undone with x's in the epilogue.
// Few row tiles: clusters of up to 8 CTAs split the columns and add their sums
// through distributed shared memory, in rank order.
#include <algorithm>
#include <atomic>

#include "int4.cuh"

LPC_DECLARE_STATUS(g_int4_status)

unsigned int lpc_status_int4(bool clear) {
  unsigned int v = 0;
  cudaMemcpyFromSymbol(&v, g_int4_status, sizeof(v));
  if (clear && v) {
    unsigned int z = 0;
    cudaMemcpyToSymbol(g_int4_status, &z, sizeof(z));
  }
  return v;
}

namespace {

using lpc::Num;
using lpc::cp16;
using lpc::cp_commit;
using lpc::cp_wait;

constexpr int THREADS = 192;   // 4 converter warps, MMA issuer, x loader
constexpr int CST = 4;         // code stages
constexpr int XST = 4;         // x stages; loops over steps are unrolled by 4, so that
                               // slots and the phases of A's two tiles are constants
constexpr int CODES = 4096;    // code bytes of a 128 x 64 tile
constexpr int MAX_TOKENS = 64;
constexpr uint32_t TMEM_COLS = 128;  // 64 sums + 2 tiles of 32; four CTAs share an SM's 512
constexpr uint32_t A_COL = 64;

// A CTA that waits for tensor memory while its cluster waits for it, beside one of
// another stream's clusters that waits the other way round, would wait for ever.  So
// shared memory is asked for such that whatever shares an SM also shares its 512
// columns: four of these CTAs and not five, two beside a wsgemm CTA of 256 columns
// (which asks for 90 KB), none beside a CTA pair of the SwiGLU kernel (182 KB, 512
// columns) or two such wsgemm CTAs.
constexpr int SM_SMEM = 228 * 1024;  // of an SM; a CTA takes 1 KB more than it asks for
constexpr int MIN_SMEM = 52 * 1024;
static_assert(5 * (MIN_SMEM + 1024) > SM_SMEM && 91 * 1024 + 3 * (MIN_SMEM + 1024) > SM_SMEM &&
                  2 * 91 * 1024 + MIN_SMEM + 1024 > SM_SMEM &&
                  182 * 1024 + MIN_SMEM + 1024 > SM_SMEM, "tensor memory");

enum { EPI_STORE = 0, EPI_RESIDUAL = 1, EPI_SWIGLU = 2 };

__device__ __forceinline__ void cp4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void ld_cluster4(uint32_t addr, float (&v)[4]) {
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3])
               : "r"(addr)
               : "memory");
}
// s c + m of two codes: with `one` in its upper bits a code is the half base + c, exactly.
__device__ __forceinline__ uint32_t weights(uint32_t w, uint32_t mask, uint32_t one, __half2 base,
                                            __half2 s, __half2 m) {
  const uint32_t a = (w & mask) | one;
  const __half2 v = __hfma2(__hsub2(*reinterpret_cast<const __half2*>(&a), base), s, m);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// lpc::mbar_wait with a hint to sleep on the barrier: four CTAs' waits would
// otherwise poll away a third of the SM's issue slots.
__device__ __forceinline__ bool try_wait(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 20000;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0u;
}
__device__ __noinline__ bool wait_on(uint32_t bar, uint32_t parity) {
  const uint64_t t0 = lpc::global_timer_ns();
  for (;;) {
    if (try_wait(bar, parity)) return true;
    if (lpc::global_timer_ns() - t0 > LPC_WAIT_LIMIT_NS) {
      atomicOr(&g_int4_status, LPC_DEV_ERR_TIMEOUT);
      return false;
    }
  }
}
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity) {
  return try_wait(bar, parity) || wait_on(bar, parity);
}

struct Args {
  const uint8_t* codes;
  const uint8_t* scaled;
  const float* factors;
  const float* x_factors;  // 2^-e of each token, or null
  const void* resid;
  void* out;
  int64_t n_out;
  int tokens, kb, epi, splits;
  uint32_t idesc;
};

// N: tokens the products are computed for (16, 32 or 64; rows of x past the last
// are zeros).  SG: groups in 64 columns (2 for groups of 32, else 1).
template <typename T, int N, int SG>
__global__ void __launch_bounds__(THREADS, 4)
    int4_many_kernel(const __grid_constant__ lpc::TmaDesc tm_x, const Args p, int group_shift) {
  constexpr int CSTAGE = CODES + SG * 512;
  constexpr int XSTAGE = N * 128;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = lpc::smem_u32(smem_raw);
  const uint32_t xring = (raw + 1023u) & ~1023u;
  const uint32_t cring = xring + XST * XSTAGE;
  const uint32_t bars = cring + CST * CSTAGE;
  auto a_full = [&](int i) { return bars + 8u * i; };
  auto a_empty = [&](int i) { return bars + 16u + 8u * i; };
  auto x_full = [&](int i) { return bars + 32u + 8u * i; };
  auto x_empty = [&](int i) { return bars + 32u + 8u * (XST + i); };
  const uint32_t done = bars + 32u + 16u * XST;
  const uint32_t tmem_slot = done + 8u;
  float* xf = reinterpret_cast<float*>(smem_raw + (tmem_slot + 8u - raw));  // [N], the tokens' 2^-e

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tile = (int)blockIdx.x / p.splits, rank = (int)blockIdx.x - tile * p.splits;
  const int kb0 = (int)((int64_t)rank * p.kb / p.splits);
  const int nk = (int)((int64_t)(rank + 1) * p.kb / p.splits) - kb0;

  const int row = threadIdx.x & 127;  // converters: row of the tile
  // the code stream: a warp copies the two tile rows of its own 32 weight rows, 16
  // bytes of each a lane (places mixed so that a thread's row reads without bank
  // conflicts), and a thread its own row's numbers
  const int64_t ng = ((int64_t)p.kb * 64) >> group_shift;
  const int cr = lane >> 2, ct = lane & 3;
  const uint8_t* csrc = p.codes + ((int64_t)(tile * 8 + (row >> 5) * 2) * p.kb + kb0) * 512 + lane * 16;
  const int64_t cnext = (int64_t)p.kb * 512;  // the next tile row
  const uint32_t cdst = cring + (row >> 5) * 1024 + cr * 64 + ((ct ^ (cr >> 1)) & 3) * 16;
  const uint8_t* nsrc = p.scaled + (int64_t)(tile * 8 + (row >> 4)) * ng * 64 + (row & 15) * 4;
  auto fetch = [&](int step, int slot) {
    if (step < nk) {
      const uint8_t* src = csrc + (uint32_t)step * 512u;
      cp16(cdst + slot * CSTAGE, src);
      cp16(cdst + slot * CSTAGE + 512, src + cnext);
      const uint32_t g = (uint32_t)(kb0 + step) * 64u >> group_shift;
#pragma unroll
      for (int i = 0; i < SG; ++i)
        cp4(cring + slot * CSTAGE + CODES + i * 512 + row * 4, nsrc + (g + i) * 64u);
    }
    cp_commit();
  };

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      lpc::mbar_init(a_full(i), 4);
      lpc::mbar_init(a_empty(i), 1);
    }
    for (int i = 0; i < XST; ++i) {
      lpc::mbar_init(x_full(i), 1);
      lpc::mbar_init(x_empty(i), 1);
    }
    lpc::mbar_init(done, 1);
    lpc::fence_mbar_init();
  }
  // the weights belong to no earlier kernel of the stream
  if (warp < 4)
    for (int i = 0; i < CST - 1; ++i) fetch(i, i);
  if (warp == 4) {
    lpc::tmem_alloc(tmem_slot, TMEM_COLS);
    lpc::tmem_relinquish();
  }
  lpc::tc_fence_before();
  __syncthreads();
  lpc::tc_fence_after();
  lpc::pdl_trigger();  // after the allocation: a dependent never holds what this grid waits for
  lpc::pdl_wait();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem_raw + (tmem_slot - raw));
  const float factor = warp < 4 ? __ldg(p.factors + (int64_t)tile * 128 + row) : 0.f;

  if (warp < 4) {
    const uint32_t a_tmem = tmem + ((uint32_t)(warp * 32) << 16) + A_COL;
    // rows 8..15 of a tile row are the nibbles beside: as low bits of 64 + c, not of 1024 + c
    const uint32_t mask = (row & 8) ? 0x00F000F0u : 0x000F000Fu;
    const uint32_t one = (row & 8) ? 0x54005400u : 0x64006400u;
    const __half2 base = *reinterpret_cast<const __half2*>(&one);
    const int r = row & 7;
    const uint8_t* src = smem_raw + (cring - raw) + (row >> 4) * 512 + r * 64;
    const uint8_t* num = smem_raw + (cring - raw) + CODES + row * 4;
    uint32_t places[4];  // of the row's four pieces
#pragma unroll
    for (int t = 0; t < 4; ++t) places[t] = ((t ^ (r >> 1)) & 3) * 16;
    bool ok = true;
    for (int first = 0; first < nk; first += CST) {
#pragma unroll
      for (int u = 0; u < CST; ++u) {  // step first + u is in slot u
        if (first + u >= nk) break;
        cp_wait<CST - 2>();
        __syncwarp();  // the warp's copies have arrived, and the slot before is free
        fetch(first + u + CST - 1, (u + CST - 1) % CST);
        __half2 sc[SG], mn[SG];
#pragma unroll
        for (int i = 0; i < SG; ++i) {
          const __half2 v = *reinterpret_cast<const __half2*>(num + u * CSTAGE + i * 512);
          sc[i] = __low2half2(v);
          mn[i] = __high2half2(v);
        }
        uint32_t v[2][16];  // 32 columns each, as pairs
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const uint4 c = *reinterpret_cast<const uint4*>(src + places[t] + u * CSTAGE);
          const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {  // columns 32 (j / 2) + 8 t + 4 (j % 2) + 0..3
            const int h = j >> 1, at = 4 * t + 2 * (j & 1), g = SG == 2 ? h : 0;
            v[h][at] = weights(w[j], mask, one, base, sc[g], mn[g]);
            v[h][at + 1] = weights(w[j] >> 8, mask, one, base, sc[g], mn[g]);
          }
        }
        // the tile's last products must be done (a warp goes on as one)
        constexpr int PAIR = 2;  // tiles of A
        const int a = u % PAIR;
        if (ok) ok = __all_sync(0xffffffffu, wait(a_empty(a), (u / PAIR % 2) ^ 1u));
        if (ok) {
          lpc::tc_fence_after();
          lpc::tmem_st16(a_tmem + 32u * a, v[0]);
          lpc::tmem_st16(a_tmem + 32u * a + 16u, v[1]);
          lpc::tmem_wait_st();
          lpc::tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) lpc::mbar_arrive(a_full(a));
      }
    }
    cp_wait<0>();
  } else if (warp == 4) {
    if (lane == 0) {
      const uint64_t bd0 = lpc::smem_desc_sw128(xring, 16, 1024);
      bool ok = true;
      for (int first = 0; first < nk && ok; first += XST) {
        const uint32_t turn = (uint32_t)(first / XST) & 1u;
#pragma unroll
        for (int u = 0; u < XST; ++u) {
          if (first + u >= nk) break;
          const int a = u & 1;
          ok = wait(x_full(u), turn) && wait(a_full(a), (u >> 1) & 1u);
          if (!ok) break;
          lpc::tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)  // 16 columns: 8 TMEM columns of A, 32 bytes of B
            lpc::umma_ts(tmem, tmem + A_COL + 32u * a + 8u * kk, bd0 + (uint32_t)(u * (XSTAGE >> 4)) + 2u * kk,
                         p.idesc, (first | u | kk) != 0);
          lpc::umma_commit(a_empty(a));
          lpc::umma_commit(x_empty(u));
        }
      }
      lpc::umma_commit(done);
    }
    __syncwarp();
  } else {
    for (int i = lane; i < N; i += 32)
      xf[i] = p.x_factors && i < p.tokens
                  ? __int_as_float(lpc::ld_dep(reinterpret_cast<const int32_t*>(p.x_factors) + i)) : 1.f;
    if (lane == 0) {
      int step = 0;
      for (; step < nk; ++step) {
        const int xs = step % XST;
        if (!wait(x_empty(xs), ((uint32_t)(step / XST) & 1u) ^ 1u)) break;
        lpc::mbar_arrive_expect_tx(x_full(xs), XSTAGE);
        lpc::tma_load_2d(xring + xs * XSTAGE, &tm_x, (kb0 + step) * 64, 0, x_full(xs));
      }
      // the last loads have landed before this CTA's shared memory is let go, even
      // where the products gave up on them
      for (int i = max(0, step - XST); i < step; ++i)
        if (!wait(x_full(i % XST), (uint32_t)(i / XST) & 1u)) break;
    }
    __syncwarp();
  }
  __syncthreads();  // xf is written

  // sums: thread = weight row, 16 tokens at a time
  T* out = static_cast<T*>(p.out);
  const T* resid = static_cast<const T*>(p.resid);
  const bool swiglu = p.epi == EPI_SWIGLU;
  const int64_t col = swiglu ? (int64_t)tile * 64 + (row >> 5) * 16 + (lane & 15)
                             : (int64_t)tile * 128 + row;
  const bool writes = col < p.n_out && !(swiglu && lane >= 16);
  // out may be resid: what a batch of outputs adds is read before any of it is written
  auto before = [&](int tk) {
    return p.epi == EPI_RESIDUAL && writes && tk < p.tokens
               ? Num<T>::to_f(resid[(int64_t)tk * p.n_out + col]) : 0.f;
  };
  // whole warps: the SwiGLU partner row is 16 lanes away
  auto emit = [&](int tk, float v, float plus) {
    v *= factor * xf[tk];
    if (swiglu) {
      const float up = __shfl_xor_sync(0xffffffffu, v, 16);
      v = __fdividef(v, 1.f + __expf(-v)) * up;
    }
    if (writes && tk < p.tokens) out[(int64_t)tk * p.n_out + col] = Num<T>::from_f(v + plus);
  };
  float* red = reinterpret_cast<float*>(smem_raw + (xring - raw));  // [token][row], the x ring is idle
  if (warp < 4) {
    const bool ok = __all_sync(0xffffffffu, wait(done, 0u));
    lpc::tc_fence_after();
#pragma unroll 1
    for (int c = 0; c < N; c += 16) {
      float plus[16];
      if (p.splits == 1)
#pragma unroll
        for (int i = 0; i < 16; ++i) plus[i] = before(c + i);
      uint32_t acc[16];
      lpc::tmem_ld16(tmem + ((uint32_t)(warp * 32) << 16) + c, acc);
      lpc::tmem_wait_ld();
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float v = ok ? __uint_as_float(acc[i]) : 0.f;
        if (p.splits == 1) emit(c + i, v, plus[i]);
        else red[(c + i) * 128 + row] = v;
      }
    }
  }
  if (p.splits > 1) {
    lpc::cluster_sync();
    // a warp adds up a token's 128 rows, a lane 4 of them; this CTA has `each` tokens
    const int each = (N + p.splits - 1) / p.splits;
    if (warp < 4) {
      const float4 f4 = __ldg(reinterpret_cast<const float4*>(p.factors + (int64_t)tile * 128) + lane);
      const float f[4] = {f4.x, f4.y, f4.z, f4.w};
      // SwiGLU: rows 4 lane .. of gate, 16 rows (4 lanes) on of up
      const int64_t n0 = swiglu ? (int64_t)tile * 64 + (lane >> 3) * 16 + (lane & 3) * 4
                                : (int64_t)tile * 128 + lane * 4;
      const bool mine = !(swiglu && (lane & 4));
#pragma unroll 1
      for (int c = warp; c < each; c += 4) {
        const int tk = rank * each + c;
        if (tk >= p.tokens) break;
        const uint32_t at = xring + (uint32_t)(tk * 128 + lane * 4) * 4;
        float part[8][4], v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < 8; ++s)
          if (s < p.splits) ld_cluster4(lpc::mapa_shared(at, s), part[s]);
#pragma unroll
        for (int s = 0; s < 8; ++s)
          if (s < p.splits)
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] += part[s][i];
        T* o = out + (int64_t)tk * p.n_out + n0;
        const T* add = resid + (int64_t)tk * p.n_out + n0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[i] *= f[i] * xf[tk];
          if (swiglu) {
            const float up = __shfl_xor_sync(0xffffffffu, v[i], 4);
            v[i] = __fdividef(v[i], 1.f + __expf(-v[i])) * up;
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (mine && n0 + i < p.n_out && p.epi == EPI_RESIDUAL) v[i] += Num<T>::to_f(add[i]);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (mine && n0 + i < p.n_out) o[i] = Num<T>::from_f(v[i]);
      }
    }
    lpc::cluster_sync();  // no CTA leaves while its sums are read
  }
  lpc::tc_fence_before();
  __syncthreads();
  if (warp == 4) {
    lpc::tc_fence_after();
    lpc::tmem_dealloc(tmem, TMEM_COLS);
  }
}

// x [tokens, k] in bf16 as fp16, each token scaled by a power of two that brings
// its largest value to about 2^14 (what that loses lies 2^-38 below that value).  A
// CTA has a token; a thread holds its first KEEP pieces of 8 values between the search
// and the conversion, so that all loads are in flight at once.
constexpr int XT = 512, KEEP = 4;
__global__ void __launch_bounds__(XT)
    int4_x_kernel(const __nv_bfloat16* x, uint4* xh, float* factors, int k) {
  lpc::pdl_trigger();
  lpc::pdl_wait();
  const int pieces = k / 8;
  const uint4* src = reinterpret_cast<const uint4*>(x) + (int64_t)blockIdx.x * pieces;
  uint4* dst = xh + (int64_t)blockIdx.x * pieces;
  __shared__ uint32_t most[XT / 32];
  uint4 held[KEEP];
#pragma unroll
  for (int j = 0; j < KEEP; ++j) {
    const int i = threadIdx.x + j * XT;
    held[j] = i < pieces ? lpc::ld_dep16(src + i) : make_uint4(0u, 0u, 0u, 0u);
  }
  // magnitudes of bf16 order as their bits do, two at a time; a NaN is the largest
  auto largest = [](uint32_t a, const uint4& u) {
    constexpr uint32_t M = 0x7FFF7FFFu;
    return __vimax3_u16x2(__vimax3_u16x2(a, u.x & M, u.y & M), u.z & M, u.w & M);
  };
  uint32_t a = 0u;
#pragma unroll
  for (int j = 0; j < KEEP; ++j) a = largest(a, held[j]);
  for (int i = threadIdx.x + KEEP * XT; i < pieces; i += XT) a = largest(a, lpc::ld_dep16(src + i));
  a = __reduce_max_sync(0xffffffffu, max(a & 0xFFFFu, a >> 16));
  if ((threadIdx.x & 31) == 0) most[threadIdx.x >> 5] = a;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < XT / 32; ++i) a = max(a, most[i]);
  int e = 0;
  if (a > 0u && a < 0x7F80u) e = min(126, 14 - ((int)(a >> 7) - 127));
  const float up = __uint_as_float((uint32_t)(127 + e) << 23);
  if (threadIdx.x == 0) factors[blockIdx.x] = __uint_as_float((uint32_t)(127 - e) << 23);
  auto scaled = [&](const uint4& u) {
    uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __half2 h = __floats2half2_rn(lpc::bf16lo(w[j]) * up, lpc::bf16hi(w[j]) * up);
      w[j] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  };
#pragma unroll
  for (int j = 0; j < KEEP; ++j) {
    const int i = threadIdx.x + j * XT;
    if (i < pieces) dst[i] = scaled(held[j]);
  }
  for (int i = threadIdx.x + KEEP * XT; i < pieces; i += XT) dst[i] = scaled(lpc::ld_dep16(src + i));
}

constexpr int SPLITS = 8;  // a portable cluster

// CTAs per row tile: the least time of the busiest SM, a CTA costing its 64-column
// steps and about 6 more.  `clusters[s]` clusters of s CTAs run at once, which is
// fewer than the SMs' room divided by s: 12,288 x 4096 at 32 tokens (96 tiles) 16.3 us
// in clusters of 5, 21.3 in clusters of 6.
int pick_splits(int tiles, int kb, const std::atomic<int>* clusters) {
  int best = 1;
  int64_t cost = INT64_MAX;
  for (int s = 1; s <= SPLITS && s <= kb; ++s) {
    const int64_t room = clusters[s].load(std::memory_order_relaxed);
    const int64_t c = (tiles + room - 1) / room * ((kb + s - 1) / s + 6);
    if (c < cost) {
      cost = c;
      best = s;
    }
  }
  return best;
}

template <typename T, int N, int SG>
int launch(const lpc::TmaDesc& tm, Args a, int tiles, int group_shift, cudaStream_t s) {
  constexpr int USED = 1024 + XST * N * 128 + CST * (CODES + SG * 512) + 512;
  constexpr int SMEM = USED > MIN_SMEM ? USED : MIN_SMEM;
  static_assert(4 * (SMEM + 1024) <= SM_SMEM, "four CTAs an SM");
  static std::atomic<uint64_t> mask{0};
  int rc = lpc::once_per_device_smem((const void*)int4_many_kernel<T, N, SG>, SMEM, mask);
  if (rc) return rc;
  cudaLaunchAttribute attr[2];
  static std::atomic<int> clusters[SPLITS + 1];  // that run at once, by their size; 0: not asked yet
  if (clusters[SPLITS].load(std::memory_order_acquire) == 0) {
    const int sms = lpc::current_device_sms();
    int each = 1;  // CTAs an SM that the answers count with: 4 run
    for (int n = 1; n <= SPLITS; ++n) {
      cudaLaunchConfig_t q = {};
      q.gridDim = dim3((unsigned)n);
      q.blockDim = dim3(THREADS);
      q.dynamicSmemBytes = SMEM;
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = (unsigned)n;
      attr[0].val.clusterDim.y = 1;
      attr[0].val.clusterDim.z = 1;
      q.attrs = attr;
      q.numAttrs = 1;
      int count = 0;
      if (cudaOccupancyMaxActiveClusters(&count, int4_many_kernel<T, N, SG>, &q) != cudaSuccess || count <= 0) {
        cudaGetLastError();
        count = each * sms / n;
      }
      if (n == 1) each = std::max(1, std::min(4, count / sms));
      clusters[n].store(std::max(1, count * 4 / each), std::memory_order_release);
    }
  }
  a.splits = pick_splits(tiles, a.kb, clusters);
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = lpc::use_pdl() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)a.splits;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * a.splits));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = SMEM;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = a.splits > 1 ? 2 : 1;
  cudaLaunchKernelEx(&cfg, int4_many_kernel<T, N, SG>, tm, a, group_shift);
  return lpc::check_launch("int4_linear");
}

template <typename T>
int launch_n(const lpc::TmaDesc& tm, const Args& a, int n, int tiles, int group_shift,
             cudaStream_t s) {
  const bool two = group_shift == 5;
  if (n == 16) return two ? launch<T, 16, 2>(tm, a, tiles, group_shift, s) : launch<T, 16, 1>(tm, a, tiles, group_shift, s);
  if (n == 32) return two ? launch<T, 32, 2>(tm, a, tiles, group_shift, s) : launch<T, 32, 1>(tm, a, tiles, group_shift, s);
  return two ? launch<T, 64, 2>(tm, a, tiles, group_shift, s) : launch<T, 64, 1>(tm, a, tiles, group_shift, s);
}

}  // namespace

namespace lpc {

int int4_many(const lpc_w4* w, const void* x, void* out, const void* resid, int64_t tokens,
              int epilogue, void* workspace, cudaStream_t s) {
  const Int4Parts parts = int4_parts(w->packed, w->n_out, w->k, w->group, w->layout);
  Args a = {};
  a.codes = parts.codes;
  a.scaled = parts.scaled;
  a.factors = parts.factors;
  a.resid = resid;
  a.out = out;
  a.n_out = w->n_out;
  a.tokens = (int)tokens;
  a.kb = w->k / 64;
  a.epi = epilogue;
  const void* xh = x;
  if (w->dtype == LPC_DTYPE_BF16) {
    // [64] factors, then the converted rows
    float* f = static_cast<float*>(workspace);
    xh = f + MAX_TOKENS;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = lpc::use_pdl() ? 1 : 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)tokens);
    cfg.blockDim = dim3(XT);
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, int4_x_kernel, (const __nv_bfloat16*)x, (uint4*)xh, f, (int)w->k);
    int rc = check_launch("int4_linear (x)");
    if (rc) return rc;
    a.x_factors = f;
  }
  const int n = tokens <= 16 ? 16 : tokens <= 32 ? 32 : 64;
  TmaDesc tm;
  int rc = make_tma_2d(&tm, xh, LPC_DTYPE_F16, (uint64_t)w->k, (uint64_t)tokens,
                       (uint64_t)w->k * 2, 64, (uint32_t)n, true);
  if (rc) return rc;
  const int64_t rows = (w->n_out + 15) / 16 * 16 * (w->layout == 1 ? 2 : 1);
  const int tiles = (int)((rows + 127) / 128);
  a.idesc = idesc_f16(0u, 128u, (uint32_t)n, 0u, 0u);
  const int shift = w->group == 128 ? 7 : w->group == 64 ? 6 : 5;
  return w->dtype == LPC_DTYPE_BF16 ? launch_n<__nv_bfloat16>(tm, a, n, tiles, shift, s)
                                    : launch_n<__half>(tm, a, n, tiles, shift, s);
}

}  // namespace lpc
