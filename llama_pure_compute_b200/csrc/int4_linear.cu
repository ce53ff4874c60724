// Decode-sized products with 4-bit weights and group scales:
//
//   y[t, n] = sum_g ( s[n, g] * sum_{k in g} x[t, k] c[n, k] + m[n, g] * sum_{k in g} x[t, k] ),
//
// epilogues: store, residual (+ resid), SwiGLU (silu(gate) * up).
//
// Bound: HBM, by the weight stream of k/2 + 4 k/group bytes a row, and behind it
// the instructions a code costs: HBM's rate leaves an SM's four schedulers about
// 1.3 instructions a 32-bit word of 8 codes and lane.  So codes are never
// converted.  mma.sync m16n8k16 takes 16 weight rows (A) by 8 tokens (B); a
// packed word holds exactly the lane's 8 codes of one product, in the order in
// which masks pick them, and a code in the low bits of a half is the subnormal
// c * 2^-24, exactly.  x enters as fp16 too.
//
// Three kernels; pick() chooses by the token count and what of x fits:
//   FEW   up to 8 tokens on larger weights, x in shared memory (int4_few_kernel, below);
//   MID   smaller weights, x from the caches (int4_mid_kernel);
//   MANY  the rest up to 64 tokens: tcgen05 (int4_many.cu), which wants whole
//         128-row tiles of converted weights, at few tokens more work than the
//         products themselves.
// Measured at groups of 128, bf16 (us; in brackets the stream at 6397 GB/s): one
// token, 128,256 x 4096 42.9 (43.7) and 4096 x 4096 3.8 (1.4: the launch, x and one
// round of loads); 22,016 x 4096 at 1 / 4 / 8 tokens 10.8 / 11.3 / 13.7 (7.5), 4096 x
// 11,008 at 4 8.6 (3.8).
//
// Packed weight: tiles of 16 rows x 64 columns, 512 contiguous bytes, 16 a
// lane, read with cp.async into the lane's own slots (no barrier), followed by
// the group numbers, 64 bytes per tile row and group.  The warps of a CTA share
// a tile row's k range and add their partial sums through shared memory; CTAs
// walk over the tile rows, and the weight stream runs on across them.
#include <algorithm>
#include <atomic>

#include "int4.cuh"

LPC_DECLARE_STATUS(g_int4_few_status)

unsigned int lpc_status_int4_few(bool clear) {
  unsigned int v = 0;
  cudaMemcpyFromSymbol(&v, g_int4_few_status, sizeof(v));
  if (clear && v) {
    unsigned int z = 0;
    cudaMemcpyToSymbol(g_int4_few_status, &z, sizeof(z));
  }
  return v;
}

namespace {

using lpc::Num;
using lpc::cp16;
using lpc::cp8;
using lpc::cp_commit;
using lpc::cp_wait;

constexpr int MAX_TOKENS = 64;


__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                    uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The 8 codes of a word as the A operand, columns 2t.. and 2t + 8..: rows r + 8
// are the upper nibbles (16-fold), rows r whole bytes, c_r + 16 c_{r+8}, so that the
// lower nibbles need no mask of their own: the accumulator of row r + 8, which the
// same lane holds, is taken off that of row r once a group.  Four instructions a
// word; the accumulator loses 4 of its 24 bits, and what the tensor core cuts of it, always
// towards zero, leaves rows r off by some 2e-5 s sum(x).  x around zero does not show it;
// x of one sign does in fp16: 2.9e-4 off at k = 4096, 4.0e-4 at 11,008, 2.1e-4 of that the
// output's own rounding (codes two bits higher in their words changed nothing and cost
// 16% on 128,256 x 4096 at one token).  Code c is the subnormal c * 2^-24.
__device__ __forceinline__ void operand(uint32_t w, uint32_t (&a)[4]) {
  a[0] = w & 0x00FF00FFu;
  a[1] = w & 0x00F000F0u;
  a[2] = __byte_perm(w, 0u, 0x4341);
  a[3] = a[2] & 0x00F000F0u;
}

template <typename T>
__device__ __forceinline__ float2 pair_f(uint32_t w) {
  if constexpr (std::is_same<T, __half>::value)
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  else
    return make_float2(lpc::bf16lo(w), lpc::bf16hi(w));
}

enum { EPI_STORE = 0, EPI_RESIDUAL = 1, EPI_SWIGLU = 2 };

// ---------------------------------------------------------------------------
// Up to 8 tokens whose x fits shared memory.  CTAs of 16 warps; each warp keeps
// its column range of x there as fp16 operands, scaled per token by a power of
// two (largest value about 2^14), so that bf16 has the four-instruction operands
// too: what the scaling loses lies 2^-38 below the largest value.  The sums of
// x over the groups are taken once, in fp32.  TC is 1 or 8: one token alone has
// half the accumulators and leaves room for two CTAs an SM.
// What took it there (128,256 x 4096, one token): 58 us with 8 warps and a barrier
// an item, 50.6 with the sums of several items at one barrier and 16 warps, 45.1
// with x's sums and numbers read once a group, 43.5 with the operands of operand(),
// 42.9 with four warps at a time for the sums, which the others do not wait for (at 8
// tokens 54 instead of 64).
// With several tokens the instructions bound it: a code word has 4 of unpacking
// and its product, whatever the token count, but the accumulators and x's operands
// of 8 tokens leave room for one CTA an SM.
// ---------------------------------------------------------------------------
constexpr int64_t MAX_SMEM = 232448;   // of a CTA
constexpr int64_t HALF_SMEM = 115712;  // of each of two CTAs on an SM

template <int GS, int MT, int TC>
struct FewCfg {
  static constexpr int NW = 16;
  static constexpr int CK = GS > 64 ? GS : 64;
  static constexpr int TILES = CK / 64;
  static constexpr int SG = CK / GS;
  static constexpr int CODES = MT * TILES * 512;
  static constexpr int STAGE = CODES + MT * SG * 64;
  static constexpr int NST = (TC == 1 ? 75 : 107) * 1024 / (NW * STAGE);
  static constexpr int RING = NST * STAGE;
  static_assert(NST >= 2, "no stage ahead");
  // bytes of x operands and sums of a warp, for `chunks` chunks and `tokens` tokens
  __host__ __device__ static constexpr int x_row(int chunks) { return chunks * CK * 2 + 64; }
  __host__ __device__ static constexpr int64_t x_bytes(int64_t chunks, int tokens) {
    return tokens * (chunks * CK * 2 + 64) + chunks * SG * 32;
  }
  // items whose partial sums are added at once: about 128 values, one a lane of four
  // warps, whatever the number of tokens
  __host__ __device__ static constexpr int batch(int tokens) {
    return tokens >= 8 / MT ? 1 : 8 / (MT * tokens);
  }
  // words between two tokens' partial sums: lanes 2t tokens and r rows apart write
  // to 32 banks
  static constexpr int TS = MT * 16 + 4;
  __host__ __device__ static constexpr int red(int tokens) { return batch(tokens) * tokens * TS; }
  static constexpr int64_t smem(int64_t k, int tokens) {
    return NW * (RING + x_bytes((k / CK + NW - 1) / NW, tokens) + 2 * red(tokens) * 4) + 32;
  }
};

template <typename T, int GS, int MT, int TC>
__global__ void __launch_bounds__(512, TC == 1 ? 2 : 1)
    int4_few_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ numbers,
                    const T* x, const T* resid, T* out, int tokens_, int64_t n_out, int k,
                    int items, int epi) {
  using C = FewCfg<GS, MT, TC>;
  constexpr int NW = C::NW;
  constexpr int NC = TC == 1 ? 1 : 2;  // columns of the products that a lane keeps
  const int tokens = TC == 1 ? 1 : tokens_;
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = lane >> 2, t = lane & 3;
  const int nchunks = k / C::CK;
  const int64_t tile_codes = (int64_t)(k / 64) * 512, tile_numbers = (int64_t)(k / GS) * 64;
  const int c0 = warp * nchunks / NW, nc = (warp + 1) * nchunks / NW - c0;
  uint8_t* ring = smem + warp * C::RING;
  const uint32_t ring_u = lpc::smem_u32(ring);
  const int most = (nchunks + NW - 1) / NW;
  const int xrow = C::x_row(most);
  uint8_t* xw = smem + NW * C::RING + warp * (int)C::x_bytes(most, tokens);
  const int rs = C::red(tokens);
  float* red = reinterpret_cast<float*>(smem + NW * (C::RING + (int)C::x_bytes(most, tokens)));
  float* xs = reinterpret_cast<float*>(xw + tokens * xrow);  // [group][8 tokens]
  // two buffers of partial sums: written by all warps (full), added by four (empty)
  const uint32_t bars = lpc::smem_u32(red + 2 * NW * rs);
  auto full = [&](int i) { return bars + 8u * i; };
  auto empty = [&](int i) { return bars + 16u + 8u * i; };

  // the weight stream: this warp's chunks of item blockIdx.x, then of the next
  const uint8_t* fcode = codes + (int64_t)blockIdx.x * MT * tile_codes + c0 * (C::TILES * 512) + lane * 16;
  const uint8_t* fnum = numbers + (int64_t)blockIdx.x * MT * tile_numbers + c0 * (C::SG * 64) + r * 8;
  const int64_t jump_code = gridDim.x * MT * tile_codes - nc * (C::TILES * 512);
  const int64_t jump_num = gridDim.x * MT * tile_numbers - nc * (C::SG * 64);
  int fleft = nc > 0 ? nc * ((items - 1 - (int)blockIdx.x) / (int)gridDim.x + 1) : 0;
  int fc = nc;
  int fto = 0;
  auto advance = [&]() {
    if (fleft > 0) {
      --fleft;
      const uint32_t dst = ring_u + fto;
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < C::TILES; ++i)
          cp16(dst + (m * C::TILES + i) * 512 + lane * 16, fcode + m * tile_codes + i * 512);
      if (t == 0)
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int g = 0; g < C::SG; ++g)
            cp8(dst + C::CODES + (m * C::SG + g) * 64 + r * 8, fnum + m * tile_numbers + g * 64);
      fcode += C::TILES * 512;
      fnum += C::SG * 64;
      if (--fc == 0) {
        fc = nc;
        fcode += jump_code;
        fnum += jump_num;
      }
    }
    cp_commit();
    fto = fto == (C::NST - 1) * C::STAGE ? 0 : fto + C::STAGE;
  };

  lpc::pdl_trigger();
  // the weights belong to no earlier kernel of the stream: their first stages
  // are requested before the kernel that writes x is waited for
#pragma unroll
  for (int i = 0; i < C::NST - 1; ++i) advance();
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      lpc::mbar_init(full(i), NW);
      lpc::mbar_init(empty(i), 4);
    }
    lpc::fence_mbar_init();
  }
  __syncthreads();
  lpc::pdl_wait();

  // x of this warp's columns, in stretches of 256 (8 a lane)
  constexpr bool SCALE = !std::is_same<T, __half>::value;
  float down[NC];  // 2^-e of tokens 2t (and 2t + 1)
#pragma unroll
  for (int i = 0; i < NC; ++i) down[i] = 1.f;
  {
    const int width = nc * C::CK;
    const T* src = x + c0 * C::CK + lane * 8;
    auto load = [&](int tk, int st) {
      return tk < tokens && st * 256 + lane * 8 < width
                 ? lpc::ld_dep16(src + (int64_t)tk * k + st * 256) : make_uint4(0u, 0u, 0u, 0u);
    };
    // magnitudes of bf16 order as their bits do, two at a time; a NaN is the largest
    auto largest = [&](uint32_t a, const uint4& u) {
      constexpr uint32_t M = 0x7FFF7FFFu;
      return __vimax3_u16x2(__vimax3_u16x2(a, u.x & M, u.y & M), u.z & M, u.w & M);
    };
    auto factor = [&](int tk, uint32_t most) {  // 2^e of a token; keeps 2^-e where it is this lane's
      const uint32_t a = __reduce_max_sync(0xffffffffu, max(most & 0xFFFFu, most >> 16));
      int e = 0;
      if (a > 0u && a < 0x7F80u) e = min(126, 14 - ((int)(a >> 7) - 127));
      const float d = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
      for (int i = 0; i < NC; ++i)
        if (tk == NC * t + i) down[i] = d;
      return __uint_as_float((uint32_t)(127 + e) << 23);
    };
    auto keep = [&](int tk, int st, const uint4& u, float up) {
      uint32_t w[4] = {u.x, u.y, u.z, u.w};
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = pair_f<T>(w[i]);
        if constexpr (SCALE) {
          const __half2 h = __floats2half2_rn(f.x * up, f.y * up);
          w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        sum += f.x * up + f.y * up;
      }
      const int col = st * 256 + lane * 8;
      if (col < width)
        *reinterpret_cast<uint4*>(xw + tk * xrow + col * 2) = make_uint4(w[0], w[1], w[2], w[3]);
#pragma unroll
      for (int o = 1; o < GS / 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      // in the units of the accumulators, which hold c * 2^-24
      if (col < width && col % GS == 0) xs[(col / GS) * 8 + tk] = sum * 0x1p-24f;
    };
    // TK tokens by ST stretches at once: every load in flight, each value read once
    auto block = [&](auto tks, auto sts, int tk0) {
      constexpr int TK = decltype(tks)::value, ST = decltype(sts)::value;
      uint4 u[TK][ST];
#pragma unroll
      for (int i = 0; i < TK; ++i)
        if (tk0 + i < tokens)
#pragma unroll
          for (int j = 0; j < ST; ++j) u[i][j] = load(tk0 + i, j);
#pragma unroll
      for (int i = 0; i < TK; ++i)
        if (tk0 + i < tokens) {
          float up = 1.f;
          if constexpr (SCALE) {
            uint32_t a = 0u;
#pragma unroll
            for (int j = 0; j < ST; ++j) a = largest(a, u[i][j]);
            up = factor(tk0 + i, a);
          }
#pragma unroll
          for (int j = 0; j < ST; ++j)
            if (j * 256 < width) keep(tk0 + i, j, u[i][j], up);
        }
    };
    using one = std::integral_constant<int, 1>;
    using four = std::integral_constant<int, 4>;
    if (width <= 256) {
      block(std::integral_constant<int, TC>{}, one{}, 0);
    } else if (width <= 1024) {
      constexpr int TK = TC == 1 ? 1 : 2;
      for (int tk = 0; tk < tokens; tk += TK) block(std::integral_constant<int, TK>{}, four{}, tk);
    } else {
      for (int tk = 0; tk < tokens; ++tk) {
        float up = 1.f;
        if constexpr (SCALE) {
          uint32_t a = 0u;
          for (int st = 0; st * 256 < width; ++st) a = largest(a, load(tk, st));
          up = factor(tk, a);
        }
        for (int st = 0; st * 256 < width; ++st) keep(tk, st, load(tk, st), up);
      }
    }
  }
  __syncwarp();
  const uint8_t* px = xw + (r < tokens ? r : 0) * xrow + t * 16;

  int at = 0, held = 0;
  uint32_t turn = 0;  // batches so far
  bool ok = true;
  const int batch = C::batch(tokens), values = tokens * C::TS;
  const int prs = (epi == EPI_SWIGLU ? 3 : 4) + (MT == 2);  // log2 of an item's output rows
  for (int item = blockIdx.x; item < items; item += gridDim.x) {
    float sum[MT][2 * NC];  // rows r, then r + 8
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < 2 * NC; ++i) sum[m][i] = 0.f;
    const uint8_t* pc = px;
    const float* ps = xs + (NC == 1 ? 0 : 2 * t);
    for (int c = 0; c < nc; ++c) {
      cp_wait<C::NST - 2>();
      __syncwarp();  // the stage has arrived, and the one before it is free
      advance();
      const uint8_t* s = ring + at;
      at = at == (C::NST - 1) * C::STAGE ? 0 : at + C::STAGE;
      uint4 wv[MT];
#pragma unroll
      for (int g = 0; g < C::SG; ++g) {
        float acc[MT][4];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[m][i] = 0.f;
#pragma unroll
        for (int hh = 0; hh < GS / 32; ++hh) {
          const int half = g * (GS / 32) + hh;
          const uint4 xv = *reinterpret_cast<const uint4*>(pc + half * 64);
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            const uint8_t* at_w = s + (m * C::TILES + (half >> 1)) * 512 + lane * 16;
            if (!(half & 1)) wv[m] = *reinterpret_cast<const uint4*>(at_w);  // and the next half's
            uint32_t a[4], b[4];
            operand(half & 1 ? wv[m].z : wv[m].x, a);
            operand(half & 1 ? wv[m].w : wv[m].y, b);
            mma(acc[m], a, xv.x, xv.y);
            mma(acc[m], b, xv.z, xv.w);
          }
        }
        float x2[NC];
        x2[0] = ps[g * 8];
        if constexpr (NC == 2) {
          const float2 v = *reinterpret_cast<const float2*>(ps + g * 8);
          x2[0] = v.x;
          x2[1] = v.y;
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const uint2 w = *reinterpret_cast<const uint2*>(s + C::CODES + (m * C::SG + g) * 64 + r * 8);
          const float2 lo = pair_f<T>(w.x), hi = pair_f<T>(w.y);
          // the codes of rows r + 8 count 16-fold: so does their minimum, and
          // the sum is divided at the end
#pragma unroll
          for (int i = 0; i < NC; ++i) {
            sum[m][i] = fmaf(lo.x, acc[m][i] - acc[m][2 + i], fmaf(lo.y, x2[i], sum[m][i]));
            sum[m][NC + i] = fmaf(hi.x, acc[m][2 + i], fmaf(hi.y, x2[i] * 16.f, sum[m][NC + i]));
          }
        }
      }
      pc += C::CK * 2;
      ps += C::SG * 8;
    }
    // partial sums of the warps, [token][row] of the item; a buffer's last ones must
    // have been added
    const int buf = (int)(turn & 1u);
    if (held == 0 && turn >= 2 && ok)
      ok = __all_sync(0xffffffffu, lpc::mbar_wait(empty(buf), ((turn >> 1) & 1u) ^ 1u, &g_int4_few_status));
    float* mine = red + (buf * NW + warp) * rs + held * values;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < NC; ++i)
        if (NC * t + i < tokens) {
          float* p = mine + (NC * t + i) * C::TS + m * 16 + r;
          p[0] = sum[m][i] * down[i] * 0x1p24f;
          p[8] = sum[m][NC + i] * down[i] * 0x1p20f;
        }
    if (++held < batch && item + (int)gridDim.x < items) continue;
    __syncwarp();
    if (lane == 0) lpc::mbar_arrive(full(buf));
    // four warps, in turns, add the parts up, a value a lane, in a fixed order; the
    // others go on
    if ((uint32_t)(warp >> 2) == (turn & 3u)) {
      const float* part = red + buf * NW * rs;
      auto total = [&](int i) {
        float v[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) v[w] = part[w * rs + i];
#pragma unroll
        for (int w = 4; w < NW; ++w) v[w & 3] += part[w * rs + i];
        return (v[0] + v[1]) + (v[2] + v[3]);
      };
      const int count = (held * tokens) << prs;
      for (int i0 = (warp & 3) * 32; i0 < count; i0 += 128) {  // whole warps
        const int i = min(i0 + lane, count - 1), row = i & ((1 << prs) - 1);
        int tk = i >> prs, sub = 0;  // row of the batch's [item][token]
        if (tokens == 1) {
          sub = tk;
          tk = 0;
        } else {
          while (tk >= tokens) {
            tk -= tokens;
            ++sub;
          }
        }
        const int64_t n = ((int64_t)(item - (held - 1 - sub) * (int)gridDim.x) << prs) + row;
        const int64_t o = (int64_t)tk * n_out + n;
        const bool writes = n < n_out && i0 + lane < count;
        const float plus = epi == EPI_RESIDUAL && writes ? Num<T>::to_f(resid[o]) : 0.f;
        if (i0 < 128 && ok)
          ok = __all_sync(0xffffffffu, lpc::mbar_wait(full(buf), (turn >> 1) & 1u, &g_int4_few_status));
        const int at_p = sub * values + tk * C::TS + row;
        float v;
        if (epi == EPI_SWIGLU) {
          // half the lanes take up before gate: 32 banks
          const int first = lane & 16;
          const float a = total(at_p + first), b = total(at_p + 16 - first);
          const float gate = first ? b : a, upv = first ? a : b;
          v = __fdividef(gate, 1.f + __expf(-gate)) * upv;
        } else {
          v = total(at_p) + plus;
        }
        if (writes) out[o] = Num<T>::from_f(v);
      }
      __syncwarp();
      if (lane == 0) lpc::mbar_arrive(empty(buf));
    }
    held = 0;
    ++turn;
  }
  cp_wait<0>();
}

// ---------------------------------------------------------------------------
// Smaller weights (pick()): blocks of up to 16 tokens, x straight from global
// memory (the L1 and L2 caches), as it is.  fp16 takes the operands above; bf16 the pairs
// 128 + c, (w & 0x000F000F) | 0x43004300, exactly (a bf16 subnormal times x would
// underflow the fp32 sum), 7 instructions a word.  The 128 is taken out again with the
// group's sum of x, which costs the fp32 accumulator about 5 of its 24 bits and
// leaves an error some hundred times below the output's rounding, and x up to 2^113.  The sum of x is
// one more product, of a row of ones, kept in shared memory for the next items.
// 4096 x 4096 at 8 / 16 tokens: 4.2 / 5.6 us (stream 1.4); the loads of x, one of each 8
// columns and token for every tile row, bound it.
// ---------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ void operand_of(uint32_t w, uint32_t (&a)[4]) {
  if constexpr (std::is_same<T, __half>::value) {
    operand(w, a);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = ((w >> (4 * i)) & 0x000F000Fu) | 0x43004300u;
  }
}
template <typename T>
__device__ __forceinline__ void mma_of(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                       uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    mma(c, a, b0, b1);
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int GS, int MT, int NT>
struct Cfg {
  static constexpr int NW = 16;
  static constexpr int CK = GS > 64 ? GS : 64;  // columns of a pipeline stage
  static constexpr int TILES = CK / 64;
  static constexpr int SG = CK / GS;            // groups of a stage
  static constexpr int STAGE = MT * (TILES * 512 + SG * 256);
  static constexpr int NST = MT * TILES == 4 ? 3 : MT * TILES == 2 ? 5 : 7;
  static constexpr int RING = NST * STAGE;
  static constexpr int RED = MT * 16 * NT * 8;  // fp32 partial sums of a warp
  static constexpr int SMEM = NW * (RING + 2 * RED * 4);
  // bytes for the sums of x, beside the above
  static constexpr int XS_MAX = 232448 - SMEM < 24576 ? 232448 - SMEM : 24576;
  static_assert(XS_MAX >= 0, "shared memory");
};

template <typename T, int GS, int MT, int NT>
__global__ void __launch_bounds__(512, 1)
    int4_mid_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ numbers,
                   const T* x, const T* resid, T* out, int tokens, int64_t n_out, int k, int items,
                   int epi, int keep_sums) {
  using C = Cfg<GS, MT, NT>;
  constexpr int NW = C::NW;
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = lane >> 2, t = lane & 3;
  const int nchunks = k / C::CK;
  const int64_t tile_codes = (int64_t)(k / 64) * 512, tile_numbers = (int64_t)(k / GS) * 64;
  const int c0 = warp * nchunks / NW, nc = (warp + 1) * nchunks / NW - c0;
  const int tok0 = blockIdx.y * (NT * 8);
  const int ntok = min(NT * 8, tokens - tok0);
  uint8_t* ring = smem + warp * C::RING;
  const uint32_t ring_u = lpc::smem_u32(ring);
  float* red = reinterpret_cast<float*>(smem + NW * C::RING);
  // sums of x of this warp's groups, [group][token]
  float* xs = reinterpret_cast<float*>(smem + C::SMEM) +
              warp * ((nchunks + NW - 1) / NW) * C::SG * NT * 8;

  // the weight stream: this warp's chunks of item blockIdx.x, then of the next
  const uint8_t* fcode = codes + (int64_t)blockIdx.x * MT * tile_codes + c0 * (C::TILES * 512) + lane * 16;
  const uint8_t* fnum = numbers + (int64_t)blockIdx.x * MT * tile_numbers + c0 * (C::SG * 64) + r * 8;
  const int64_t jump_code = gridDim.x * MT * tile_codes - nc * (C::TILES * 512);
  const int64_t jump_num = gridDim.x * MT * tile_numbers - nc * (C::SG * 64);
  int fleft = nc > 0 ? nc * ((items - 1 - (int)blockIdx.x) / (int)gridDim.x + 1) : 0;
  int fc = nc;
  uint32_t fdst = ring_u;
  auto advance = [&]() {
    if (fleft > 0) {
      --fleft;
#pragma unroll
      for (int m = 0; m < MT; ++m) {
#pragma unroll
        for (int i = 0; i < C::TILES; ++i)
          cp16(fdst + (m * C::TILES + i) * 512 + lane * 16, fcode + m * tile_codes + i * 512);
#pragma unroll
        for (int g = 0; g < C::SG; ++g)
          cp8(fdst + MT * C::TILES * 512 + (m * C::SG + g) * 256 + lane * 8,
              fnum + m * tile_numbers + g * 64);
      }
      fcode += C::TILES * 512;
      fnum += C::SG * 64;
      if (--fc == 0) {
        fc = nc;
        fcode += jump_code;
        fnum += jump_num;
      }
    }
    cp_commit();
    fdst += C::STAGE;
    if (fdst == ring_u + C::RING) fdst = ring_u;
  };

  lpc::pdl_trigger();
  // the weights belong to no earlier kernel of the stream: their first stages
  // are requested before the kernel that writes x is waited for
#pragma unroll
  for (int i = 0; i < C::NST - 1; ++i) advance();
  lpc::pdl_wait();

  // x of token tok0 + 8 j + r: 8 columns at 32 h + 8 t of every 64.  A column
  // without a token repeats the first one; its sums are not stored.
  const T* xp[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j)
    xp[j] = x + (int64_t)(tok0 + (8 * j + r < ntok ? 8 * j + r : 0)) * k + c0 * C::CK + 8 * t;
  constexpr uint32_t ONE = std::is_same<T, __half>::value ? 0x3C003C00u : 0x3F803F80u;
  const uint32_t one[4] = {ONE, ONE, ONE, ONE};

  const uint8_t* s = ring;
  int buf = 0;
  bool fresh = true;  // the sums of x are not in xs
  for (int item = blockIdx.x; item < items; item += gridDim.x) {
    float sum[MT][NT][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[m][j][i] = 0.f;

    auto chunks = [&](auto with_sums) {
      constexpr bool SUMS = decltype(with_sums)::value;
      for (int c = 0; c < nc; ++c) {
        advance();
        cp_wait<C::NST - 1>();
        const int col = c * C::CK;
#pragma unroll
        for (int g = 0; g < C::SG; ++g) {
          float acc[MT][NT][4], ones[NT][4];
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              ones[j][i] = 0.f;
#pragma unroll
              for (int m = 0; m < MT; ++m) acc[m][j][i] = 0.f;
            }
          // 32-column halves of this group: GS 128 has 4, 64 has 2, 32 has 1
#pragma unroll
          for (int hh = 0; hh < GS / 32; ++hh) {
            const int half = g * (GS / 32) + hh;
            uint4 xv[NT];
#pragma unroll
            for (int j = 0; j < NT; ++j)
              xv[j] = lpc::ld_dep16(xp[j] + col + 32 * half);
#pragma unroll
            for (int m = 0; m < MT; ++m) {
              const uint2 w = *reinterpret_cast<const uint2*>(
                  s + (m * C::TILES + (half >> 1)) * 512 + lane * 16 + (half & 1) * 8);
              uint32_t a[4], b[4];
              operand_of<T>(w.x, a);
              operand_of<T>(w.y, b);
#pragma unroll
              for (int j = 0; j < NT; ++j) {
                mma_of<T>(acc[m][j], a, xv[j].x, xv[j].y);
                mma_of<T>(acc[m][j], b, xv[j].z, xv[j].w);
              }
            }
            if constexpr (SUMS) {
#pragma unroll
              for (int j = 0; j < NT; ++j) {
                mma_of<T>(ones[j], one, xv[j].x, xv[j].y);
                mma_of<T>(ones[j], one, xv[j].z, xv[j].w);
              }
            }
          }
          float* px = xs + (c * C::SG + g) * (NT * 8) + 2 * t;
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            if constexpr (SUMS) {
              if (keep_sums && r == 0)
                *reinterpret_cast<float2*>(px + 8 * j) = make_float2(ones[j][0], ones[j][1]);
            } else {
              const float2 v = *reinterpret_cast<const float2*>(px + 8 * j);
              ones[j][0] = v.x;
              ones[j][1] = v.y;
            }
          }
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            const uint2 w = *reinterpret_cast<const uint2*>(
                s + MT * C::TILES * 512 + (m * C::SG + g) * 256 + lane * 8);
            const float2 lo = pair_f<T>(w.x), hi = pair_f<T>(w.y);
            float s0, m0, s1, m1;
            if constexpr (std::is_same<T, __half>::value) {
              s0 = lo.x * 16777216.f;
              m0 = lo.y;
              s1 = hi.x * 1048576.f;
              m1 = hi.y;
            } else {
              s0 = lo.x;
              m0 = fmaf(-128.f, lo.x, lo.y);
              s1 = hi.x;
              m1 = fmaf(-128.f, hi.x, hi.y);
            }
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              if constexpr (std::is_same<T, __half>::value) {
                acc[m][j][0] -= acc[m][j][2];
                acc[m][j][1] -= acc[m][j][3];
              }
              sum[m][j][0] = fmaf(s0, acc[m][j][0], fmaf(m0, ones[j][0], sum[m][j][0]));
              sum[m][j][1] = fmaf(s0, acc[m][j][1], fmaf(m0, ones[j][1], sum[m][j][1]));
              sum[m][j][2] = fmaf(s1, acc[m][j][2], fmaf(m1, ones[j][0], sum[m][j][2]));
              sum[m][j][3] = fmaf(s1, acc[m][j][3], fmaf(m1, ones[j][1], sum[m][j][3]));
            }
          }
        }
        s += C::STAGE;
        if (s == ring + C::RING) s = ring;
      }
    };
    if (fresh) {
      chunks(std::true_type{});
      fresh = !keep_sums;
      __syncwarp();
    } else {
      chunks(std::false_type{});
    }
    // partial sums of the warps, [token][row] of the item, added in warp order
    float* mine = red + (buf * NW + warp) * C::RED;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        float* p = mine + (8 * j + 2 * t) * (MT * 16) + m * 16 + r;
        p[0] = sum[m][j][0];
        p[MT * 16] = sum[m][j][1];
        p[8] = sum[m][j][2];
        p[MT * 16 + 8] = sum[m][j][3];
      }
    __syncthreads();
    const float* all = red + buf * NW * C::RED;
    auto total = [&](int at) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) v += all[w * C::RED + at];
      return v;
    };
    if (epi == EPI_SWIGLU) {
      if constexpr (MT == 2)
        for (int i = threadIdx.x; i < ntok * 16; i += NW * 32) {
          const int tk = i >> 4, row = i & 15;
          const int64_t n = (int64_t)item * 16 + row;
          if (n >= n_out) continue;
          const float gate = total(tk * 32 + row), upv = total(tk * 32 + 16 + row);
          out[(int64_t)(tok0 + tk) * n_out + n] =
              Num<T>::from_f(__fdividef(gate, 1.f + __expf(-gate)) * upv);
        }
    } else {
      for (int i = threadIdx.x; i < ntok * (MT * 16); i += NW * 32) {
        const int tk = i / (MT * 16), row = i % (MT * 16);
        const int64_t n = (int64_t)item * (MT * 16) + row;
        if (n >= n_out) continue;
        float v = total(i);
        const int64_t o = (int64_t)(tok0 + tk) * n_out + n;
        if (epi == EPI_RESIDUAL) v += Num<T>::to_f(resid[o]);
        out[o] = Num<T>::from_f(v);
      }
    }
    buf ^= 1;
  }
  cp_wait<0>();
}

// ---------------------------------------------------------------------------
// layout
// ---------------------------------------------------------------------------
// Source row of row `i` of tile row `p`, or -1 for padding.
__device__ __forceinline__ int64_t source_row(int64_t p, int i, int64_t n_out, int layout) {
  const int64_t n = (layout == 1 ? p >> 1 : p) * 16 + i;
  if (n >= n_out) return -1;
  return layout == 1 && (p & 1) ? n_out + n : n;
}
// Row and column (in the 64) of nibble `i`, half `p` of word j of lane (r, t).
__device__ __forceinline__ int nibble_row(int r, int i) { return r + 8 * (i & 1); }
__device__ __forceinline__ int nibble_col(int t, int j, int i, int p) {
  return 32 * (j >> 1) + 8 * t + 4 * (j & 1) + 2 * (i >> 1) + p;
}

// One thread: one packed word.
__global__ void int4_pack_kernel(const uint8_t* __restrict__ src, uint32_t* __restrict__ dst,
                                 int64_t words, int64_t n_out, int k, int layout) {
  const int64_t at = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (at >= words) return;
  const int j = (int)(at & 3), lane = (int)((at >> 2) & 31);
  const int64_t tk = at >> 7;
  const int64_t p = tk / (k / 64);
  const int kb = (int)(tk - p * (k / 64));
  const int r = lane >> 2, t = lane & 3;
  uint32_t w = 0u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t row = source_row(p, nibble_row(r, i), n_out, layout);
    if (row < 0) continue;
    const int col = kb * 64 + nibble_col(t, j, i, 0);  // even: the pair shares a byte
    const uint32_t byte = src[row * (k / 2) + col / 2];
    w |= (byte & 15u) << (4 * i);
    w |= (byte >> 4) << (4 * i + 16);
  }
  dst[at] = w;
}

template <typename T>
__global__ void int4_pack_numbers_kernel(const T* __restrict__ s, const T* __restrict__ m,
                                         T* __restrict__ dst, int64_t count, int64_t n_out, int ng,
                                         int layout) {
  const int64_t at = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;  // (tile row, group, r)
  if (at >= count) return;
  const int r = (int)(at & 7);
  const int64_t pg = at >> 3;
  const int64_t p = pg / ng;
  const int g = (int)(pg - p * ng);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int64_t row = source_row(p, r + 8 * h, n_out, layout);
    dst[at * 4 + 2 * h] = row < 0 ? Num<T>::from_f(0.f) : s[row * ng + g];
    dst[at * 4 + 2 * h + 1] = row < 0 ? Num<T>::from_f(0.f) : m[row * ng + g];
  }
}

// One thread: one row of a tile row, the power that brings its numbers into
// fp16's range and the numbers in it.
template <typename T>
__global__ void int4_pack_scaled_kernel(const T* __restrict__ s, const T* __restrict__ m,
                                        __half2* __restrict__ scaled, float* __restrict__ factors,
                                        int64_t count, int64_t n_out, int ng, int layout) {
  const int64_t at = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;  // (tile row, row)
  if (at >= count) return;
  const int64_t p = at >> 4;
  const int i = (int)(at & 15);
  const int64_t row = source_row(p, i, n_out, layout);
  float top = 0.f;
  for (int g = 0; row >= 0 && g < ng; ++g) {
    const float a = fmaf(15.f, fabsf(Num<T>::to_f(s[row * ng + g])), fabsf(Num<T>::to_f(m[row * ng + g])));
    if (a < INFINITY) top = fmaxf(top, a);
  }
  int e = 0;
  if (top > 0.f) e = max(-126, min(126, 14 - ((int)(__float_as_uint(top) >> 23) - 127)));
  const float up = __uint_as_float((uint32_t)(127 + e) << 23);
  factors[at] = __uint_as_float((uint32_t)(127 - e) << 23);
  for (int g = 0; g < ng; ++g) {
    float a = 0.f, b = 0.f;
    if (row >= 0) {
      a = Num<T>::to_f(s[row * ng + g]) * up;
      b = Num<T>::to_f(m[row * ng + g]) * up;
    }
    scaled[(p * ng + g) * 16 + i] = __floats2half2_rn(a, b);
  }
}

// One thread: one packed word, 8 values written as 4 pairs.
template <typename T>
__global__ void int4_unpack_kernel(const uint32_t* __restrict__ codes, const T* __restrict__ numbers,
                                   T* __restrict__ out, int64_t words, int64_t n_out, int k,
                                   int group, int layout) {
  const int64_t at = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (at >= words) return;
  const int j = (int)(at & 3), lane = (int)((at >> 2) & 31);
  const int64_t tk = at >> 7;
  const int64_t p = tk / (k / 64);
  const int kb = (int)(tk - p * (k / 64));
  const int r = lane >> 2, t = lane & 3;
  const uint32_t w = codes[at];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t row = source_row(p, nibble_row(r, i), n_out, layout);
    if (row < 0) continue;
    const int col = kb * 64 + nibble_col(t, j, i, 0);
    const T* nb = numbers + ((p * (k / group) + col / group) * 8 + r) * 4 + 2 * (i & 1);
    const float s = Num<T>::to_f(nb[0]), m = Num<T>::to_f(nb[1]);
    __align__(4) T v[2];
    v[0] = Num<T>::from_f(fmaf((float)((w >> (4 * i)) & 15u), s, m));
    v[1] = Num<T>::from_f(fmaf((float)((w >> (4 * i + 16)) & 15u), s, m));
    *reinterpret_cast<uint32_t*>(out + row * k + col) = *reinterpret_cast<const uint32_t*>(v);
  }
}

// Items of MT tile rows each.
int few_items(const lpc_w4* w, int mt) {
  const int64_t tr = (w->n_out + 15) / 16 * (w->layout == 1 ? 2 : 1);
  return (int)((tr + mt - 1) / mt);
}

template <typename T, int GS, int MT, int TC>
int launch_few(const lpc_w4* w, const void* x, void* out, const void* resid, int64_t tokens,
               int epi, cudaStream_t s) {
  using C = FewCfg<GS, MT, TC>;
  static std::atomic<uint64_t> mask{0};
  int rc = lpc::once_per_device_smem((const void*)int4_few_kernel<T, GS, MT, TC>, (int)MAX_SMEM, mask);
  if (rc) return rc;
  const int items = few_items(w, MT);
  const int64_t smem = C::smem(w->k, (int)tokens);
  const int slots = lpc::current_device_sms() * (TC == 1 && smem <= HALF_SMEM ? 2 : 1);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = lpc::use_pdl() ? 1 : 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)std::min(items, slots));
  cfg.blockDim = dim3(512);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const lpc::Int4Parts p = lpc::int4_parts(w->packed, w->n_out, w->k, w->group, w->layout);
  cudaLaunchKernelEx(&cfg, int4_few_kernel<T, GS, MT, TC>, (const uint8_t*)p.codes,
                     (const uint8_t*)p.numbers, (const T*)x,
                     (const T*)resid, (T*)out, (int)tokens, w->n_out, w->k, items, epi);
  return lpc::check_launch("int4_linear");
}

// Two tile rows an item share x's operands and the barrier; one where that
// leaves an SM without work.
template <typename T, int GS, int TC>
int launch_few_mt(const lpc_w4* w, const void* x, void* out, const void* resid, int64_t tokens,
                  int epi, cudaStream_t s) {
  const bool one = few_items(w, 1) <= lpc::current_device_sms() * (TC == 1 ? 2 : 1);
  if (w->layout == 0 && one) return launch_few<T, GS, 1, TC>(w, x, out, resid, tokens, epi, s);
  return launch_few<T, GS, 2, TC>(w, x, out, resid, tokens, epi, s);
}

template <typename T, int GS, int MT, int NT>
int launch_mid(const lpc_w4* w, const void* x, void* out, const void* resid, int64_t tokens, int epi,
           cudaStream_t s) {
  using C = Cfg<GS, MT, NT>;
  constexpr int NW = C::NW;
  static std::atomic<uint64_t> mask{0};
  int rc = lpc::once_per_device_smem((const void*)int4_mid_kernel<T, GS, MT, NT>,
                                     C::SMEM + C::XS_MAX, mask);
  if (rc) return rc;
  const int items = few_items(w, MT);
  // the sums of x are computed with the first item and kept for the next ones
  const int64_t sums = (int64_t)NW * ((w->k / C::CK + NW - 1) / NW) * C::SG * NT * 8 * 4;
  const int slots = lpc::current_device_sms();
  const int keep = items > slots && sums <= C::XS_MAX;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = lpc::use_pdl() ? 1 : 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)std::min(items, slots), (unsigned)((tokens + NT * 8 - 1) / (NT * 8)));
  cfg.blockDim = dim3(NW * 32);
  cfg.dynamicSmemBytes = C::SMEM + (keep ? (int)sums : 0);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const lpc::Int4Parts p = lpc::int4_parts(w->packed, w->n_out, w->k, w->group, w->layout);
  cudaLaunchKernelEx(&cfg, int4_mid_kernel<T, GS, MT, NT>, (const uint8_t*)p.codes,
                     (const uint8_t*)p.numbers, (const T*)x, (const T*)resid, (T*)out, (int)tokens,
                     w->n_out, w->k, items, epi, keep);
  return lpc::check_launch("int4_linear");
}

// Which kernel takes the products (int4_many.cu has MANY).
enum Kernel { FEW, MID, MANY };
// MID has no preparation of x, FEW a faster weight stream: MID up to (8 + 3 tokens) 2^20
// values.  Measured, us, few / mid at 1 / 4 / 8 tokens: 2048 x 4096 3.0 / 2.9, 4.1 / 3.0
// at 4; 4096 x 4096 3.8 / 4.0, 4.5 / 4.1, 5.8 / 4.2; 6144 x 4096 4.8 / 6.6, 5.8 / 6.8,
// 7.2 / 6.8; 12,288 x 4096 7.7 / 9.9, 7.6 / 9.9, 9.4 / 10.1.
// More than 16 tokens cost MID a pass over the weight per 16, and MANY hardly more than
// few do: MID where blocks^2 times values are at most MID_MOST.  Measured, us, mid /
// many: 14,336 x 4096 at 16 tokens 18.5 / 19.4, 22,016 x 4096 25.0 / 21.2; at 32 tokens
// 4096 x 4096 10.2 / 11.3, 6144 x 4096 14.6 / 12.8; at 64 4096 x 1024 11.0 / 10.7,
// 2048 x 4096 15.4 / 11.3 (MANY before its weights' subtraction, 2 to 6% less than now).
constexpr int64_t MID_MOST = 72 << 20;
// x fits the few-token kernel's shared memory, with one tile row an item or two
// (the rings round differently).
template <int GS, int TC>
bool few_fits(int k, int64_t tokens) {
  return tokens <= TC && std::max(FewCfg<GS, 1, TC>::smem(k, (int)tokens),
                                  FewCfg<GS, 2, TC>::smem(k, (int)tokens)) <= MAX_SMEM;
}
template <int GS>
Kernel pick(const lpc_w4* w, int64_t tokens) {
  const int64_t values = (w->n_out << w->layout) * w->k, blocks = (tokens + 15) / 16;
  if (values > (8 + 3 * tokens) << 20 &&
      (few_fits<GS, 1>(w->k, tokens) || few_fits<GS, 8>(w->k, tokens)))
    return FEW;
  return blocks * blocks * values <= MID_MOST ? MID : MANY;
}
Kernel pick(const lpc_w4* w, int64_t tokens) {
  return w->group == 128 ? pick<128>(w, tokens) : w->group == 64 ? pick<64>(w, tokens) : pick<32>(w, tokens);
}

// Two tile rows an item share the loads of x; one where two would leave SMs without
// an item.  Measured, us, one / two: 2048 x 4096 at 16 tokens 4.3 / 5.0, 4096 x 4096
// 6.5 / 5.6, 4096 x 11,008 14.7 / 11.1.
template <typename T, int GS, int NT>
int launch_mid_mt(const lpc_w4* w, const void* x, void* out, const void* resid, int64_t tokens,
                  int epi, cudaStream_t s) {
  if (w->layout == 0 && few_items(w, 1) <= lpc::current_device_sms())
    return launch_mid<T, GS, 1, NT>(w, x, out, resid, tokens, epi, s);
  return launch_mid<T, GS, 2, NT>(w, x, out, resid, tokens, epi, s);
}

template <typename T, int GS>
int launch_nt(const lpc_w4* w, const void* x, void* out, const void* resid, int64_t tokens, int epi,
              cudaStream_t s) {
  if (pick<GS>(w, tokens) == MID)
    return tokens <= 8 ? launch_mid_mt<T, GS, 1>(w, x, out, resid, tokens, epi, s)
                       : launch_mid_mt<T, GS, 2>(w, x, out, resid, tokens, epi, s);
  if (few_fits<GS, 1>(w->k, tokens))
    return launch_few_mt<T, GS, 1>(w, x, out, resid, tokens, epi, s);
  return launch_few_mt<T, GS, 8>(w, x, out, resid, tokens, epi, s);
}

template <typename T>
int launch_gs(const lpc_w4* w, const void* x, void* out, const void* resid, int64_t tokens, int epi,
              cudaStream_t s) {
  if (w->group == 128) return launch_nt<T, 128>(w, x, out, resid, tokens, epi, s);
  if (w->group == 64) return launch_nt<T, 64>(w, x, out, resid, tokens, epi, s);
  return launch_nt<T, 32>(w, x, out, resid, tokens, epi, s);
}

bool shape_ok(int64_t n_out, int k, int group, int layout) {
  return n_out > 0 && n_out <= (1 << 24) && k > 0 && k <= (1 << 20) && n_out * k <= (1LL << 38) &&
         k % 64 == 0 &&
         (group == 32 || group == 64 || group == 128) && k % group == 0 &&
         (layout == 0 || layout == 1);
}

int weight_check(const lpc_w4* w, const char* what) {
  if (!w || !w->packed || !lpc::aligned16(w->packed) ||
      !shape_ok(w->n_out, w->k, w->group, w->layout)) {
    lpc::set_error("%s: invalid packed weight", what);
    return LPC_ERR_INVALID;
  }
  if (w->dtype != LPC_DTYPE_BF16 && w->dtype != LPC_DTYPE_F16) {
    lpc::set_error("%s: only bf16 and fp16 are supported", what);
    return LPC_ERR_UNSUPPORTED;
  }
  return LPC_OK;
}

}  // namespace

extern "C" int64_t lpc_int4_weight_bytes(int64_t n_out, int k, int group, int layout) {
  if (!shape_ok(n_out, k, group, layout)) return 0;
  return lpc::int4_parts(nullptr, n_out, k, group, layout).bytes;
}

extern "C" int64_t lpc_int4_linear_workspace_bytes(const lpc_w4* w, int64_t tokens) {
  if (weight_check(w, "int4_linear") || tokens <= 0 || tokens > MAX_TOKENS || pick(w, tokens) != MANY ||
      w->dtype == LPC_DTYPE_F16)
    return 0;
  return tokens * (int64_t)w->k * 2 + MAX_TOKENS * 4;
}

extern "C" int lpc_int4_pack(const lpc_w4* w, const void* codes, const void* scales,
                             const void* mins, void* stream) {
  using namespace lpc;
  int rc = weight_check(w, "int4_pack");
  if (rc) return rc;
  if (!codes || !scales || !mins) {
    set_error("int4_pack: null pointer");
    return LPC_ERR_INVALID;
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t tr = lpc::int4_tile_rows(w->n_out, w->layout);
  const int64_t words = tr * (w->k / 64) * 128;
  const int ng = w->k / w->group;
  const int64_t count = tr * ng * 8;
  const Int4Parts p = int4_parts(w->packed, w->n_out, w->k, w->group, w->layout);
  int4_pack_kernel<<<(unsigned)((words + 255) / 256), 256, 0, s>>>(
      (const uint8_t*)codes, (uint32_t*)p.codes, words, w->n_out, w->k, w->layout);
  // 16-bit numbers are moved, not computed with: one type serves both
  int4_pack_numbers_kernel<__half><<<(unsigned)((count + 255) / 256), 256, 0, s>>>(
      (const __half*)scales, (const __half*)mins, (__half*)p.numbers, count, w->n_out, ng,
      w->layout);
  const unsigned rows = (unsigned)((tr * 16 + 127) / 128);
  if (w->dtype == LPC_DTYPE_BF16)
    int4_pack_scaled_kernel<__nv_bfloat16><<<rows, 128, 0, s>>>(
        (const __nv_bfloat16*)scales, (const __nv_bfloat16*)mins, (__half2*)p.scaled, p.factors,
        tr * 16, w->n_out, ng, w->layout);
  else
    int4_pack_scaled_kernel<__half><<<rows, 128, 0, s>>>(
        (const __half*)scales, (const __half*)mins, (__half2*)p.scaled, p.factors, tr * 16,
        w->n_out, ng, w->layout);
  if ((rc = check_launch("int4_pack"))) return rc;
  // the products read the weight before they wait on the kernel before them
  if (cudaStreamSynchronize(s) != cudaSuccess) {
    set_error("int4_pack: synchronisation failed");
    return LPC_ERR_CUDA;
  }
  return LPC_OK;
}

extern "C" int lpc_int4_unpack(const lpc_w4* w, void* out, void* stream) {
  using namespace lpc;
  int rc = weight_check(w, "int4_unpack");
  if (rc) return rc;
  if (!out || !aligned16(out)) {
    set_error("int4_unpack: out must be given and 16-byte aligned");
    return LPC_ERR_INVALID;
  }
  const int64_t tr = lpc::int4_tile_rows(w->n_out, w->layout);
  const int64_t words = tr * (w->k / 64) * 128;
  const Int4Parts parts = int4_parts(w->packed, w->n_out, w->k, w->group, w->layout);
  const uint8_t *base = parts.codes, *nb = parts.numbers;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const unsigned grid = (unsigned)((words + 255) / 256);
  if (w->dtype == LPC_DTYPE_BF16)
    int4_unpack_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>((const uint32_t*)base,
                                                           (const __nv_bfloat16*)nb,
                                                           (__nv_bfloat16*)out, words, w->n_out,
                                                           w->k, w->group, w->layout);
  else
    int4_unpack_kernel<__half><<<grid, 256, 0, s>>>((const uint32_t*)base, (const __half*)nb,
                                                    (__half*)out, words, w->n_out, w->k, w->group,
                                                    w->layout);
  return check_launch("int4_unpack");
}

extern "C" int lpc_int4_linear(const lpc_w4* w, const void* x, void* out, const void* resid,
                               int64_t tokens, int epilogue, void* workspace,
                               int64_t workspace_bytes, void* stream) {
  using namespace lpc;
  int rc = weight_check(w, "int4_linear");
  if (rc) return rc;
  if (tokens < 0 || tokens > MAX_TOKENS) {
    set_error("int4_linear: takes at most %d tokens, got %lld", MAX_TOKENS, (long long)tokens);
    return LPC_ERR_INVALID;
  }
  if (epilogue < 0 || epilogue > 2 || (epilogue == EPI_SWIGLU) != (w->layout == 1)) {
    set_error("int4_linear: epilogue %d does not fit a weight of layout %d", epilogue, w->layout);
    return LPC_ERR_INVALID;
  }
  if (tokens == 0) return LPC_OK;
  if (!x || !out || !aligned16(x) || (epilogue == EPI_RESIDUAL && !resid)) {
    set_error("int4_linear: x (16-byte aligned), out and, for the residual epilogue, resid must be "
              "given");
    return LPC_ERR_INVALID;
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (pick(w, tokens) != MANY)
    return w->dtype == LPC_DTYPE_BF16
               ? launch_gs<__nv_bfloat16>(w, x, out, resid, tokens, epilogue, s)
               : launch_gs<__half>(w, x, out, resid, tokens, epilogue, s);
  const int64_t need = lpc_int4_linear_workspace_bytes(w, tokens);
  if (need && (!workspace || workspace_bytes < need || !aligned16(workspace))) {
    set_error("int4_linear: workspace of %lld bytes required, got %lld", (long long)need,
              (long long)workspace_bytes);
    return LPC_ERR_INVALID;
  }
  return int4_many(w, x, out, resid, tokens, epilogue, workspace, s);
}
