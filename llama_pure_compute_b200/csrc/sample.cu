// Sampling of one token a row from logits, with temperature, top-k, top-p and
// min-p and a given random number u in [0, 1).
//
// Definition.  Logits are ordered from the largest down, equal ones by index;
// w_i = exp((l_i - max) / temperature).
//   top-k   keeps the first k of the order;
//   top-p   of these the ones before which at most p * (their sum) stands;
//   min-p   of these the ones with w_i >= min_p.
// Token: the lowest index at which the running sum of the kept weights, in the
// order of the indices, exceeds u * (their sum).  temperature 0: the first of
// the order.  -inf and NaN are never drawn; a row of nothing else gives -1.
//
// A cluster of 1, 2, 4 or 8 CTAs holds a row in its shared memory (one read of
// the logits) and passes over it there:
//   * Weights are integers: round(2^44 w), w in 64 bits.  Their sums are exact,
//     whatever the order in which threads add, so the parts of a cluster agree on
//     every comparison, and the products p * sum and u * sum are compared exactly.
//     A sum is off by at most 2^-45 an element relative to the largest weight.  fp32
//     sums would move a token's border by ~2^-22: one row in a hundred draws another
//     token where 100,000 tokens are about equally likely.
//   * 2^y is 2^e * 2^(j/32) * a polynomial of degree 4 on +-1/64 (argument reduction
//     by a table, Tang 1989; the series' next term is 1.2e-12): nine fp64
//     operations, a third of exp2()'s.
//   * Every filter keeps a prefix of the order, so a filter is one place in it: a
//     value and, among equals, an index.  A histogram over 2048 bins of 1/64 octave
//     of the weight, of counts or of fp32 weights, says in which bins the place lies;
//     their few elements go to a list and are ranked exactly, by pairs.  With top-k
//     the list has all that is kept, and the rest is done on it.
//   * Where the list would not hold them (many equal logits, thousands kept by top-k,
//     places beyond the bins), the place is found by radix select: histograms over 11
//     bits of the order-preserving integer of the value, of counts or of integer
//     weights.
//   * The token: sums of each warp's stretch, a scan over the cluster's warps, and
//     the warp whose stretch holds the border walks it.
#include <atomic>

#include "lpc_common.cuh"

LPC_DECLARE_STATUS(g_sample_status)

unsigned int lpc_status_sample(bool clear) {
  unsigned int v = 0;
  cudaMemcpyFromSymbol(&v, g_sample_status, sizeof(v));
  if (clear && v) {
    unsigned int z = 0;
    cudaMemcpyToSymbol(g_sample_status, &z, sizeof(z));
  }
  return v;
}

namespace {

using lpc::Num;

constexpr int THREADS = 512;
constexpr int WARPS = THREADS / 32;
constexpr int MAX_CLUSTER = 8;
constexpr int BINS = 2048;                       // 11 bits a round
constexpr int HIST_BYTES = BINS * 8;             // low and high words of a bin's sum
constexpr double FIXED = 17592186044416.0;       // 2^44
constexpr double ROUND52 = 4503599627370496.0;   // 2^52: adding it rounds to an integer
constexpr int LIST = 512;                        // elements that are ranked by pairs
constexpr int OCTAVE = 64;                       // bins an octave of the weight
// What the fp32 histogram may be off, relative to all weights: its elements by 2^-16 of
// rounding and 4e-6 of fp32 arithmetic, twice, and what lies below its 32 octaves, at most
// 770,048 * 2^-32 = 1.8e-4.
constexpr double SLACK = 2.5e-4;
constexpr int SLICE_BYTES = 64 * 1024;           // preferred share of a CTA
constexpr int MAX_SLICE_BYTES = 188 * 1024;
constexpr int BATCH = 4;                         // 16-byte loads in flight a thread

struct Args {
  const void* logits;
  int64_t row_stride;                   // elements
  int vocab, slice;                     // elements a row, elements a CTA
  const float* uniforms;
  const float *temperature, *top_p, *min_p;  // per row, or null: the numbers below
  const int32_t* top_k;
  float t, p, m;
  int32_t k;
  int64_t* out;
};

// log2 of the step between the integers of neighbouring values (fp16 and bf16
// widened to fp32)
template <typename T> constexpr int GRAIN = 0;
template <> constexpr int GRAIN<__half> = 13;
template <> constexpr int GRAIN<__nv_bfloat16> = 16;

// Integer with the order of the floats; -0 and +0 are equal.
__device__ __forceinline__ int32_t order_of(float f) {
  const int32_t s = __float_as_int(f);
  return s >= 0 ? s : (int32_t)(0x80000000u - (uint32_t)s);
}
__device__ __forceinline__ float value_of(int32_t key) {
  return __int_as_float(key >= 0 ? key : (int32_t)(0x80000000u - (uint32_t)key));
}

// One 16-byte chunk of logits as floats.
template <typename T>
struct Chunk {
  static constexpr int N = 16 / (int)sizeof(T);
  uint4 raw;
  __device__ __forceinline__ float get(int i) const {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(i == 0 ? raw.x : i == 1 ? raw.y : i == 2 ? raw.z : raw.w);
    } else {
      const uint32_t w = i < 2 ? raw.x : i < 4 ? raw.y : i < 6 ? raw.z : raw.w;
      if constexpr (sizeof(T) == 2 && GRAIN<T> == 16) {
        return (i & 1) ? lpc::bf16hi(w) : lpc::bf16lo(w);
      } else {
        return __half2float(__ushort_as_half((unsigned short)((i & 1) ? w >> 16 : w & 0xffffu)));
      }
    }
  }
};

__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int m) {
  return ((uint64_t)__shfl_xor_sync(~0u, (uint32_t)(v >> 32), m) << 32) |
         __shfl_xor_sync(~0u, (uint32_t)v, m);
}
__device__ __forceinline__ uint64_t shfl_up64(uint64_t v, int d) {
  return ((uint64_t)__shfl_up_sync(~0u, (uint32_t)(v >> 32), d) << 32) |
         __shfl_up_sync(~0u, (uint32_t)v, d);
}
__device__ __forceinline__ uint64_t warp_sum(uint64_t v) {
#pragma unroll
  for (int m = 16; m; m >>= 1) v += shfl_xor64(v, m);
  return v;
}
__device__ __forceinline__ uint64_t warp_scan(uint64_t v, int lane) {  // inclusive
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint64_t o = shfl_up64(v, d);
    if (lane >= d) v += o;
  }
  return v;
}

// floor(f * n) for 0 <= f < 1, exactly.
__device__ __forceinline__ uint64_t part_of(float f, uint64_t n) {
  const uint32_t b = __float_as_uint(f);
  const int e = (int)(b >> 23);                       // f = mant * 2^(e - 150)
  const uint64_t mant = e ? (b & 0x7fffffu) | 0x800000u : b & 0x7fffffu;
  const int sh = 150 - (e ? e : 1);                   // 24 .. 149
  const uint64_t lo = mant * n, hi = __umul64hi(mant, n);
  if (sh >= 128) return 0;                            // mant * n < 2^88
  if (sh >= 64) return hi >> (sh - 64);
  return (lo >> sh) | (hi << (64 - sh));
}

__device__ __forceinline__ uint32_t ld_remote(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint4 ld_remote16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared::cluster.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ void st_remote64(uint32_t addr, uint64_t v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}

struct Entry {  // an element in the order: by offset from the largest, then by index
  uint32_t index, off;
};
__device__ __forceinline__ uint64_t place_of(const Entry& e) { return (uint64_t)e.off << 32 | e.index; }

struct Shared {
  double table[32];                       // 2^44 * 2^(j/32)
  uint32_t listed;                        // elements that this CTA put on its list
  uint32_t window[2];                     // first and last bin that may hold the place
  unsigned long long cut;                 // place of the last that stays
  uint64_t list_sum;
  uint64_t sums[3][MAX_CLUSTER * WARPS];  // written by every CTA of the cluster
  uint64_t found[2];                      // a located index, written by its finder
  uint64_t warp_best[WARPS];
  uint64_t scan[WARPS];
  uint64_t cross_before, cross_in;        // sum before the crossing bin, and in it
  int cross_bin;
};

template <typename T>
class Row {
 public:
  static constexpr int N = Chunk<T>::N;
  const Args& a;
  Shared& sh;
  uint4* chunks;              // this CTA's share of the row, -inf outside it
  uint32_t* hist[2];          // low words, then high words
  int rank, ctas, warp, lane;
  int nchunks, segment;       // chunks of this CTA; of a warp (a multiple of 32)
  int first;                  // row index of element 0 of chunk 0 (may lie before the share)
  int begin, end;             // row indexes of the share
  int32_t kmax;               // order_of(largest)
  double top, scale;          // largest, log2(e) / temperature
  int turn = 0;               // which histogram the next round takes
  int slot = 0;               // which sums the next exchange takes
  int found_slot = 0;

  __device__ Row(const Args& args, Shared& s) : a(args), sh(s) {}

  __device__ __forceinline__ Chunk<T> chunk(int c) const {
    Chunk<T> r;
    r.raw = chunks[c];
    return r;
  }
  float topf, octaves, lowest;  // largest; -OCTAVE log2(e) / temperature; offset of the last bin
  uint32_t tab_lo, tab_hi;      // table entry `lane`

  // round(2^44 w) of a finite logit; `exact`: 2^44 w itself.  ALL: every lane of the
  // warp is here, and the table comes from the lanes' registers.
  template <bool ALL>
  __device__ __forceinline__ uint64_t weight(float f, double& exact) const {
    constexpr double A1 = 0.02166084939249829, A2 = 0.00023459619820224677;  // (ln2/32)^k / k!
    constexpr double A3 = 1.6938509724371819e-06, A4 = 9.172562701824643e-09;
    constexpr double MAGIC = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to an integer
    const double d = f == topf ? 0.0 : (double)f - top;
    const double t = fma(d, scale, MAGIC);
    const double r = fma(d, scale, MAGIC - t);
    const int n = __double2loint(t);
    const double poly = fma(fma(fma(fma(A4, r, A3), r, A2), r, A1), r, 1.0);
    uint32_t lo, hi;
    if constexpr (ALL) {
      lo = __shfl_sync(~0u, tab_lo, n & 31);
      hi = __shfl_sync(~0u, tab_hi, n & 31);
    } else {
      lo = (uint32_t)__double2loint(sh.table[n & 31]);
      hi = (uint32_t)__double2hiint(sh.table[n & 31]);
    }
    const double power = __hiloint2double((int)hi + ((n >> 5) << 20), (int)lo);
    const bool some = d * scale > -32.0 * 46;  // less rounds to nothing
    exact = some ? poly * power : 0.0;
    return some ? (uint64_t)__double_as_longlong(fma(poly, power, ROUND52)) & 0xfffffffffffffull : 0ull;
  }
  template <bool ALL>
  __device__ __forceinline__ uint64_t weight(float f) const {
    double e;
    return weight<ALL>(f, e);
  }
  __device__ __forceinline__ uint32_t off_of(float f) const {
    return (uint32_t)kmax - (uint32_t)order_of(f);
  }
  // Bin of a logit, rising along the order; BINS and more: below all bins.  `rest`:
  // the logit's distance from the middle of its bin.
  __device__ __forceinline__ uint32_t bin_of(float f, float& rest) const {
    const float d = f - topf;
    const float t = fmaf(d, octaves, 8388608.f);  // 2^23: rounds to an integer
    rest = fmaf(d, octaves, 8388608.f - t);
    return d < lowest ? BINS : __float_as_uint(t) & 0x7fffffu;
  }
  __device__ __forceinline__ uint32_t bin_of(float f) const {
    float rest;
    return bin_of(f, rest);
  }

  // fn(chunk, index of its first element, whether it exists) for the warp's chunks,
  // every lane of the warp at once.
  template <typename F>
  __device__ __forceinline__ void each(F fn) const {
    const int end = min(nchunks, (warp + 1) * segment);
    for (int c0 = warp * segment; c0 < end; c0 += 32) {
      const int c = c0 + lane;
      Chunk<T> x;
      x.raw = make_uint4(0, 0, 0, 0);
      if (c < end) x = chunk(c);
      fn(x, first + c * N, c < end);
    }
  }

  // Sum of v over the cluster's warps, and of the warps before each; `mine` is
  // this warp's.  Every thread gets the total.
  __device__ uint64_t exchange(uint64_t mine) {
    const int s = slot;
    slot = slot == 2 ? 0 : slot + 1;
    if (lane < ctas)
      st_remote64(lpc::mapa_shared(lpc::smem_u32(&sh.sums[s][rank * WARPS + warp]), lane), mine);
    lpc::cluster_sync();
    uint64_t v = 0;
    for (int i = lane; i < ctas * WARPS; i += 32) v += sh.sums[s][i];
    return warp_sum(v);
  }

  // This warp's sum of fn(value, index).
  template <typename F>
  __device__ uint64_t sum_of(F fn) const {
    uint64_t mine = 0;
    each([&](const Chunk<T>& x, int at, bool in) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const uint64_t v = fn(x.get(i), at + i);
        mine += in ? v : 0ull;
      }
    });
    return warp_sum(mine);
  }

  // Lowest row index at which the running sum of fn(value, index) exceeds
  // target(total); `mine` is this warp's sum.  Every thread of the cluster gets it.
  // total > target.
  template <typename F, typename G>
  __device__ int locate(uint64_t mine, F fn, G target_of) {
    const int s = slot;
    const uint64_t total = exchange(mine);
    const uint64_t target = target_of(total);
    uint64_t upto = 0;  // the warps before this one
    for (int i = lane; i < rank * WARPS + warp; i += 32) upto += sh.sums[s][i];
    upto = warp_sum(upto);
    const int f = found_slot;
    found_slot ^= 1;
    if (upto <= target && target < upto + mine) {
      bool done = false;
      each([&](const Chunk<T>& x, int at, bool in) {
        if (done) return;
        uint64_t part = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const uint64_t v = fn(x.get(i), at + i);
          part += in ? v : 0ull;
        }
        const uint64_t scan = warp_scan(part, lane);
        const unsigned over = __ballot_sync(~0u, upto + scan > target);
        if (over) {
          done = true;
          const int who = __ffs(over) - 1;
          // its elements once more, by all lanes together
          uint64_t run = upto + scan - part;
          int found = -1;
#pragma unroll
          for (int i = 0; i < N; ++i) {
            run += fn(x.get(i), at + i);
            if (found < 0 && run > target) found = at + i;
          }
          if (lane == who)
            for (int r = 0; r < ctas; ++r)
              st_remote64(lpc::mapa_shared(lpc::smem_u32(&sh.found[f]), r), (uint64_t)found);
        } else {
          upto += (uint64_t)__shfl_sync(~0u, (uint32_t)scan, 31) |
                  ((uint64_t)__shfl_sync(~0u, (uint32_t)(scan >> 32), 31) << 32);
        }
      });
    }
    lpc::cluster_sync();
    return (int)sh.found[f];
  }

  // Histogram over the bins: of counts, or of fp32 weights in units of 2^-15 of a bin's
  // middle.  Every thread gets the cluster's bins 4 tid to 4 tid + 3.
  template <bool MASS>
  __device__ void histogram(uint64_t (&v)[4]) {
    uint32_t* h = hist[0];
    for (int i = threadIdx.x; i < BINS; i += THREADS) h[i] = 0u;
    if (threadIdx.x == 0) sh.listed = 0;
    __syncthreads();
    each([&](const Chunk<T>& x, int, bool in) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float rest;
        const uint32_t bin = bin_of(x.get(i), rest);
        // 2^15 * 2^(-rest / OCTAVE), by two terms of the series (2e-7 off)
        const float e = rest * (-0.69314718f / OCTAVE);
        const float m = fmaf(fmaf(e, 0.5f, 1.f) * e, 32768.f, 32768.f + 8388608.f);
        if (in && bin < BINS) atomicAdd(h + bin, MASS ? __float_as_uint(m) & 0x7fffffu : 1u);
      }
    });
    lpc::cluster_sync();
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = 0;
    const uint32_t at = lpc::smem_u32(h + 4 * threadIdx.x);
    for (int r = 0; r < ctas; ++r) {
      const uint4 l = ld_remote16(lpc::mapa_shared(at, r));
      v[0] += l.x, v[1] += l.y, v[2] += l.z, v[3] += l.w;
    }
  }

  // The bin whose running count first exceeds `target` (-1: none), from each thread's four;
  // sh.cross_before and sh.cross_in: the count before it and in it.
  __device__ int crossing(const uint64_t (&v)[4], uint64_t target) {
    const uint64_t own = v[0] + v[1] + v[2] + v[3];
    uint64_t run = warp_scan(own, lane);
    if (lane == 31) sh.scan[warp] = run;
    if (threadIdx.x == 0) sh.cross_bin = -1;
    __syncthreads();
    for (int i = 0; i < warp; ++i) run += sh.scan[i];
    run -= own;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (run <= target && target < run + v[i]) {
        sh.cross_bin = 4 * (int)threadIdx.x + i;
        sh.cross_before = run;
        sh.cross_in = v[i];
      }
      run += v[i];
    }
    __syncthreads();
    return sh.cross_bin;
  }
  // The bins between which the running sum of the weights passes p * (their sum), with
  // SLACK on either side: sh.window.  False: it may pass below all bins.
  __device__ bool window(const uint64_t (&v)[4], float p) {
    double w[4], own = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = (double)v[i] * (double)exp2f(-(float)(4 * (int)threadIdx.x + i) / OCTAVE);
      own += w[i];
    }
    double run = own;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const double o = __shfl_up_sync(~0u, run, d);
      if (lane >= d) run += o;
    }
    double* scan = reinterpret_cast<double*>(sh.scan);
    if (lane == 31) scan[warp] = run;
    if (threadIdx.x == 0) sh.window[0] = sh.window[1] = BINS;
    __syncthreads();
    double total = 0, others = 0;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) {
      if (i < warp) others += scan[i];
      total += scan[i];
    }
    run += others - own;
    const double lo = ((double)p - SLACK) * total, hi = ((double)p + SLACK) * total;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool first = threadIdx.x == 0 && i == 0;
      if ((first || run <= lo) && lo < run + w[i]) atomicMin(&sh.window[0], 4 * threadIdx.x + i);
      if ((first || run <= hi) && hi < run + w[i]) atomicMin(&sh.window[1], 4 * threadIdx.x + i);
      run += w[i];
    }
    __syncthreads();
    return sh.window[0] < BINS && sh.window[1] < BINS;
  }

  // The elements for which want(value, index) puts them on this CTA's list (in hist[1]);
  // LIST of them at most are kept, all are counted.
  __device__ __forceinline__ void list(bool want, float f, int at) {
    const unsigned who = __ballot_sync(~0u, want);
    if (!who) return;
    uint32_t base = 0;
    if (lane == __ffs(who) - 1) base = atomicAdd(&sh.listed, (uint32_t)__popc(who));
    base = __shfl_sync(~0u, base, __ffs(who) - 1) + (uint32_t)__popc(who & ((1u << lane) - 1u));
    if (want && base < (uint32_t)LIST)
      reinterpret_cast<Entry*>(hist[1])[base] = Entry{(uint32_t)at, off_of(f)};
  }
  // The cluster's lists, with their weights, in this CTA's hist[0]; their length, or -1
  // where they are longer than LIST.  The lists are complete in every CTA.
  struct Listed {
    uint64_t place, weight;
  };
  __device__ int gather() {
    lpc::cluster_sync();
    int total = 0, start = 0;
    const uint32_t counts = lpc::smem_u32(&sh.listed);
    for (int r = 0; r < ctas; ++r) total += (int)ld_remote(lpc::mapa_shared(counts, r));
    if (total > LIST) return -1;
    Listed* all = reinterpret_cast<Listed*>(hist[0]);
    const uint32_t from = lpc::smem_u32(hist[1]);
    for (int r = 0; r < ctas; ++r) {
      const int n = (int)ld_remote(lpc::mapa_shared(counts, r));
      const uint32_t list = lpc::mapa_shared(from, r);
      for (int i = threadIdx.x; i < n; i += THREADS) {
        Entry e;
        e.index = ld_remote(list + 8u * i);
        e.off = ld_remote(list + 8u * i + 4u);
        all[start + i] = Listed{place_of(e), weight<false>(value_of((int32_t)((uint32_t)kmax - e.off)))};
      }
      start += n;
    }
    __syncthreads();
    return total;
  }

  // One round of the select: sums of `measure` in bins of 2^shift of the offset
  // from the largest, over offsets [lo, hi]; finds the first bin whose running
  // sum, begun at `above`, exceeds target(above + total).  False: none does.
  template <bool MASS, typename G>
  __device__ bool round(uint32_t lo, uint32_t hi, int shift, uint64_t above, G target_of) {
    uint32_t* h = hist[turn];
    turn ^= 1;
    for (int i = threadIdx.x; i < BINS * (MASS ? 2 : 1); i += THREADS) h[i] = 0u;
    __syncthreads();
    for (int c = warp * segment + lane; c < min(nchunks, (warp + 1) * segment); c += 32) {
      const Chunk<T> x = chunk(c);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float f = x.get(i);
        const uint32_t off = (uint32_t)kmax - (uint32_t)order_of(f);
        if (off - lo <= hi - lo && f != -INFINITY) {
          const uint32_t bin = (off - lo) >> shift;
          if constexpr (MASS) {
            const uint64_t w = weight<false>(f);
            if (w) {
              const uint32_t was = atomicAdd(h + bin, (uint32_t)w);
              const uint32_t up = (uint32_t)(w >> 32) + (was + (uint32_t)w < was ? 1u : 0u);
              if (up) atomicAdd(h + BINS + bin, up);
            }
          } else {
            atomicAdd(h + bin, 1u);
          }
        }
      }
    }
    if (threadIdx.x == 0) sh.cross_bin = -1;
    lpc::cluster_sync();
    // four bins a thread, summed over the cluster
    uint64_t v[4] = {0, 0, 0, 0};
    const uint32_t at = lpc::smem_u32(h + 4 * threadIdx.x);
    for (int r = 0; r < ctas; ++r) {
      const uint32_t from = lpc::mapa_shared(at, r);
      const uint4 l = ld_remote16(from);
      v[0] += l.x, v[1] += l.y, v[2] += l.z, v[3] += l.w;
      if constexpr (MASS) {
        const uint4 u = ld_remote16(from + BINS * 4);
        v[0] += (uint64_t)u.x << 32, v[1] += (uint64_t)u.y << 32;
        v[2] += (uint64_t)u.z << 32, v[3] += (uint64_t)u.w << 32;
      }
    }
    const uint64_t own = v[0] + v[1] + v[2] + v[3];
    uint64_t run = warp_scan(own, lane);
    if (lane == 31) sh.scan[warp] = run;
    __syncthreads();
    uint64_t others = 0, total = 0;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) {
      const uint64_t s = sh.scan[i];
      total += s;
      if (i < warp) others += s;
    }
    const uint64_t target = target_of(above + total);
    run += above + others - own;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (run <= target && target < run + v[i]) {
        sh.cross_bin = 4 * (int)threadIdx.x + i;
        sh.cross_before = run;
        sh.cross_in = v[i];
      }
      run += v[i];
    }
    __syncthreads();
    return sh.cross_bin >= 0;
  }
};

struct Count { static constexpr bool value = false; };
struct Mass { static constexpr bool value = true; };

static_assert(BINS == 4 * THREADS, "four bins a thread");

// The token of a row of which the list (n elements, in hist[0]) holds the first top_k of
// the order.  One CTA, every thread.
template <typename T>
__device__ void draw_from_list(Row<T>& row, int n, int top_k, float top_p, double least, float u,
                               int64_t* out) {
  Shared& sh = row.sh;
  typename Row<T>::Listed* all = reinterpret_cast<typename Row<T>::Listed*>(row.hist[0]);
  static_assert(LIST <= THREADS, "an element a thread");
  const int i = threadIdx.x;
  const bool in = i < n;
  const uint64_t place = in ? all[i].place : ~0ull, w = in ? all[i].weight : 0ull;
  uint64_t run = 0;
  int rank = 0;
  if (in)
    for (int j = 0; j < n; ++j)
      if (all[j].place < place) {
        run += all[j].weight;
        ++rank;
      }
  bool stays = in && rank < top_k;
  auto total = [&](uint64_t v) {
    v = warp_sum(v);
    __syncthreads();
    if (row.lane == 0) sh.scan[row.warp] = v;
    __syncthreads();
    uint64_t s = 0;
#pragma unroll
    for (int x = 0; x < WARPS; ++x) s += sh.scan[x];
    return s;
  };
  if (top_p < 1.f) {
    const uint64_t target = part_of(top_p, total(stays ? w : 0ull));
    stays = stays && run <= target;
  }
  double exact = 0;
  if (in) row.template weight<false>(value_of((int32_t)((uint32_t)row.kmax - (uint32_t)(place >> 32))), exact);
  stays = stays && exact >= least;
  const uint64_t target = part_of(u, total(stays ? w : 0ull));
  // by index from here on
  if (in) all[i].place = (uint64_t)(uint32_t)place << 32 | (stays ? 1u : 0u);
  __syncthreads();
  if (stays) {
    uint64_t before = 0;
    for (int j = 0; j < n; ++j)
      if ((uint32_t)(all[j].place >> 32) < (uint32_t)place && (all[j].place & 1u)) before += all[j].weight;
    if (before <= target && target < before + w) *out = (int64_t)(uint32_t)place;
  }
}

template <typename T>
__global__ void __launch_bounds__(THREADS, 2) sample_kernel(const Args a) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ Shared sh;
  constexpr int N = Chunk<T>::N;
  Row<T> row(a, sh);
  row.rank = (int)lpc::cluster_ctarank();
  uint32_t ctas;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
  row.ctas = (int)ctas;
  row.warp = threadIdx.x >> 5;
  row.lane = threadIdx.x & 31;
  row.hist[0] = reinterpret_cast<uint32_t*>(smem);
  row.hist[1] = reinterpret_cast<uint32_t*>(smem + HIST_BYTES);
  row.chunks = reinterpret_cast<uint4*>(smem + 2 * HIST_BYTES);
  const int64_t r = blockIdx.x / ctas;

  // ---- the share of the row, and the first of the order ----
  const int begin = min(row.rank * a.slice, a.vocab);
  const int count = min(a.slice, a.vocab - begin);
  const T* src = static_cast<const T*>(a.logits) + r * a.row_stride + begin;
  const int skew = (int)((reinterpret_cast<uintptr_t>(src) & 15u) / sizeof(T));
  row.first = begin - skew;
  row.begin = begin;
  row.end = begin + max(count, 0);
  row.nchunks = count > 0 ? (skew + count + N - 1) / N : 0;
  row.segment = ((row.nchunks + WARPS - 1) / WARPS + 31) / 32 * 32;
  lpc::pdl_wait();
  const float u = a.uniforms[r];
  const float temperature = a.temperature ? a.temperature[r] : a.t;
  const float top_p = a.top_p ? a.top_p[r] : a.p;
  const float min_p = a.min_p ? a.min_p[r] : a.m;
  const int32_t top_k = a.top_k ? a.top_k[r] : a.k;
  float best = -INFINITY;
  int best_at = 0;
  const uint4* vec = reinterpret_cast<const uint4*>(src - skew);
  const int seg_end = min(row.nchunks, (row.warp + 1) * row.segment);
  for (int c0 = row.warp * row.segment + row.lane; c0 < seg_end; c0 += 32 * BATCH) {
    Chunk<T> xs[BATCH];
#pragma unroll
    for (int j = 0; j < BATCH; ++j) {
      const int c = c0 + 32 * j;
      const int e0 = c * N - skew;  // share index of the chunk's first element
      if (c < seg_end && e0 >= 0 && e0 + N <= count) xs[j].raw = lpc::ld_dep16(vec + c);
    }
#pragma unroll
    for (int j = 0; j < BATCH; ++j) {
      const int c = c0 + 32 * j;
      if (c >= seg_end) break;
      const int e0 = c * N - skew;
      Chunk<T> x = xs[j];
      if (e0 < 0 || e0 + N > count) {
        alignas(16) T part[N];
        for (int i = 0; i < N; ++i)
          part[i] = e0 + i >= 0 && e0 + i < count ? src[e0 + i] : Num<T>::from_f(-INFINITY);
        x.raw = *reinterpret_cast<const uint4*>(part);
      }
      bool nan = false;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float f = x.get(i);
        nan |= f != f;
        if (f > best) {
          best = f;
          best_at = begin + e0 + i;
        }
      }
      if (nan) {
        alignas(16) T part[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float f = x.get(i);
          part[i] = Num<T>::from_f(f != f ? -INFINITY : f);
        }
        x.raw = *reinterpret_cast<const uint4*>(part);
      }
      row.chunks[c] = x.raw;
    }
  }
  uint64_t mine = ((uint64_t)((uint32_t)order_of(best) ^ 0x80000000u) << 32) | (uint32_t)~best_at;
#pragma unroll
  for (int m = 16; m; m >>= 1) mine = max(mine, shfl_xor64(mine, m));
  // every CTA of the cluster has to have started before its memory is written
  lpc::cluster_sync();
  if (row.lane < row.ctas)
    st_remote64(lpc::mapa_shared(lpc::smem_u32(&sh.sums[0][row.rank * WARPS + row.warp]), row.lane),
                mine);
  row.slot = 1;
  lpc::cluster_sync();
  mine = 0;
  for (int i = row.lane; i < row.ctas * WARPS; i += 32) mine = max(mine, sh.sums[0][i]);
#pragma unroll
  for (int m = 16; m; m >>= 1) mine = max(mine, shfl_xor64(mine, m));

  row.kmax = (int32_t)((uint32_t)(mine >> 32) ^ 0x80000000u);
  const int32_t kmax = row.kmax;
  const bool bad = !(temperature >= 0.f && temperature < INFINITY) || !(u >= 0.f && u < 1.f) ||
                   !(top_p > 0.f && top_p <= 1.f) || !(min_p >= 0.f && min_p <= 1.f);
  const bool none = kmax == order_of(-INFINITY);
  if (bad || none || temperature == 0.f) {  // the same for the whole cluster
    if (row.rank == 0 && threadIdx.x == 0) {
      if (bad) atomicOr(&g_sample_status, LPC_DEV_ERR_BOUNDS);
      a.out[r] = bad || none ? -1 : (int64_t)(uint32_t)~(uint32_t)mine;
    }
    return;
  }
  row.topf = value_of(kmax);
  row.top = (double)row.topf;
  const double per_unit = 1.4426950408889634074 / (double)temperature;
  row.scale = 32.0 * per_unit;
  row.octaves = (float)(-OCTAVE * per_unit);
  row.lowest = (float)(-(BINS - 1) / (OCTAVE * per_unit));
  if (threadIdx.x < 32) sh.table[threadIdx.x] = exp2((double)threadIdx.x / 32.0) * FIXED;
  __syncthreads();
  row.tab_lo = (uint32_t)__double2loint(sh.table[row.lane]);
  row.tab_hi = (uint32_t)__double2hiint(sh.table[row.lane]);
  // where fp32 has the bins: not for infinities, nor for temperatures that nobody uses
  const bool binned = fabsf(row.topf) < 1e30f && per_unit < 1e25 && per_unit > 1e-25;
  const double least = (double)min_p * FIXED;

  // ---- the place in the order up to which logits stay: offsets from the
  // largest below `cut`, and `ties` of the ones at it (-1: all) ----
  constexpr int G = GRAIN<T>;
  const uint32_t off_all = (uint32_t)kmax - (uint32_t)order_of(-INFINITY) - 1u;
  uint32_t cut = off_all;
  uint64_t ties = ~0ull, present = ~0ull;  // kept at `cut`, and all there are
  // offset, sum before it and sum at it of the first value at which the
  // running sum exceeds the target
  auto select = [&](auto mass, uint32_t last, auto target_of, uint32_t& off, uint64_t& before,
                    uint64_t& in) -> bool {
    constexpr bool MASS = decltype(mass)::value;
    uint32_t lo = 0, hi = last;
    uint64_t above = 0, target = 0;
    bool known = false;
    for (int shift = 21;;) {
      auto goal = [&](uint64_t total) { return known ? target : (target = target_of(total)); };
      if (!row.template round<MASS>(lo, hi, shift, above, goal)) return false;
      known = true;
      lo += (uint32_t)sh.cross_bin << shift;
      above = sh.cross_before;
      if (shift == G) break;
      hi = min(hi, lo + ((1u << shift) - 1u));
      shift = max(G, shift - 11);
    }
    off = lo;
    before = above;
    in = sh.cross_in;
    return true;
  };
  if (top_k > 0 && top_k < a.vocab) {
    // at most LIST elements in the bins down to the one of the last: all on the list
    uint64_t v[4];
    if (top_k <= LIST && binned) {
      row.template histogram<false>(v);
      const int bin = row.crossing(v, (uint64_t)top_k - 1u);
      if (bin >= 0 && sh.cross_before + sh.cross_in <= (uint64_t)LIST) {
        row.each([&](const Chunk<T>& x, int at, bool in) {
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const float f = x.get(i);
            row.list(in && row.bin_of(f) <= (uint32_t)bin, f, at + i);
          }
        });
        const int n = row.gather();
        lpc::cluster_sync();  // the lists have been read: the others may go
        if (row.rank == 0) draw_from_list(row, n, top_k, top_p, least, u, a.out + r);
        return;
      }
    }
    lpc::cluster_sync();  // histograms have been read
    uint64_t before, in;
    if (select(Count{}, cut, [&](uint64_t) { return (uint64_t)top_k - 1u; }, cut, before, in)) {
      ties = (uint64_t)top_k - before;
      present = in;
    }
    lpc::cluster_sync();
  }
  uint64_t mine_kept = 0;  // this warp's sum of the weights that stay, where it is known
  bool known = false;
  int last = a.vocab;      // highest index that stays of those at `cut`
  if (top_p < 1.f && ties == ~0ull && binned) {
    uint64_t v[4];
    row.template histogram<true>(v);
    if (row.window(v, top_p)) {
      const uint32_t w0 = sh.window[0], w1 = sh.window[1];
      uint64_t all = 0, above = 0, kept = 0;
      row.each([&](const Chunk<T>& x, int at, bool in) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float f = x.get(i);
          double exact;
          uint64_t w = row.template weight<true>(f, exact);
          w = in ? w : 0ull;
          const uint32_t bin = row.bin_of(f);
          all += w;
          above += bin < w0 ? w : 0ull;
          kept += bin < w0 && exact >= least ? w : 0ull;
          row.list(in && bin >= w0 && bin <= w1, f, at + i);
        }
      });
      mine_kept = warp_sum(kept);
      const uint64_t total = row.exchange(warp_sum(all));
      const uint64_t before = row.exchange(warp_sum(above));
      const int n = row.gather();
      if (n >= 0) {
        const uint64_t target = part_of(top_p, total);
        if (threadIdx.x == 0) sh.cut = 0;
        __syncthreads();
        typename Row<T>::Listed* all_listed = reinterpret_cast<typename Row<T>::Listed*>(row.hist[0]);
        for (int i = threadIdx.x; i < n; i += THREADS) {
          const uint64_t place = all_listed[i].place;
          uint64_t run = before;
          for (int j = 0; j < n; ++j)
            if (all_listed[j].place < place) run += all_listed[j].weight;
          if (run <= target) atomicMax(&sh.cut, (unsigned long long)place + 1ull);
        }
        __syncthreads();
        const uint64_t place = sh.cut;  // 1 more than the last that stays
        if (place) {
          cut = (uint32_t)((place - 1) >> 32);
          last = (int)(uint32_t)(place - 1);
          // the list's elements that stay, to the warps that have them
          uint64_t more = 0;
          const int lo = max(row.begin, row.first + row.warp * row.segment * N);
          const int hi = min(row.end, row.first + (row.warp + 1) * row.segment * N);
          for (int i = row.lane; i < n; i += 32) {
            const uint64_t e = all_listed[i].place;
            const int at = (int)(uint32_t)e;
            double exact;
            row.template weight<false>(value_of((int32_t)((uint32_t)kmax - (uint32_t)(e >> 32))), exact);
            if (e < place && at >= lo && at < hi && exact >= least) more += all_listed[i].weight;
          }
          mine_kept += warp_sum(more);
          known = true;
        }
      }
    }
    lpc::cluster_sync();  // histograms and lists have been read
  }
  if (top_p < 1.f && !known) {
    // of the last value's weight only `ties` count
    const uint64_t w_cut = ties == ~0ull ? 0 : row.template weight<false>(value_of((int32_t)((uint32_t)kmax - cut)));
    const uint64_t extra = ties == ~0ull ? 0 : (present - ties) * w_cut;
    uint32_t off;
    uint64_t before, in;
    uint64_t target = 0;
    if (select(Mass{}, cut,
               [&](uint64_t total) { return target = part_of(top_p, total - extra); }, off, before,
               in)) {
      const uint64_t w = row.template weight<false>(value_of((int32_t)((uint32_t)kmax - off)));
      cut = off;
      ties = (target - before) / w + 1u;
      present = in / w;
    }
  }
  if (!known && ties < present) {
    auto tied = [&](float f, int) -> uint64_t { return row.off_of(f) == cut && f != -INFINITY; };
    last = row.locate(row.sum_of(tied), tied, [&](uint64_t) { return ties - 1u; });
  }
  auto stays = [&](float f, int at) -> uint64_t {
    const uint32_t off = row.off_of(f);
    double exact;
    const uint64_t w = row.template weight<true>(f, exact);
    return off > cut || (off == cut && at > last) || !(exact >= least) ? 0ull : w;
  };
  if (!known) mine_kept = row.sum_of(stays);
  const int token = row.locate(mine_kept, stays, [&](uint64_t total) { return part_of(u, total); });
  if (row.rank == 0 && threadIdx.x == 0) a.out[r] = token;
}

template <typename T>
int launch(const Args& args, int64_t rows, int ctas, cudaStream_t s) {
  static std::atomic<uint64_t> mask{0};
  const int most = 2 * HIST_BYTES + MAX_SLICE_BYTES + 32;
  if (int rc = lpc::once_per_device_smem((const void*)sample_kernel<T>, most, mask)) return rc;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = lpc::use_pdl() ? 1 : 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * ctas));
  cfg.blockDim = dim3(THREADS);
  // a chunk more than the share: it may begin inside one
  cfg.dynamicSmemBytes = 2 * HIST_BYTES + ((size_t)args.slice * sizeof(T) + 15) / 16 * 16 + 16;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, sample_kernel<T>, args);
  if (e != cudaSuccess) {
    lpc::set_error("sample_tokens: launch failed: %s", cudaGetErrorString(e));
    return LPC_ERR_CUDA;
  }
  return lpc::check_launch("sample_tokens");
}

}  // namespace

extern "C" int lpc_sample_tokens(const void* logits, int64_t row_stride, const float* uniforms,
                                 const float* temperature, const int32_t* top_k,
                                 const float* top_p, const float* min_p, float temperature_all,
                                 int32_t top_k_all, float top_p_all, float min_p_all, int64_t* out,
                                 int64_t rows, int64_t vocab, int dtype, void* stream) {
  using namespace lpc;
  const int es = dtype_size(dtype);
  if (!es) {
    set_error("sample_tokens: unsupported dtype %d", dtype);
    return LPC_ERR_UNSUPPORTED;
  }
  if (rows < 0 || vocab <= 0 || (rows > 1 && row_stride < vocab)) {
    set_error("sample_tokens: invalid sizes (rows=%lld vocab=%lld row_stride=%lld)",
              (long long)rows, (long long)vocab, (long long)row_stride);
    return LPC_ERR_INVALID;
  }
  if ((!temperature && !(temperature_all >= 0.f && temperature_all < INFINITY)) ||
      (!top_p && !(top_p_all > 0.f && top_p_all <= 1.f)) ||
      (!min_p && !(min_p_all >= 0.f && min_p_all <= 1.f))) {
    set_error("sample_tokens: temperature must be >= 0, top_p in (0, 1], min_p in [0, 1]");
    return LPC_ERR_INVALID;
  }
  if (vocab > (int64_t)MAX_CLUSTER * MAX_SLICE_BYTES / es || rows > 0x7fffffffLL / MAX_CLUSTER) {
    set_error("sample_tokens: at most %lld logits a row of this type and %lld rows",
              (long long)MAX_CLUSTER * MAX_SLICE_BYTES / es, 0x7fffffffLL / MAX_CLUSTER);
    return LPC_ERR_UNSUPPORTED;
  }
  if (rows == 0) return LPC_OK;
  if (!logits || !uniforms || !out) {
    set_error("sample_tokens: null pointer");
    return LPC_ERR_INVALID;
  }
  if (reinterpret_cast<uintptr_t>(logits) % es) {
    set_error("sample_tokens: logits are not aligned to their type");
    return LPC_ERR_INVALID;
  }
  // CTAs a row: what brings its share to 64 KB (two CTAs an SM then overlap
  // reading and computing); more while the rows leave SMs idle and a warp still
  // has a kilobyte
  int ctas = 1;
  while (ctas < MAX_CLUSTER && vocab * es > (int64_t)ctas * SLICE_BYTES) ctas *= 2;
  while (ctas < MAX_CLUSTER && rows * ctas * 2 <= current_device_sms() &&
         vocab * es > (int64_t)ctas * WARPS * 512)
    ctas *= 2;
  Args args;
  args.logits = logits;
  args.row_stride = row_stride;
  args.vocab = (int)vocab;
  // a multiple of 16 bytes: every share begins as the row does
  const int64_t unit = 16 / es;
  args.slice = (int)(((vocab + ctas - 1) / ctas + unit - 1) / unit * unit);
  args.uniforms = uniforms;
  args.temperature = temperature;
  args.top_k = top_k;
  args.top_p = top_p;
  args.min_p = min_p;
  args.t = temperature_all;
  args.k = top_k_all;
  args.p = top_p_all;
  args.m = min_p_all;
  args.out = out;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == LPC_DTYPE_F32) return launch<float>(args, rows, ctas, s);
  if (dtype == LPC_DTYPE_BF16) return launch<__nv_bfloat16>(args, rows, ctas, s);
  return launch<__half>(args, rows, ctas, s);
}
