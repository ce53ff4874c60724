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
//     value and, among equals, an index.  A pass then compares floats: bins, min-p
//     and the like are turned into the smallest float that passes.
//   * A histogram over 2048 bins of 1/64 octave of the weight, of counts or of fp32
//     weights, says in which bins the place lies; their few elements go to a list and
//     are ranked exactly, by pairs.  With top-k the list has all that is kept, and the
//     rest is done on it.
//   * Where the list would not hold them (many equal logits, thousands kept by top-k,
//     places beyond the bins), the place is found by radix select: histograms over 11
//     bits of the order-preserving integer of the value, of counts or of integer
//     weights.
//   * The token: sums of each warp's stretch, a scan over the cluster's warps, and
//     the warp whose stretch holds the border walks it.
// Bound: issue slots (65 % of them at 512 rows; fp64 17 %).  512 rows of 32,000 bf16 with
// top-p 57 us, 75 instructions an element: a row takes 40,000 cycles with a second one on its
// SM, 4,000 of them loads, 10,000 the histogram, 14,500 the weights' pass, 5,000 the token.
// Without filters 35 (43 instructions), top-k 50 38 (33), greedy 14 (17); 256 rows of 128,256
// 77, with top-p 193, as some rows' lists overflow.  Two CTAs an SM leave 64 registers; what
// does not fit, 44 to 92 bytes of one-CTA rows and 176 to 192 of clusters', is spilled.
// fp32 weights first and the integers only near a border gained 15 % there and lost 35 % on
// flat rows (registers, rows that need both); 1024 threads a row were slower.
#include <atomic>
#include <type_traits>

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

// 512 threads and shares of 84 KB at most: two CTAs an SM, so that one reads while the other
// computes
constexpr int THREADS = 512;
constexpr int WARPS = THREADS / 32;
constexpr int MAX_CLUSTER = 8;
constexpr int BINS = 2048;                       // 11 bits a round
constexpr int MINE = BINS / THREADS;             // bins a thread, at most
constexpr int HIST_BYTES = BINS * 8;             // low and high words of a bin's sum
constexpr int LIST = 1024;                       // elements of a list
constexpr int PAIRS = 512;                       // elements that are ranked by pairs: of top-k
constexpr int SHORT = 128;                       // and of top-p; beyond it by search
constexpr int LIST_BYTES = LIST * 8;
constexpr double FIXED = 17592186044416.0;       // 2^44
constexpr double ROUND52 = 4503599627370496.0;   // 2^52: adding it rounds to an integer
constexpr int OCTAVE = 64;                       // bins an octave of the weight
// What the histogram may be off, relative to all weights, in a running sum and once more in
// p * (their sum): its elements by 2^-16 of rounding and 4e-6 of fp32 arithmetic (3.9e-5 in
// all), their fp32 sums by 33 roundings on the way (a thread's 4 bins, 5 steps of a scan, 16
// warps, 8 CTAs; 4e-6 in all) and exp2f's 2 ulp; 5e-5 covers them.  Then what lies below its
// 32 octaves, at most 2^-32 of the largest an element.  (By 5e-4 for all rows 256 of 128,256
// with top-p 0.95 took 250 us, so 197: more of them have a list that holds their window.)
__device__ __forceinline__ float slack_of(int vocab) { return 5e-5f + (float)vocab * 2.33e-10f; }
constexpr int SLICE_BYTES = 84 * 1024;           // preferred share of a CTA
constexpr int LONG = 24000;                      // elements of a row worth several CTAs
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
  static __device__ __forceinline__ uint4 nothing() {  // -inf
    constexpr uint32_t w = sizeof(T) == 4 ? 0xff800000u : GRAIN<T> == 16 ? 0xff80ff80u : 0xfc00fc00u;
    return make_uint4(w, w, w, w);
  }
  // The largest; NaN if there is one.
  __device__ __forceinline__ float largest() const {
    if constexpr (sizeof(T) == 4) {
      return max_nan(max_nan(get(0), get(1)), max_nan(get(2), get(3)));
    } else {
      const uint32_t m = max2_nan(max2_nan(raw.x, raw.y), max2_nan(raw.z, raw.w));
      Chunk<T> x;
      x.raw.x = m;
      return max_nan(x.get(0), x.get(1));
    }
  }
  static __device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
  }
  static __device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b) {
    uint32_t d;
    if constexpr (GRAIN<T> == 16)
      asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    else
      asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
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
// The two halves of a barrier of all threads of the cluster.
__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint64_t warp_min(uint64_t v) {  // over the warp
#pragma unroll
  for (int m = 16; m; m >>= 1) v = min(v, shfl_xor64(v, m));
  return v;
}
__device__ __forceinline__ void atom_add(uint32_t addr, uint32_t v) {
  asm volatile("red.shared.add.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void st_remote64(uint32_t addr, uint64_t v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}

struct Entry {  // an element in the order: by offset from the largest, then by index
  uint32_t index, off;
};
struct Listed {
  uint64_t place, weight;  // place: offset, index
};
static_assert(LIST * (int)sizeof(Listed) <= HIST_BYTES && LIST * (int)sizeof(Entry) <= LIST_BYTES, "");

struct Shared {
  double table[32];                       // 2^44 * 2^(j/32)
  uint64_t sums[3][MAX_CLUSTER * WARPS];  // written by every CTA of the cluster
  uint64_t found[2];                      // a located index, written by its finder
  uint64_t scan[WARPS];
  uint64_t parts[2][MAX_CLUSTER];         // sums of each CTA's bins
  uint64_t cross[3];                      // the crossing bin (~0: none), the sum before it and in it
  uint64_t last;                          // 1 more than the place of the last that stays (0: none)
  uint64_t window[2];                     // first and last bin that may hold the place
  uint32_t listed;                        // elements that this CTA put on its list
};

// ONE: a CTA a row, else a cluster.
template <typename T, bool ONE>
class Row {
 public:
  static constexpr int N = Chunk<T>::N;
  static constexpr int CTAS = ONE ? 1 : MAX_CLUSTER;  // at most
  Shared& sh;
  uint4* chunks;              // this CTA's share of the row, -inf outside it
  uint32_t* hist;             // BINS low words, BINS high words; or the cluster's list
  Entry* own_list;
  int rank, ctas, warp, lane;
  int nchunks, segment;       // chunks of this CTA; of a warp (a multiple of 32)
  int first;                  // row index of element 0 of chunk 0 (may lie before the share)
  int begin, end;             // row indexes of the share
  int32_t kmax;               // order_of(largest)
  float topf, floorf;         // largest; a logit that weighs nothing (2^-60)
  double top, scale;          // largest; 32 log2(e) / temperature
  float octaves, lowest;      // -OCTAVE log2(e) / temperature; offset of the last bin
  uint32_t tab_lo, tab_hi;    // table entry `lane`, its index taken off the exponent
  int slot = 0;               // which sums the next exchange takes
  int found_slot = 0, part_slot = 0;

  __device__ explicit Row(Shared& s) : sh(s) {}

  // Every thread of the cluster.
  __device__ __forceinline__ void sync() const {
    if constexpr (ONE) __syncthreads();
    else lpc::cluster_sync();
  }
  // In CTA r's shared memory, at the place of `where` in this one's.  The way over the
  // cluster costs several times a plain access.
  __device__ __forceinline__ void store(uint64_t* where, int r, uint64_t v) const {
    if (ONE || r == rank) *where = v;
    else st_remote64(lpc::mapa_shared(lpc::smem_u32(where), r), v);
  }
  __device__ __forceinline__ uint32_t load(const uint32_t* where, int r) const {
    return ONE || r == rank ? *where : ld_remote(lpc::mapa_shared(lpc::smem_u32(where), r));
  }
  __device__ __forceinline__ void store_all(uint64_t* where, uint64_t v) const {
#pragma unroll
    for (int r = 0; r < CTAS; ++r)
      if (ONE || r < ctas) store(where, r, v);
  }

  // 2^44 w of a logit, before (`exact`) and after rounding.  ALL: every lane of the warp
  // is here, and the table comes from the lanes' registers.
  template <bool ALL>
  __device__ __forceinline__ uint64_t weight(float f, double* exact = nullptr) const {
    // (ln2/32)^k / k!
    constexpr double A1 = 0.02166084939249829, A2 = 0.00023459619820224677;
    constexpr double A3 = 1.6938509724371819e-06, A4 = 9.172562701824643e-09;
    constexpr double MAGIC = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to an integer
    const double d = (double)fmaxf(f, floorf) - top;
    const double t = fma(d, scale, MAGIC);
    const double r = fma(d, scale, MAGIC - t);
    const int n = __double2loint(t);              // 32 e + j
    const double poly = fma(fma(fma(fma(A4, r, A3), r, A2), r, A1), r, 1.0);
    uint32_t lo, hi;
    if constexpr (ALL) {
      lo = __shfl_sync(~0u, tab_lo, n);
      hi = __shfl_sync(~0u, tab_hi, n) + (uint32_t)n * 32768u;  // + e << 20
    } else {
      lo = (uint32_t)__double2loint(sh.table[n & 31]);
      hi = (uint32_t)__double2hiint(sh.table[n & 31]) + (uint32_t)((n >> 5) << 20);
    }
    const double power = __hiloint2double((int)hi, (int)lo);
    if (exact) *exact = poly * power;
    return (uint64_t)__double_as_longlong(fma(poly, power, ROUND52)) - 0x4330000000000000ull;
  }
  __device__ __forceinline__ uint32_t off_of(float f) const {
    return (uint32_t)kmax - (uint32_t)order_of(f);
  }
  __device__ __forceinline__ float at_off(uint32_t off) const {
    return value_of((int32_t)((uint32_t)kmax - off));
  }
  // Bin of a logit, rising along the order; BINS: below all bins.
  __device__ __forceinline__ uint32_t bin_of(float f) const {
    const float d = f - topf;
    return d < lowest ? BINS : __float_as_uint(fmaf(d, octaves, 8388608.f)) & 0x7fffffu;
  }

  // The smallest float for which pass() holds, which holds from some float up to the
  // largest logit on: the 32 around a guess, else all there are.  The whole warp.
  template <typename F>
  __device__ float smallest(double guess, F pass) const {
    int32_t lo = order_of(-3.402823466e38f), hi = kmax;
    const int32_t near = order_of((float)fmax(guess, -3e38));
    if (near > lo + 64 && near < hi - 64) {
      const unsigned ok = __ballot_sync(~0u, pass(value_of(near - 16 + lane)));
      if (ok && ok != ~0u) return value_of(near - 16 + __ffs(ok) - 1);
    }
    while (lo < hi) {
      const uint32_t span = (uint32_t)hi - (uint32_t)lo;
      const int32_t c = (int32_t)((uint32_t)lo + (uint32_t)(((uint64_t)span * (uint32_t)lane) >> 5));
      const unsigned ok = __ballot_sync(~0u, pass(value_of(c)));
      const int s = ok ? __ffs(ok) - 1 : 32;  // the first that passes
      if (s < 32) hi = __shfl_sync(~0u, c, s);
      if (s > 0) lo = __shfl_sync(~0u, c, s - 1) + 1;
    }
    return value_of(hi);
  }

  // The smallest float of the bins up to `bin`.
  __device__ float bin_start(int bin, double unit) const {
    return smallest(top - ((double)bin + 0.5) / OCTAVE * unit,
                    [&](float f) { return bin_of(f) <= (uint32_t)bin; });
  }

  // fn(chunk, index of its first element) for the warp's chunks, every lane of the warp
  // at once; -inf where there is none.
  template <typename F>
  __device__ __forceinline__ void each(F fn) const {
    each_of(warp * segment, min(nchunks, (warp + 1) * segment), fn);
  }
  template <typename F>
  __device__ __forceinline__ void each_of(int start, int stop, F fn) const {
    for (int c0 = start; c0 < stop; c0 += 32) {
      const int c = c0 + lane;
      Chunk<T> x;
      if (c < stop) x.raw = chunks[c];
      else x.raw = Chunk<T>::nothing();
      fn(x, first + c * N);
    }
  }

  // fn(chunk) for the chunks that this thread wrote, to change them.
  template <typename F>
  __device__ void each_own(F fn) const {
    const int stop = min(nchunks, (warp + 1) * segment);
    for (int c = warp * segment + lane; c < stop; c += 32) {
      Chunk<T> x;
      x.raw = chunks[c];
      fn(x);
      chunks[c] = x.raw;
    }
  }

  // Every warp's `mine` for the whole cluster, in the order of the row: where they are
  // after the next sync().
  __device__ const uint64_t* offer(uint64_t mine) {
    const int s = slot;
    slot = slot == 2 ? 0 : slot + 1;
    if (lane < ctas) store(&sh.sums[s][rank * WARPS + warp], lane, mine);
    return sh.sums[s];
  }
  __device__ const uint64_t* exchange(uint64_t mine) {
    const uint64_t* sums = offer(mine);
    sync();
    return sums;
  }
  __device__ uint64_t total_of(const uint64_t* sums) const {
    uint64_t v = 0;
    for (int i = lane; i < ctas * WARPS; i += 32) v += sums[i];
    return warp_sum(v);
  }

  // Of n <= 128 sums the one (-1: none) in which the running sum exceeds target; `before`:
  // the sum before it.  The whole warp.
  __device__ int crossing_of(const uint64_t* sums, int n, uint64_t target, uint64_t& before) const {
    uint64_t v[4], own = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = 4 * lane + i < n ? sums[4 * lane + i] : 0ull;
      own += v[i];
    }
    uint64_t run = before + warp_scan(own, lane) - own, at = 0;
    int which = -1;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (run <= target && target < run + v[i]) {
        which = 4 * lane + i;
        at = run;
      }
      run += v[i];
    }
    const unsigned who = __ballot_sync(~0u, which >= 0);
    if (!who) return -1;
    const int l = __ffs(who) - 1;
    before = (uint64_t)__shfl_sync(~0u, (uint32_t)at, l) |
             (uint64_t)__shfl_sync(~0u, (uint32_t)(at >> 32), l) << 32;
    return __shfl_sync(~0u, which, l);
  }

  // Lowest row index at which the running sum of fn(value, index) exceeds
  // target(total); `mine` is this warp's sum.  total > target.  It goes to *out, or, if
  // that is null, to every thread of the cluster.  The CTA that has it shares the warp's
  // stretch out to all its warps.
  template <typename F, typename G>
  __device__ int locate(uint64_t mine, F fn, G target_of, int64_t* out) {
    const uint64_t* sums = exchange(mine);
    const uint64_t target = target_of(total_of(sums));
    uint64_t before = 0;
    const int owner = crossing_of(sums, ctas * WARPS, target, before);
    const int f = found_slot;
    found_slot ^= 1;
    if (owner >= 0 && owner / WARPS == rank) {
      const int start = owner % WARPS * segment, stop = min(nchunks, start + segment);
      int from = start, to = stop;
      bool mine_it = warp == owner % WARPS;
      if (segment > 32) {  // several steps of a warp
        const int share = (segment + WARPS - 1) / WARPS;
        from = start + warp * share;
        to = min(stop, from + share);
        uint64_t sum = 0;
        each_of(from, to, [&](const Chunk<T>& x, int at) {
#pragma unroll
          for (int i = 0; i < N; ++i) sum += fn(x.get(i), at + i);
        });
        sum = warp_sum(sum);
        if (lane == 0) sh.scan[warp] = sum;
        __syncthreads();
        mine_it = crossing_of(sh.scan, WARPS, target, before) == warp;
      }
      if (mine_it) {
        bool done = false;
        each_of(from, to, [&](const Chunk<T>& x, int at) {
          if (done) return;
          uint64_t run[N], part = 0;
#pragma unroll
          for (int i = 0; i < N; ++i) run[i] = part += fn(x.get(i), at + i);
          const uint64_t scan = warp_scan(part, lane);
          const unsigned over = __ballot_sync(~0u, before + scan > target);
          if (over) {
            done = true;
            if (lane == __ffs(over) - 1) {
              int found = N - 1;
#pragma unroll
              for (int i = N - 2; i >= 0; --i)
                if (before + scan - part + run[i] > target) found = i;
              if (out) *out = at + found;
              else store_all(&sh.found[f], (uint64_t)(at + found));
            }
          } else {
            before += (uint64_t)__shfl_sync(~0u, (uint32_t)scan, 31) |
                      ((uint64_t)__shfl_sync(~0u, (uint32_t)(scan >> 32), 31) << 32);
          }
        });
      }
    }
    if (out) return 0;
    sync();
    return (int)sh.found[f];
  }
  // This warp's sum of fn(value, index).
  template <typename F>
  __device__ uint64_t sum_of(F fn) const {
    uint64_t mine = 0;
    each([&](const Chunk<T>& x, int at) {
#pragma unroll
      for (int i = 0; i < N; ++i) mine += fn(x.get(i), at + i);
    });
    return warp_sum(mine);
  }

  // Histogram over the bins: of counts, or of fp32 weights in units of 2^-15 of a bin's
  // middle.
  template <bool MASS>
  __device__ void histogram() {
    for (int i = threadIdx.x; i < BINS; i += THREADS) hist[i] = 0u;
    if (threadIdx.x == 0) sh.listed = 0;
    __syncthreads();
    const uint32_t base = lpc::smem_u32(hist) - 4u * 0x4b000000u;  // the bits of 2^23
    // what lies below all bins goes to unused words: a branch an element cost 7 instructions
    // of 82 (512 rows of 32,000 with top-p: 62.4 us, so 58.9)
    const uint32_t nowhere = lpc::smem_u32(hist + BINS + lane);
    each([&](const Chunk<T>& x, int) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float d = x.get(i) - topf;
        const float t = fmaf(d, octaves, 8388608.f);
        uint32_t add = 1u;
        if constexpr (MASS) {
          // 2^15 * 2^(-rest / OCTAVE), by two terms of the series (2e-7 off)
          constexpr float STEP = -0.69314718f / OCTAVE;
          const float rest = fmaf(d, octaves, 8388608.f - t);
          add = __float_as_uint(fmaf(fmaf(rest, 16384.f * STEP * STEP, 32768.f * STEP), rest,
                                     32768.f + 8388608.f)) - 0x4b000000u;
        }
        atom_add(d >= lowest ? base + 4u * __float_as_uint(t) : nowhere, add);
      }
    });
    sync();
  }
  // Each CTA has BINS / ctas bins of the cluster's, a thread up to MINE of them.
  __device__ __forceinline__ int bins_a_thread() const { return ONE ? MINE : max(1, MINE / ctas); }
  __device__ __forceinline__ int first_bin() const {
    return ONE ? MINE * (int)threadIdx.x : rank * (BINS / ctas) + (int)threadIdx.x * bins_a_thread();
  }
  template <bool WIDE>
  __device__ __forceinline__ void merge(uint64_t (&v)[MINE]) const {
    const int m = bins_a_thread(), at = first_bin();
    const bool has = ONE || (int)threadIdx.x * m < BINS / ctas;
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
      v[i] = 0;
      if (!has || i >= m) continue;
      uint32_t lo[CTAS], hi[CTAS];
#pragma unroll
      for (int r = 0; r < CTAS; ++r) {  // all in flight
        lo[r] = hi[r] = 0;
        if (ONE || r < ctas) {
          lo[r] = load(hist + at + i, r);
          if constexpr (WIDE) hi[r] = load(hist + BINS + at + i, r);
        }
      }
#pragma unroll
      for (int r = 0; r < CTAS; ++r) v[i] += (uint64_t)hi[r] << 32 | lo[r];
    }
  }
  // The bin whose running sum, begun at `above`, first exceeds target(above + total)
  // (-1: none); sh.cross: it, the sum before it and in it.
  template <bool WIDE, typename G>
  __device__ int crossing(uint64_t above, G target_of) {
    uint64_t v[MINE], own = 0;
    merge<WIDE>(v);
#pragma unroll
    for (int i = 0; i < MINE; ++i) own += v[i];
    uint64_t run = warp_scan(own, lane);
    if (lane == 31) sh.scan[warp] = run;
    if (threadIdx.x == 0) sh.cross[0] = ~0ull;
    __syncthreads();
    uint64_t total = 0;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) {
      const uint64_t s = sh.scan[i];
      total += s;
      if (i < warp) run += s;
    }
    run += above - own;
    const int s = part_slot;
    part_slot ^= 1;
    if constexpr (ONE) {
      total += above;
    } else {
      if (threadIdx.x == 0) store_all(&sh.parts[s][rank], total);
      sync();
      total = above;
#pragma unroll
      for (int r = 0; r < CTAS; ++r)
        if (r < ctas) {
          total += sh.parts[s][r];
          if (r < rank) run += sh.parts[s][r];
        }
    }
    const uint64_t target = target_of(total);
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
      if (run <= target && target < run + v[i]) {
        store_all(&sh.cross[0], (uint64_t)(first_bin() + i));
        store_all(&sh.cross[1], run);
        store_all(&sh.cross[2], v[i]);
      }
      run += v[i];
    }
    sync();
    return (int)sh.cross[0];
  }
  // The bins between which the running sum of the weights passes p * (their sum), with
  // `slack` of all on either side: sh.window.  False: it may pass below all bins.
  __device__ bool window(float p, float slack) {
    uint64_t v[MINE];
    merge<false>(v);
    float w[MINE], own = 0;
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
      w[i] = (float)v[i] * exp2f(-(float)(first_bin() + i) / OCTAVE);
      own += w[i];
    }
    float run = own;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const float o = __shfl_up_sync(~0u, run, d);
      if (lane >= d) run += o;
    }
    float* scan = reinterpret_cast<float*>(sh.scan);
    if (lane == 31) scan[warp] = run;
    if (threadIdx.x == 0) {
      sh.window[0] = sh.window[1] = BINS;
      sh.last = 0;
    }
    __syncthreads();
    float total = 0;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) {
      if (i < warp) run += scan[i];
      total += scan[i];
    }
    run -= own;
    const int s = part_slot;
    part_slot ^= 1;
    if constexpr (!ONE) {
      if (threadIdx.x == 0) store_all(&sh.parts[s][rank], __float_as_uint(total));
      sync();
      total = 0;
#pragma unroll
      for (int r = 0; r < CTAS; ++r)
        if (r < ctas) {
          const float x = __uint_as_float((uint32_t)sh.parts[s][r]);
          if (r < rank) run += x;
          total += x;
        }
    }
    const float lo = (p - slack) * total, hi = (p + slack) * total;
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
      const int bin = first_bin() + i;
      if ((bin == 0 || run <= lo) && lo < run + w[i]) store_all(&sh.window[0], (uint64_t)bin);
      if ((bin == 0 || run <= hi) && hi < run + w[i]) store_all(&sh.window[1], (uint64_t)bin);
      run += w[i];
    }
    sync();
    return sh.window[0] < BINS && sh.window[1] < BINS;
  }

  // Puts the elements of a chunk in [from, below) on this CTA's list; LIST of them at most
  // are kept, all are counted.
  __device__ __forceinline__ void list(const Chunk<T>& x, int at, float from, float below) {
    unsigned mine = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) mine |= x.get(i) >= from && !(x.get(i) >= below) ? 1u << i : 0u;
    if (!mine) return;
    uint32_t to = atomicAdd(&sh.listed, (uint32_t)__popc(mine));
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (mine >> i & 1u) {
        if (to < (uint32_t)LIST) own_list[to] = Entry{(uint32_t)(at + i), off_of(x.get(i))};
        ++to;
      }
  }
  // The cluster's lists, with their weights, where this CTA's histogram was; their
  // length, or -1 where they are longer than `most`.
  // After a sync() since they were written and the histograms read.
  __device__ int gather(int most) {
    int n = 0;
    if (lane < ctas) n = (int)load(&sh.listed, lane);
    int upto = n;  // inclusive
#pragma unroll
    for (int d = 1; d < MAX_CLUSTER; d <<= 1) {
      const int o = __shfl_up_sync(~0u, upto, d);
      if (lane >= d) upto += o;
    }
    const int total = __shfl_sync(~0u, upto, MAX_CLUSTER - 1);
    if (total > most) return -1;
    Listed* all = reinterpret_cast<Listed*>(hist);
    for (int i0 = 0; i0 < total; i0 += THREADS) {
      const int i = i0 + (int)threadIdx.x;
      int r = 0, start = 0;  // the list that has element i
#pragma unroll
      for (int x = 0; x < MAX_CLUSTER; ++x) {
        const int end_x = __shfl_sync(~0u, upto, x);
        if (i >= end_x) {
          r = x + 1;
          start = end_x;
        }
      }
      if (i < total) {
        const uint32_t* from = &own_list[i - start].index;
        const uint32_t index = load(from, r), off = load(from + 1, r);
        all[i] = Listed{(uint64_t)off << 32 | index, weight<false>(at_off(off))};
      }
    }
    __syncthreads();
    return total;
  }

  // The smallest x in [lo, hi] up to which the listed elements (key(place) <= x, those with
  // an offset of `only` where that is not ~0), on top of `before`, weigh more than target; hi
  // if none.  A warp a pivot.
  __device__ uint32_t search(int n, bool by_index, uint32_t only, uint32_t lo, uint32_t hi,
                             uint64_t before, uint64_t target) {
    const Listed* all = reinterpret_cast<const Listed*>(hist);
    while (lo < hi) {
      const uint32_t x = lo + (uint32_t)((uint64_t)(hi - lo) * (uint32_t)warp / WARPS);
      uint64_t sum = 0;
      for (int i = lane; i < n; i += 32) {
        const uint64_t place = all[i].place;
        const uint32_t off = (uint32_t)(place >> 32);
        if (by_index ? off == only && (uint32_t)place <= x : off <= x) sum += all[i].weight;
      }
      sum = warp_sum(sum);
      if (lane == 0) sh.scan[warp] = before + sum > target;
      __syncthreads();
      const unsigned over = __ballot_sync(~0u, lane < WARPS && sh.scan[lane & (WARPS - 1)] != 0);
      const int s = over ? __ffs(over) - 1 : WARPS;  // the first pivot that is enough
      const uint32_t range = hi - lo, old = lo;
      if (s < WARPS) hi = old + (uint32_t)((uint64_t)range * (uint32_t)s / WARPS);
      if (s > 0) lo = old + (uint32_t)((uint64_t)range * (uint32_t)(s - 1) / WARPS) + 1u;
      __syncthreads();
    }
    return hi;
  }
  // The listed elements' weight up to an offset, without it.
  __device__ uint64_t listed_before(int n, uint32_t off) const {
    const Listed* all = reinterpret_cast<const Listed*>(hist);
    uint64_t sum = 0;
    for (int i = lane; i < n; i += 32)
      if ((uint32_t)(all[i].place >> 32) < off) sum += all[i].weight;
    return warp_sum(sum);
  }

  // One round of the radix select: sums of counts or weights in bins of 2^shift of the
  // offset from the largest, over offsets [lo, hi].  Crossing as above.
  template <bool MASS, typename G>
  __device__ int round(uint32_t lo, uint32_t hi, int shift, uint64_t above, G target_of) {
    sync();  // the histogram before has been read
    for (int i = threadIdx.x; i < BINS * 2; i += THREADS) hist[i] = 0u;
    __syncthreads();
    each([&](const Chunk<T>& x, int) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float f = x.get(i);
        const uint32_t off = off_of(f);
        if (off - lo <= hi - lo && f != -INFINITY) {
          const uint32_t bin = (off - lo) >> shift;
          const uint64_t w = MASS ? weight<false>(f) : 1ull;
          const uint32_t was = atomicAdd(hist + bin, (uint32_t)w);
          const uint32_t up = (uint32_t)(w >> 32) + (was + (uint32_t)w < was ? 1u : 0u);
          if (up) atomicAdd(hist + BINS + bin, up);
        }
      }
    });
    sync();
    return crossing<true>(above, target_of);
  }
  // Offset, sum before it and sum at it of the first value, of offsets up to `last`, at
  // which the running sum exceeds target(total); false: none does.
  template <bool MASS, typename G>
  __device__ bool select(uint32_t last, G target_of, uint32_t& off, uint64_t& before, uint64_t& in) {
    constexpr int G0 = GRAIN<T>;
    uint32_t lo = 0, hi = last;
    uint64_t above = 0, target = 0;
    bool known = false;
    for (int shift = 21;;) {
      auto goal = [&](uint64_t total) { return known ? target : (target = target_of(total)); };
      const int bin = round<MASS>(lo, hi, shift, above, goal);
      if (bin < 0) return false;
      known = true;
      lo += (uint32_t)bin << shift;
      above = sh.cross[1];
      if (shift == G0) break;
      hi = min(hi, lo + ((1u << shift) - 1u));
      shift = max(G0, shift - 11);
    }
    off = lo;
    before = above;
    in = sh.cross[2];
    return true;
  }
};

// The token of a row of which the list (n elements, where the histogram was) holds the
// first top_k of the order.  One CTA, every thread.
template <typename T, bool ONE>
__device__ void draw_from_list(Row<T, ONE>& row, int n, int top_k, float top_p, float least, float u,
                               int64_t* out) {
  Shared& sh = row.sh;
  Listed* all = reinterpret_cast<Listed*>(row.hist);
  constexpr int EACH = PAIRS / THREADS;
  uint64_t place[EACH], w[EACH];
  bool stays[EACH];
  uint64_t run[EACH];
  auto total = [&]() {
    uint64_t v = 0;
#pragma unroll
    for (int e = 0; e < EACH; ++e) v += stays[e] ? w[e] : 0ull;
    v = warp_sum(v);
    __syncthreads();
    if (row.lane == 0) sh.scan[row.warp] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int x = 0; x < WARPS; ++x) v += sh.scan[x];
    return v;
  };
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int i = (int)threadIdx.x + e * THREADS;
    const bool in = i < n;
    place[e] = in ? all[i].place : ~0ull;
    w[e] = in ? all[i].weight : 0ull;
    run[e] = 0;
    int rank = 0;
    if (in)
#pragma unroll 4
      for (int j = 0; j < n; ++j)
        if (all[j].place < place[e]) {
          run[e] += all[j].weight;
          ++rank;
        }
    stays[e] = in && rank < top_k;
  }
  if (top_p < 1.f) {
    const uint64_t target = part_of(top_p, total());
#pragma unroll
    for (int e = 0; e < EACH; ++e) stays[e] = stays[e] && run[e] <= target;
  }
#pragma unroll
  for (int e = 0; e < EACH; ++e)
    stays[e] = stays[e] && row.at_off((uint32_t)(place[e] >> 32)) >= least;
  const uint64_t target = part_of(u, total());
  // by index from here on; every thread has read the places
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int i = (int)threadIdx.x + e * THREADS;
    if (i < n) all[i].place = stays[e] ? (uint64_t)(uint32_t)place[e] : ~0ull;
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < EACH; ++e)
    if (stays[e]) {
      const uint64_t at = (uint32_t)place[e];
      uint64_t before = 0;
#pragma unroll 4
      for (int j = 0; j < n; ++j)
        if (all[j].place < at) before += all[j].weight;
      if (before <= target && target < before + w[e]) *out = (int64_t)at;
    }
}

template <typename T, bool ONE>
__global__ void __launch_bounds__(THREADS, 2) sample_kernel(const Args a) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ Shared sh;
  constexpr int N = Chunk<T>::N;
  Row<T, ONE> row(sh);
  uint32_t ctas = 1;
  if constexpr (!ONE) asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
  row.rank = ONE ? 0 : (int)lpc::cluster_ctarank();
  row.ctas = (int)ctas;
  row.warp = threadIdx.x >> 5;
  row.lane = threadIdx.x & 31;
  row.hist = reinterpret_cast<uint32_t*>(smem);
  row.own_list = reinterpret_cast<Entry*>(smem + HIST_BYTES);
  row.chunks = reinterpret_cast<uint4*>(smem + HIST_BYTES + LIST_BYTES);
  const int64_t r = blockIdx.x / ctas;

  // ---- the share of the row, and its largest ----
  const int begin = min(row.rank * a.slice, a.vocab);
  const int count = min(a.slice, a.vocab - begin);
  const T* src = static_cast<const T*>(a.logits) + r * a.row_stride + begin;
  const int skew = (int)((reinterpret_cast<uintptr_t>(src) & 15u) / sizeof(T));
  row.first = begin - skew;
  row.begin = begin;
  row.end = begin + count;
  row.nchunks = count > 0 ? (skew + count + N - 1) / N : 0;
  row.segment = ((row.nchunks + WARPS - 1) / WARPS + 31) / 32 * 32;
  // every CTA of the cluster has to have started before its memory is written
  if constexpr (!ONE) cluster_arrive();
  if (threadIdx.x < 32) sh.table[threadIdx.x] = exp2((double)threadIdx.x / 32.0) * FIXED;
  lpc::pdl_wait();
  const float u = a.uniforms[r];
  const float temperature = a.temperature ? a.temperature[r] : a.t;
  const float top_p = a.top_p ? a.top_p[r] : a.p;
  const float min_p = a.min_p ? a.min_p[r] : a.m;
  const int32_t top_k = a.top_k ? a.top_k[r] : a.k;
  float best = -INFINITY;
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
      if (e0 < 0 || e0 + N > count) {  // the row's ends
        alignas(16) T part[N];
        for (int i = 0; i < N; ++i)
          part[i] = e0 + i >= 0 && e0 + i < count ? src[e0 + i] : Num<T>::from_f(-INFINITY);
        x.raw = *reinterpret_cast<const uint4*>(part);
      }
      float m = x.largest();
      if (m != m) {  // NaN counts as -inf
        alignas(16) T part[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float f = x.get(i);
          part[i] = Num<T>::from_f(f != f ? -INFINITY : f);
        }
        x.raw = *reinterpret_cast<const uint4*>(part);
        m = x.largest();
      }
      best = fmaxf(best, m);
      row.chunks[c] = x.raw;
    }
  }
#pragma unroll
  for (int m = 16; m; m >>= 1) best = fmaxf(best, __shfl_xor_sync(~0u, best, m));
  if constexpr (!ONE) cluster_wait();
  {
    const uint64_t* all = row.exchange(__float_as_uint(best));
    best = -INFINITY;
    for (int i = row.lane; i < row.ctas * WARPS; i += 32) best = fmaxf(best, __uint_as_float((uint32_t)all[i]));
#pragma unroll
    for (int m = 16; m; m >>= 1) best = fmaxf(best, __shfl_xor_sync(~0u, best, m));
  }
  const bool bad = !(temperature >= 0.f && temperature < INFINITY) || !(u >= 0.f && u < 1.f) ||
                   !(top_p > 0.f && top_p <= 1.f) || !(min_p >= 0.f && min_p <= 1.f);
  if (bad || best == -INFINITY) {  // the same for the whole cluster
    if (row.rank == 0 && threadIdx.x == 0) {
      if (bad) atomicOr(&g_sample_status, LPC_DEV_ERR_BOUNDS);
      a.out[r] = -1;
    }
    return;
  }
  if (temperature == 0.f) {
    uint64_t at = ~0ull;
    row.each([&](const Chunk<T>& x, int i0) {
#pragma unroll
      for (int i = N - 1; i >= 0; --i)
        if (x.get(i) == best) at = min(at, (uint64_t)(i0 + i));
    });
    const uint64_t* all = row.exchange(warp_min(at));
    if (row.rank == 0 && row.warp == 0) {
      at = ~0ull;
      for (int i = row.lane; i < row.ctas * WARPS; i += 32) at = min(at, all[i]);
      at = warp_min(at);
      if (row.lane == 0) a.out[r] = (int64_t)at;
    }
    return;
  }
  if (best == INFINITY) {  // infinities weigh alike, the others nothing
    row.each_own([&](Chunk<T>& x) {
      alignas(16) T part[N];
#pragma unroll
      for (int i = 0; i < N; ++i) part[i] = Num<T>::from_f(x.get(i) == INFINITY ? 0.f : -INFINITY);
      x.raw = *reinterpret_cast<const uint4*>(part);
    });
    best = 0.f;
  }
  row.kmax = order_of(best);
  row.topf = value_of(row.kmax);
  row.top = (double)row.topf;
  // no steeper than what leaves the float below the largest nothing, so that every float's
  // exponent stays a small integer
  const double step = row.top - (double)value_of(row.kmax - 1);
  double per_unit = 1.4426950408889634074 / (double)temperature;
  double unit = 0.69314718055994530942 * (double)temperature;  // 1 / per_unit
  if (step * per_unit > 61.0) {
    per_unit = 61.0 / step;
    unit = step / 61.0;
  }
  row.scale = 32.0 * per_unit;
  row.floorf = fmaxf(__double2float_rd(row.top - 60.0 * unit), -3.402823466e38f);
  row.octaves = (float)(-OCTAVE * per_unit);
  row.lowest = (float)(-(double)(BINS - 1) / OCTAVE * unit);
  __syncthreads();
  row.tab_lo = (uint32_t)__double2loint(sh.table[row.lane]);
  row.tab_hi = (uint32_t)__double2hiint(sh.table[row.lane]) - (uint32_t)row.lane * 32768u;
  // where fp32 has the bins: not for temperatures that nobody uses
  const bool binned = fabsf(row.topf) < 1e30f && per_unit < 1e25 && per_unit > 1e-25;
  // min-p: the smallest logit that weighs enough
  float least = -INFINITY;
  if (min_p > 0.f)
    least = row.smallest(row.top + log2((double)min_p) * unit, [&](float f) {
      double exact;
      row.template weight<false>(f, &exact);
      return exact >= (double)min_p * FIXED;
    });

  // ---- the place in the order up to which logits stay: values above `cut`, and of
  // those at it the ones with an index up to `last` ----
  float cut = -3.402823466e38f;
  int last = a.vocab;
  // the same as an offset from the largest, how many stay of those at it (~0: all), and
  // how many there are
  uint32_t cut_off = row.off_of(cut);
  uint64_t ties = ~0ull, present = ~0ull;
  if (top_k > 0 && top_k < a.vocab) {
    // few elements in the bins down to the one of the last: all on the list
    if (top_k <= PAIRS && binned) {
      row.template histogram<false>();
      const int bin = row.template crossing<false>(0, [&](uint64_t) { return (uint64_t)top_k - 1u; });
      if (bin >= 0 && sh.cross[1] + sh.cross[2] <= (uint64_t)PAIRS) {
        const float from = row.bin_start(bin, unit);
        row.each([&](const Chunk<T>& x, int at) {
          if (x.largest() >= from) row.list(x, at, from, INFINITY);
        });
        row.sync();
        const int n = row.gather(PAIRS);
        row.sync();  // the lists have been read: the other CTAs may go
        if (row.rank == 0) draw_from_list(row, n, top_k, top_p, least, u, a.out + r);
        return;
      }
    }
    uint64_t before, in;
    if (row.template select<false>(cut_off, [&](uint64_t) { return (uint64_t)top_k - 1u; }, cut_off,
                                   before, in)) {
      ties = (uint64_t)top_k - before;
      present = in;
    }
  }
  uint64_t mine_kept = 0;  // this warp's sum of the weights that stay, where it is known
  bool known = false;
  if (top_p < 1.f && ties == ~0ull && binned) {
    if (top_k > 0 && top_k < a.vocab) row.sync();  // a histogram before has been read
    row.template histogram<true>();
    if (row.window(top_p, slack_of(a.vocab))) {
      const uint32_t w0 = (uint32_t)sh.window[0], w1 = (uint32_t)sh.window[1];
      const float above_from = w0 == 0 ? INFINITY : row.bin_start((int)w0 - 1, unit);
      const float list_from = row.bin_start((int)w1, unit);
      uint64_t all = 0, above = 0;
      const float kept_from = fmaxf(above_from, least);
      auto pass = [&](auto two) {  // kept apart from above where min-p is higher
        row.each([&](const Chunk<T>& x, int at) {
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const float f = x.get(i);
            const uint64_t w = row.template weight<true>(f);
            all += w;
            if (f >= above_from) above += w;
            if constexpr (decltype(two)::value)
              if (f >= kept_from) mine_kept += w;
          }
          row.list(x, at, list_from, above_from);
        });
      };
      if (kept_from > above_from) {
        pass(std::true_type{});
      } else {
        pass(std::false_type{});
        mine_kept = above;
      }
      mine_kept = warp_sum(mine_kept);
      const uint64_t* alls = row.offer(warp_sum(all));
      const uint64_t* aboves = row.exchange(warp_sum(above));
      const uint64_t total = row.total_of(alls), before = row.total_of(aboves);
      const int n = row.gather(LIST);
      if (n > 0) {
        const uint64_t target = part_of(top_p, total);
        const Listed* listed = reinterpret_cast<const Listed*>(row.hist);
        // the first value, and of those like it the first index, at which the sum passes:
        // the last that stays
        const uint32_t off0 = w0 == 0 ? 0u : row.off_of(above_from), off1 = row.off_of(list_from);
        uint64_t place = 0;
        if (n <= SHORT) {
          if (threadIdx.x < (unsigned)n) {
            const uint64_t at = listed[threadIdx.x].place, w = listed[threadIdx.x].weight;
            uint64_t run = before;
#pragma unroll 4
            for (int j = 0; j < n; ++j)
              if (listed[j].place < at) run += listed[j].weight;
            if (run <= target && target < run + w) sh.last = at + 1u;
          }
          __syncthreads();
          place = sh.last;
        } else {
          const uint32_t off = row.search(n, false, 0u, off0, off1, before, target);
          const uint64_t upto = before + row.listed_before(n, off);
          const uint32_t index = row.search(n, true, off, 0u, (uint32_t)a.vocab, upto, target);
          if (index < (uint32_t)a.vocab) place = ((uint64_t)off << 32 | index) + 1u;
        }
        if (place) {  // 1 more than the last that stays
          cut = row.at_off((uint32_t)((place - 1) >> 32));
          last = (int)(uint32_t)(place - 1);
          // the list's elements that stay, to the warps that have them
          uint64_t more = 0;
          const int lo = max(row.begin, row.first + row.warp * row.segment * N);
          const int hi = min(row.end, row.first + (row.warp + 1) * row.segment * N);
          for (int i = row.lane; i < n; i += 32) {
            const uint64_t e = listed[i].place;
            const int at = (int)(uint32_t)e;
            if (e < place && at >= lo && at < hi && row.at_off((uint32_t)(e >> 32)) >= least)
              more += listed[i].weight;
          }
          mine_kept += warp_sum(more);
          known = true;
        }
      }
    }
  }
  if (!known) {
    if (top_p < 1.f) {
      // of the last value's weight only `ties` count
      const uint64_t extra =
          ties == ~0ull ? 0 : (present - ties) * row.template weight<false>(row.at_off(cut_off));
      uint64_t before, in, target = 0;
      uint32_t off;
      if (row.template select<true>(cut_off,
                                    [&](uint64_t total) { return target = part_of(top_p, total - extra); },
                                    off, before, in)) {
        const uint64_t w = row.template weight<false>(row.at_off(off));
        cut_off = off;
        ties = (target - before) / w + 1u;
        present = in / w;
      }
    }
    cut = row.at_off(cut_off);
    if (ties < present) {
      auto tied = [&](float f, int) -> uint64_t { return f == cut; };
      last = row.locate(row.sum_of(tied), tied, [&](uint64_t) { return ties - 1u; }, nullptr);
    }
  }
  if (least > cut) {
    cut = least;
    last = a.vocab;
  }
  auto draw = [&](uint64_t total) { return part_of(u, total); };
  if (last < a.vocab) {
    auto stays = [&](float f, int at) -> uint64_t {
      const uint64_t w = row.template weight<true>(f);
      return f > cut || (f == cut && at <= last) ? w : 0ull;
    };
    row.locate(known ? mine_kept : row.sum_of(stays), stays, draw, a.out + r);
  } else {
    auto stays = [&](float f, int) -> uint64_t {
      const uint64_t w = row.template weight<true>(f);
      return f >= cut ? w : 0ull;
    };
    row.locate(known ? mine_kept : row.sum_of(stays), stays, draw, a.out + r);
  }
}

template <typename T, bool ONE>
int launch_as(const Args& args, int64_t rows, int ctas, cudaStream_t s) {
  static std::atomic<uint64_t> mask{0};
  const int most = HIST_BYTES + LIST_BYTES + MAX_SLICE_BYTES + 32;
  if (int rc = lpc::once_per_device_smem((const void*)sample_kernel<T, ONE>, most, mask)) return rc;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = lpc::use_pdl() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)ctas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * ctas));
  cfg.blockDim = dim3(THREADS);
  // a chunk more than the share: it may begin inside one
  cfg.dynamicSmemBytes = HIST_BYTES + LIST_BYTES + ((size_t)args.slice * sizeof(T) + 15) / 16 * 16 + 16;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = ONE ? 1 : 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, sample_kernel<T, ONE>, args);
  if (e != cudaSuccess) {
    lpc::set_error("sample_tokens: launch failed: %s", cudaGetErrorString(e));
    return LPC_ERR_CUDA;
  }
  return lpc::check_launch("sample_tokens");
}
template <typename T>
int launch(const Args& args, int64_t rows, int ctas, cudaStream_t s) {
  return ctas == 1 ? launch_as<T, true>(args, rows, ctas, s) : launch_as<T, false>(args, rows, ctas, s);
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
  // CTAs a row: what brings its share to SLICE_BYTES; one is best while it can hold the row,
  // as a barrier of a cluster costs 0.7 us and a row takes six to nine (37 rows of 16,000 with
  // top-p: 14 us by one CTA each, 18 by two or four).  Few long rows get four or eight, while
  // that takes half the SMs at most (beyond it clusters wait for one another): one row of
  // 32,000 11.1 us by one, 6.9 by eight, with top-p 19.5 and 15.5, with top-k 50 11.8 either
  // way; 16 rows 11.6 by one, 9.3 by four, 8.5 by eight, with top-k 50 12.1, 12.1, 14.3.
  int ctas = 1, most = MAX_CLUSTER;
  while (ctas < MAX_CLUSTER && vocab * es > (int64_t)ctas * SLICE_BYTES) ctas *= 2;
  while (most > ctas && rows * most * 2 > current_device_sms()) most /= 2;
  if (vocab > LONG && most >= 4) ctas = most;
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
