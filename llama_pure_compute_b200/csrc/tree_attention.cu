// Attention of a tree of drafted tokens over a KV cache (sm_100a, tcgen05).
//
// out[b, h, t] = sum_j p_j V_j, p = softmax over the visible keys j of
// scale * q[b, h, t] . K_j, fp32 accumulation.  Visible to node t of sequence b:
// the n = seq_lens[b] keys of the context and the nodes i whose bit i is set in
// masks[b, t]; node i is cache row n + i.  A node that sees nothing gives zeros.
//
// The G * T query rows (G heads share a KV head, T <= 64 nodes) meet the same keys,
// so K and V are read once for all of them: an item is one (sequence, KV head,
// block of 128 or 256 rows).  Up to ~250 rows a key's bytes cost more than its
// arithmetic (2 G T flops a byte of K and V), beyond it the tensor cores do.
//
// Schedule.  Every item is a row of 128-key tiles behind START tiles' worth of set-up.
// The items, one after another, are cut into equal stretches, one a CTA and one CTA
// an SM, from the lengths as the device holds them: ragged batches are balanced and
// one long sequence fills the GPU.  A CTA that holds a whole item writes its output;
// parts of items go to a workspace (at most two a CTA, whatever the lengths) and a
// second kernel joins them.
//   Where few items of short capacity would spend their time on that, an item is a
// cluster of 1 to 8 CTAs, which share its tiles and join their parts through
// distributed shared memory (one sequence of 1000 keys, 32 heads: 11.5 us; as
// stretches 15, of which the cutting took 1 and the second kernel 5).
//
// CTA, 12 warps:
//   warp 8      TMA: Q of the stretch's items, K and V tiles through one ring in
//               the order K0 K1 V0 K2 V1 ...
//   warp 9      TMEM, tcgen05.mma: S = Q K^T (M = 128 rows, N = 128 keys), O += P V
//               (P from tensor memory).  Two streams, so that the tensor core works
//               on one while the other's softmax runs:
//                 up to 128 rows: even tiles and odd tiles of the item, each with its
//                   own running maximum, sum and O, joined at the item's end;
//                 more: rows 0-127 and 128-255, both on every tile.
//   warps 0-3, 4-7  softmax of stream 0 and 1.  Thread r has row r: its 128 scores in
//               one read, maximum, exp2 against a reference that moves only when the
//               maximum has grown by more than 8 (factor 256: no overflow, same
//               softmax), P rounded to the data type, as the product's other operand V has
//               it (half a step at most, 2^-8 or 2^-11 of p; fp16's range: RAISE; the
//               sum is of the unrounded), O rescaled in tensor memory when the
//               reference moves.
//   warps 10-11 the tiles that hold nodes or end the sequence: V rows that no node
//               sees are cleared (0 * NaN would reach every row), and so are visible
//               ones that are not finite; those are added in the epilogue, row by row,
//               to the nodes that do see them.
// Tensor memory: S0 S1 O0 O1, 128 columns each.
//
// Times (us, from a CUDA graph; bytes' or operations' floor): 32 sequences of up to 4096 keys, 8
// KV heads of 96 rows 62 (45), of 16 rows 58 (43): 0.8 us a tile of 64 KB while all SMs load, 2.5
// us a further item of a stretch (pipeline out and in, O), 5 to 6 around (cutting, join).  3
// sequences of 60,000 keys, 8 KV heads of 512 rows 327 to 335 for some milliseconds (225 at the
// burst rate of dense products), 405 after seconds of it, at the 1.35 GHz that the power cap leaves
// (271 at the sustained rate): 1.1 and 0.93 PFLOP/s.  A tile of 256 rows takes
// 3150 cycles, 2048 of them MMA: a stream's softmax 1920 (scores 95, maximum 345, exponentials
// 1380), 200 to hand P over, 1030 for its PV and next S.  Slower, all measured: S in two
// buffers of 64 keys (507: Q is read twice as often), two softmax threads a row (383), a
// quarter of the exponentials as polynomials (no gain; the 32 sequences 69).
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "lpc_common.cuh"

LPC_DECLARE_STATUS(g_tree_status)

unsigned int lpc_status_tree_attention(bool clear) {
  unsigned int v = 0;
  cudaMemcpyFromSymbol(&v, g_tree_status, sizeof(v));
  if (clear && v) {
    unsigned int z = 0;
    cudaMemcpyToSymbol(g_tree_status, &z, sizeof(z));
  }
  return v;
}

namespace {

using lpc::Num;

constexpr int MAX_NODES = 64;
constexpr int ROWS = 128;                   // query rows a tile (UMMA M)
constexpr int KEYS = 128;                   // keys a tile
constexpr int BOX = 64;                     // columns a TMA box: one 128-byte swizzle row
constexpr int HALF_BYTES = 128 * BOX * 2;   // 128 rows of a box
constexpr int NTHREADS = 384;
constexpr uint32_t TMEM_COLS = 512;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float GROWTH = 8.0f;              // log2 units that a maximum may pass its reference
// log2 of the weight at the reference.  fp16 holds weights below 2^-14 as subnormals and none
// below 2^-25: 20,000 keys of 2^-25.5 of the largest each were lost, 3e-4 of the result.  With
// 2^7 the largest is 2^15 after GROWTH, and a weight is off by 2^-32 of the largest or its half step.
template <typename T> constexpr float RAISE = 0.0f;
template <> constexpr float RAISE<__half> = 7.0f;
constexpr int LAUNCH_REGS = 168, REGS_LOAD = 96, REGS_SOFTMAX = 200;
static_assert(128 * REGS_LOAD + 256 * REGS_SOFTMAX <= NTHREADS * LAUNCH_REGS,
              "register split exceeds the block's launch allocation");

// Tiles that an item's begin and end cost: the pipeline fills and drains, O is written.
// 32 sequences of up to 4096 keys, 8 KV heads of 96 rows: 65.5 us counted as three, 64.5 as
// four, 63 as five; 16 rows, D = 64 and long sequences differ by 2 %.
constexpr int START = 5;

// What a sequence holds: n keys of context, keys and nodes together up to `end`,
// `tiles` of them; its cache row 0 (of KV head 0).
struct Sequence {
  int64_t row0;
  int n, end, tiles, pad;
};
constexpr int KNOWN = 16;       // sequences from a CTA's first on that it keeps
struct Shared {
  float2 ml[2][ROWS];           // [stream][row]: maximum and sum, up to 128 rows
  Sequence known[KNOWN];
  unsigned long long bad[2];    // visible nodes of the segment whose V is not finite
  uint32_t scan[NTHREADS / 32];
  uint32_t found[2];
};
constexpr int BAR_BYTES = 336;

// HD: columns as the MMA sees them, 64 (head_dim 32 or 64) or 128.  WIDE: 256 rows an item.
template <int HD, bool WIDE>
struct Shape {
  static constexpr int TILE = HD / BOX * HALF_BYTES;         // K, V or Q tile
  static constexpr int QTILES = WIDE ? 2 : 1;                // of an item
  static constexpr int QBUFS = WIDE ? 1 : 2;                 // items whose Q is held
  static constexpr int ITEM_ROWS = QTILES * ROWS;
  static constexpr int SLOTS = (14 * HALF_BYTES - QTILES * QBUFS * TILE) / TILE;  // 224 KB with Q
  static constexpr int TILES = (QTILES * QBUFS + SLOTS) * TILE;
  static constexpr int SMEM = TILES + BAR_BYTES + (int)sizeof(Shared);
  static constexpr int64_t PART = (int64_t)ITEM_ROWS * (HD + 2);  // floats of a part
};

struct TmaDesc4 { alignas(64) unsigned char bytes[128]; };

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const void* tmap, int c0, int c1, int c2,
                                            int c3, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(tmap), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
      : "memory");
}
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint64_t pack_f2(float lo, float hi) {
  return ((uint64_t)__float_as_uint(hi) << 32) | __float_as_uint(lo);
}
__device__ __forceinline__ float lo_f(uint64_t v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float hi_f(uint64_t v) { return __uint_as_float((uint32_t)(v >> 32)); }
__device__ __forceinline__ uint64_t fma_f2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add_f2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&v);
}

struct Params {
  const void *q, *k, *v;
  void* out;
  const int32_t* seq_lens;
  const int64_t* masks;
  int64_t masks_stride;        // of a sequence; 0: one tree for all
  const int64_t* seq_base;     // null: dense
  const int32_t* seq_cap;
  int64_t max_seq_len, total_rows;
  float* parts;                // 2 a CTA
  int2* split;                 // the item that a CTA begins and does not finish (-1: none),
                               // and the last CTA that has a part of it
  int batch, nodes, heads, kv_heads, group, head_dim, row_blocks;
  int cluster;                 // CTAs an item; 0: stretches
  float scale_log2;
};

__device__ __forceinline__ Sequence sequence_of(const Params& p, int b, bool report) {
  Sequence s;
  int64_t cap = p.max_seq_len;
  s.row0 = (int64_t)b * p.kv_heads * p.max_seq_len;
  bool bad = false;
  int n = lpc::ld_dep(p.seq_lens + b);
  if (p.seq_base) {
    s.row0 = lpc::ld_dep(p.seq_base + b);
    cap = lpc::ld_dep(p.seq_cap + b);
    if (s.row0 < 0 || cap < 0 || s.row0 > p.total_rows - cap) {
      bad = true;
      s.row0 = 0;
      cap = 0;
    }
  }
  bad |= n < 0 || n > cap;
  s.n = max(0, min(n, (int)cap));
  s.end = min(s.n + p.nodes, (int)cap);
  s.tiles = max(1, (s.end + KEYS - 1) / KEYS);
  if (bad && report) atomicOr(&g_tree_status, LPC_DEV_ERR_BOUNDS);
  return s;
}

// The stretches: all = q * used + rem units, the first rem CTAs have one more.
struct Cut {
  uint32_t used, q, rem;
  __device__ Cut(uint32_t all, uint32_t grid) : used(min(all, grid)), q(all / used), rem(all - q * used) {}
  __device__ __forceinline__ uint32_t begin(uint32_t c) const { return c * q + min(c, rem); }
  __device__ __forceinline__ uint32_t owner(uint32_t x) const {
    const uint32_t big = rem * (q + 1);
    return x < big ? x / (q + 1) : rem + (x - big) / q;
  }
};

// A CTA's stretch, walked item by item.  Every role walks it on its own.
struct Walk {
  const Params& p;
  const Sequence* known;  // of sequences b0 to b0 + KNOWN - 1
  uint32_t pos, stop;     // units still to do: [pos, stop)
  uint32_t base;          // the first unit of sequence b
  int b, b0;
  Sequence s;
  // the present segment
  int kvh, rb;            // KV head, block of rows
  int item;               // (b * kv_heads + kvh) * row_blocks + rb
  int j0, count;          // first tile, tiles
  uint32_t last;          // the unit of the item's last tile
  bool whole;

  __device__ Walk(const Params& params, const Shared& sh, uint32_t at, uint32_t end, uint32_t begin,
                  int seq)
      : p(params), known(sh.known), pos(at), stop(end), base(begin), b(seq), b0(seq) {
    s = sh.known[0];
  }
  __device__ __forceinline__ bool next() {
    while (pos < stop) {
      const uint32_t unit = (uint32_t)(s.tiles + START);
      const uint32_t per = unit * (uint32_t)(p.kv_heads * p.row_blocks);
      if (pos - base >= per) {
        base += per;
        ++b;
        s = b - b0 < KNOWN ? known[b - b0] : sequence_of(p, b, false);
        continue;
      }
      const uint32_t within = pos - base, i = within / unit;
      const int y = (int)(within - i * unit);
      const int y1 = (int)min((uint32_t)unit, (uint32_t)y + (stop - pos));
      last = pos + (uint32_t)(s.tiles + START - 1 - y);
      pos += (uint32_t)(y1 - y);
      j0 = max(0, y - START);
      count = max(0, y1 - START) - j0;
      if (count == 0) continue;  // the set-up alone: whoever has the first tile does it
      kvh = (int)i / p.row_blocks;
      rb = (int)i - kvh * p.row_blocks;
      item = (b * p.kv_heads + kvh) * p.row_blocks + rb;
      whole = count == s.tiles;
      return true;
    }
    return false;
  }
  // whether tile j (of the item) needs masks: it holds nodes or ends the sequence
  __device__ __forceinline__ bool tail(int j) const { return (j + 1) * KEYS > s.n; }
  __device__ __forceinline__ int tails() const {  // such tiles in the segment
    return min(count, max(0, j0 + count - s.n / KEYS));
  }
};

// Bits of the nodes in the cache, of `nodes` and `end - n`.
__device__ __forceinline__ uint64_t node_bits(int count) {
  return count >= 64 ? ~0ull : count <= 0 ? 0ull : (1ull << count) - 1ull;
}

// Joined columns of a KV head's query row, four a time, to the output.
template <typename T, int FOURS>
__device__ __forceinline__ void store_row(const Params& p, int b, int kvh, int row, int col,
                                          const float4 (&o)[FOURS], float L) {
  const float inv = L > 0.f || L != L ? 1.f / L : 0.f;
  const int head = row / p.nodes, node = row - head * p.nodes;
  T* out = static_cast<T*>(p.out) +
           (((int64_t)b * p.nodes + node) * p.heads + kvh * p.group + head) * p.head_dim + col;
  uint32_t x[2 * FOURS];
#pragma unroll
  for (int f = 0; f < FOURS; ++f) {
    x[2 * f] = pack2<T>(o[f].x * inv, o[f].y * inv);
    x[2 * f + 1] = pack2<T>(o[f].z * inv, o[f].w * inv);
  }
  if constexpr (FOURS == 1) *reinterpret_cast<uint2*>(out) = make_uint2(x[0], x[1]);
  else *reinterpret_cast<uint4*>(out) = make_uint4(x[0], x[1], x[2], x[3]);
}
__device__ __forceinline__ float4 ld_remote16(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ float2 ld_remote8(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}

// One thread of the warp, chosen so that the compiler knows it to be one: operands of
// tcgen05.mma and TMA then go to uniform registers directly.  By `lane == 0` an MMA of 64
// cycles took 85 to 120 to issue: 3 sequences of 60,000 keys, 512 rows a KV head 369 us, so
// 339; 32 of up to 4096 keys, 6 KV heads of 26 rows, D = 64 38.6 us, so 35.7.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(one));
  return one != 0;
}

template <typename T, int HD, bool WIDE>
__global__ void __launch_bounds__(NTHREADS, 1)
    tree_attention_kernel(const __grid_constant__ TmaDesc4 tmQ, const __grid_constant__ TmaDesc4 tmK,
                          const __grid_constant__ TmaDesc4 tmV, const Params p, uint32_t idesc_qk,
                          uint32_t idesc_pv) {
  using S = Shape<HD, WIDE>;
  constexpr int TILE = S::TILE, SLOTS = S::SLOTS, NBOX = HD / BOX;
  // tiles are swizzled by their addresses' bits below 1024
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t raw = lpc::smem_u32(smem_raw);
  if (raw & 1023u) {
    atomicOr(&g_tree_status, LPC_DEV_ERR_TIMEOUT);
    return;
  }
  const uint32_t sQ = raw;
  const uint32_t sRing = raw + S::QTILES * S::QBUFS * TILE;
  const uint32_t bars = raw + S::TILES;
  Shared& sh = *reinterpret_cast<Shared*>(smem_raw + S::TILES + BAR_BYTES);
  auto full = [&](uint32_t c) { return bars + 8u * (c % SLOTS); };
  auto empty = [&](uint32_t c) { return bars + 8u * (SLOTS + c % SLOTS); };
  auto slot_parity = [&](uint32_t c) { return (c / SLOTS) & 1u; };
  auto slot = [&](uint32_t c) { return sRing + (c % SLOTS) * (uint32_t)TILE; };
  const uint32_t misc = bars + 16u * SLOTS;
  auto q_full = [&](int r) { return misc + 8u * (r % S::QBUFS); };
  auto q_empty = [&](int r) { return misc + 16u + 8u * (r % S::QBUFS); };
  auto q_parity = [&](int r) { return (uint32_t)(r / S::QBUFS) & 1u; };
  const uint32_t fixed = misc + 32u, o_free = misc + 40u, ml_full = misc + 48u, to_fix = misc + 56u;
  auto s_full = [&](int t) { return misc + 64u + 8u * t; };
  auto p_half = [&](int t) { return misc + 80u + 8u * t; };
  auto p_full = [&](int t) { return misc + 96u + 8u * t; };
  auto o_done = [&](int t) { return misc + 112u + 8u * t; };
  const uint32_t tmem_slot = misc + 128u;
  volatile uint32_t* tmem_slot_ptr =
      reinterpret_cast<volatile uint32_t*>(smem_raw + (tmem_slot - raw));
  static_assert(16 * SLOTS + 132 <= BAR_BYTES, "barriers");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  unsigned int* st = &g_tree_status;
  if (warp == 8 && lane == 0) {
    lpc::tma_prefetch_desc(&tmQ);
    lpc::tma_prefetch_desc(&tmK);
    lpc::tma_prefetch_desc(&tmV);
  }
  if (threadIdx.x < 2 * SLOTS) lpc::mbar_init(bars + 8u * threadIdx.x, 1);
  if (warp == 2) {  // in the order of their places
    constexpr int counts[16] = {1, 1, 1, 1, 2, 8, 8, 1, 1, 1, 4, 4, 4, 4, 1, 1};
    int n = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (lane == i) n = counts[i];
    if (lane < 16) lpc::mbar_init(misc + 8u * lane, n);
  }
  lpc::fence_mbar_init();
  lpc::pdl_wait();

  if (warp == 9) {
    lpc::tmem_alloc(tmem_slot, TMEM_COLS);
    lpc::tmem_relinquish();
  }

  // ---- this CTA's stretch: all units, then the sequence that its first lies in ----
  const uint32_t copies = (uint32_t)(p.kv_heads * p.row_blocks);  // items of a sequence
  auto block_scan = [&](uint32_t v, uint32_t& total) -> uint32_t {  // exclusive
    uint32_t run = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t o = __shfl_up_sync(~0u, run, d);
      if (lane >= d) run += o;
    }
    if (lane == 31) sh.scan[warp] = run;
    __syncthreads();
    uint32_t others = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < NTHREADS / 32; ++i) {
      const uint32_t w = sh.scan[i];
      if (i < warp) others += w;
      total += w;
    }
    __syncthreads();
    return others + run - v;
  };
  const uint32_t c = blockIdx.x;
  Cut cut(1, 1);
  uint32_t pos, stop;
  if (p.cluster) {
    // item c / cluster, and an equal share of its tiles
    const uint32_t item = c / (uint32_t)p.cluster, rank = c - item * (uint32_t)p.cluster;
    const int b = (int)(item / copies);
    const Sequence own = sequence_of(p, b, item == b * copies && rank == 0 && threadIdx.x == 0);
    const uint32_t first = (item - b * copies) * (uint32_t)(own.tiles + START) + START;
    pos = first + (uint32_t)own.tiles * rank / (uint32_t)p.cluster;
    stop = first + (uint32_t)own.tiles * (rank + 1) / (uint32_t)p.cluster;
    if (threadIdx.x == 0) {
      sh.known[0] = own;
      sh.found[0] = (uint32_t)b;
      sh.found[1] = 0;
    }
  } else {
    if (threadIdx.x == 0) sh.found[0] = sh.found[1] = 0;
    uint32_t all = 0, mine = 0, before = 0;
    Sequence own;
    for (int b0 = 0; b0 < p.batch; b0 += NTHREADS) {
      const int b = b0 + (int)threadIdx.x;
      mine = 0;
      if (b < p.batch) {
        own = sequence_of(p, b, blockIdx.x == 0);
        mine = (uint32_t)(own.tiles + START) * copies;
      }
      uint32_t total;
      before = block_scan(mine, total);
      all += total;
    }
    cut = Cut(all, gridDim.x);
    pos = c < cut.used ? cut.begin(c) : 0;
    stop = c < cut.used ? cut.begin(c + 1) : 0;
    uint32_t upto = 0;
    for (int b0 = 0; b0 < p.batch; b0 += NTHREADS) {
      const int b = b0 + (int)threadIdx.x;
      uint32_t total = 0;
      if (p.batch > NTHREADS) {
        mine = 0;
        if (b < p.batch) {
          own = sequence_of(p, b, false);
          mine = (uint32_t)(own.tiles + START) * copies;
        }
        before = block_scan(mine, total);
      }
      if (upto + before <= pos && pos < upto + before + mine) {
        sh.found[0] = (uint32_t)b;
        sh.found[1] = upto + before;
      }
      upto += total;
    }
    __syncthreads();
    if (p.batch <= NTHREADS) {
      const int at = (int)threadIdx.x - (int)sh.found[0];
      if ((int)threadIdx.x < p.batch && at >= 0 && at < KNOWN) sh.known[at] = own;
    } else if (threadIdx.x < KNOWN && (int)(sh.found[0] + threadIdx.x) < p.batch) {
      sh.known[threadIdx.x] = sequence_of(p, (int)(sh.found[0] + threadIdx.x), false);
    }
  }
  lpc::tc_fence_before();
  __syncthreads();
  lpc::tc_fence_after();
  const uint32_t tmem = *tmem_slot_ptr;
  lpc::pdl_trigger();  // only with the tensor memory in hand: the next grid may take what is left

  const int seq = (int)sh.found[0];
  const uint32_t seq_first = sh.found[1];
  // an item in several parts, joined here
  const bool joined = p.cluster > 1 && sh.known[0].tiles > 1;

  // ring places of the K and V tiles of a segment's tile i: K0 K1 V0 K2 V1 ...
  auto k_at = [](uint32_t ring, int i) { return ring + (uint32_t)(i == 0 ? 0 : 2 * i - 1); };
  auto v_at = [](uint32_t ring, int i, int n) {
    return ring + (uint32_t)(i == n - 1 ? 2 * n - 1 : 2 * i + 2);
  };

  if (warp >= 8) {
    // hands registers to the softmax warps: 128 x 96 + 256 x 200 <= 384 x 168 (the
    // host refuses to launch with any other count)
    asm volatile("setmaxnreg.dec.sync.aligned.u32 96;\n" ::: "memory");
    if (warp == 8) {
      // ---------------- loads ----------------
      if (elect_one()) {
        bool ok = true;
        uint32_t issued = 0;
        int r = 0;
        int2 begun = make_int2(-1, -1);
        Walk w(p, sh, pos, stop, seq_first, seq);
        while (ok && w.next()) {
          if (!(ok = lpc::mbar_wait(q_empty(r), q_parity(r) ^ 1u, st))) break;
          lpc::mbar_arrive_expect_tx(q_full(r), S::QTILES * TILE);
          const uint32_t q_at = sQ + (uint32_t)(r % S::QBUFS) * TILE;
          for (int t = 0; t < S::QTILES; ++t)
#pragma unroll
            for (int h = 0; h < NBOX; ++h)
              tma_load_4d(q_at + t * TILE + h * HALF_BYTES, &tmQ, h * BOX, w.rb * S::ITEM_ROWS + t * ROWS,
                          w.b * p.kv_heads + w.kvh, 0, q_full(r));
          const int row = p.seq_base ? (int)w.s.row0 : 0;
          const int b4 = p.seq_base ? 0 : w.b;
          auto load = [&](const void* map, int i) -> bool {
            if (!lpc::mbar_wait(empty(issued), slot_parity(issued) ^ 1u, st)) return false;
            lpc::mbar_arrive_expect_tx(full(issued), TILE);
#pragma unroll
            for (int h = 0; h < NBOX; ++h)
              tma_load_4d(slot(issued) + h * HALF_BYTES, map, h * BOX,
                          row + (w.j0 + i) * KEYS, w.kvh, b4, full(issued));
            ++issued;
            return true;
          };
          ok = load(&tmK, 0);
          for (int i = 0; i < w.count && ok; ++i) {
            if (i + 1 < w.count) ok = load(&tmK, i + 1);
            ok = ok && load(&tmV, i);
          }
          ++r;
          if (w.j0 == 0 && !w.whole) begun = make_int2(w.item, (int)cut.owner(w.last));
        }
        if (p.split) p.split[c] = begun;
        if (!ok)  // copies in flight land before the CTA ends
          for (uint32_t x = issued > SLOTS ? issued - SLOTS : 0; x < issued; ++x)
            lpc::mbar_wait(full(x), slot_parity(x), st);
      }
    } else if (warp == 9) {
      // ---------------- tensor core ----------------
      if (elect_one()) {
        bool ok = true;
        uint32_t ring = 0, done[2] = {0, 0}, fixes = 0;  // P tiles of each stream; segments with tails
        int r = 0;
        const uint64_t dQ = lpc::smem_desc_sw128(sQ, 16, 1024);
        const uint64_t dK = lpc::smem_desc_sw128(sRing, 16, 1024);
        const uint64_t dV = lpc::smem_desc_sw128(sRing, HALF_BYTES, 1024);
        auto issue_s = [&](int t, uint32_t at, bool release) -> bool {
          if (!lpc::mbar_wait(full(at), slot_parity(at), st)) return false;
          lpc::tc_fence_after();
          const uint64_t aq = dQ + (uint64_t)(((WIDE ? t : r % S::QBUFS) * TILE) >> 4);
          const uint64_t bk = dK + (uint64_t)(((at % SLOTS) * (uint32_t)TILE) >> 4);
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk) {
            const uint32_t off = (uint32_t)(((kk >> 2) * HALF_BYTES) >> 4) + 2u * (kk & 3);
            lpc::umma_ss(tmem + 128u * t, aq + off, bk + off, idesc_qk, kk != 0);
          }
          lpc::umma_commit(s_full(t));
          if (release) lpc::umma_commit(empty(at));
          return true;
        };
        auto issue_pv = [&](int t, uint32_t at, bool first, bool release) -> bool {
          const uint32_t ph = done[t]++ & 1u;
          if (!lpc::mbar_wait(p_half(t), ph, st)) return false;
          if (!lpc::mbar_wait(full(at), slot_parity(at), st)) return false;
          lpc::tc_fence_after();
          const uint64_t bv = dV + (uint64_t)(((at % SLOTS) * (uint32_t)TILE) >> 4);
#pragma unroll
          for (int kk = 0; kk < KEYS / 16; ++kk) {
            if (kk == KEYS / 32) {
              if (!lpc::mbar_wait(p_full(t), ph, st)) return false;
              lpc::tc_fence_after();
            }
            lpc::umma_ts(tmem + 256u + 128u * t, tmem + 128u * t + 8u * kk,
                         bv + (uint64_t)((kk * 16 * 128) >> 4), idesc_pv, !first || kk != 0);
          }
          if (release) lpc::umma_commit(empty(at));
          return true;
        };
        Walk w(p, sh, pos, stop, seq_first, seq);
        while (ok && w.next()) {
          const int n = w.count;
          if (!(ok = lpc::mbar_wait(q_full(r), q_parity(r), st))) break;
          lpc::tc_fence_after();
          // Tails may be cleared from the scores of the first of them on: every use of the
          // ring's slots before theirs has landed by then, so the clearing warps cannot take
          // an older phase for theirs.
          const int tails = w.tails();
          bool ready = false;  // O of the segment before, and with it sh.bad, has been read
          auto ask = [&](int i) {
            if (tails && i == n - tails) lpc::mbar_arrive(to_fix);
          };
          // S of tile i; the last one of the segment releases Q
          auto scores = [&](int t, int i) -> bool {
            const bool last = WIDE ? t == 1 : true;
            if (!issue_s(t, k_at(ring, i), last)) return false;
            if (last && i == n - 1) lpc::umma_commit(q_empty(r));
            if (ready && (!WIDE || t == 0)) ask(i);
            return true;
          };
          bool clean = false;  // the segment's tails are
          auto values = [&](int t, int i) -> bool {
            if (!clean && w.tail(w.j0 + i)) {
              if (!lpc::mbar_wait(fixed, fixes & 1u, st)) return false;
              ++fixes;
              clean = true;
            }
            const bool first = WIDE ? i == 0 : i < 2;
            if (!issue_pv(t, v_at(ring, i, n), first, WIDE ? t == 1 : true)) return false;
            // the stream's last: O is complete
            if (WIDE ? i == n - 1 : i + 2 >= n) lpc::umma_commit(o_done(t));
            return true;
          };
          auto o_ready = [&]() -> bool {
            ready = r == 0 || lpc::mbar_wait(o_free, (uint32_t)(r - 1) & 1u, st);
            if (ready) ask(0);
            if (ready && !WIDE) ask(1);  // their scores are on the way
            return ready;
          };
          if constexpr (WIDE) {
            ok = scores(0, 0) && scores(1, 0) && o_ready();
            for (int i = 0; i < n && ok; ++i) {
              ok = values(0, i) && (i + 1 >= n || scores(0, i + 1)) && values(1, i) &&
                   (i + 1 >= n || scores(1, i + 1));
            }
          } else {
            ok = scores(0, 0) && (n < 2 || scores(1, 1)) && o_ready();
            for (int i = 0; i < n && ok; ++i)
              ok = values(i & 1, i) && (i + 2 >= n || scores(i & 1, i + 2));
          }
          ring += 2u * (uint32_t)n;
          ++r;
        }
      }
    } else {
      // ---------------- V rows of the tiles at the end of a sequence ----------------
      bool ok = true;
      uint32_t ring = 0, fixes = 0;
      Walk w(p, sh, pos, stop, seq_first, seq);
      while (ok && w.next()) {
        const int tails = w.tails();
        // nodes that the sequence has no rows for: looked at where its last tile is, which need
        // not be a tail (a context that fills its rows and ends with a tile)
        const bool past = w.s.end - w.s.n < p.nodes && w.kvh == 0 && w.rb == 0 &&
                          w.j0 + w.count == w.s.tiles;
        uint64_t seen = 0;  // by any node
        if (tails || past) {
          for (int t = lane; t < p.nodes; t += 32)
            seen |= (uint64_t)p.masks[w.b * p.masks_stride + t];
#pragma unroll
          for (int m = 16; m; m >>= 1) seen |= __shfl_xor_sync(~0u, seen, m);
          if (past && (seen & node_bits(p.nodes) & ~node_bits(w.s.end - w.s.n)) && lane == 0)
            atomicOr(&g_tree_status, LPC_DEV_ERR_BOUNDS);  // a visible node past the rows
          seen &= node_bits(w.s.end - w.s.n);
        }
        if (tails) {
          // asked for only once the epilogue before has read sh.bad
          ok = __all_sync(~0u, lpc::mbar_wait(to_fix, fixes & 1u, st));
          if (!ok) break;
          ++fixes;
          uint64_t bad = 0;
          for (int i = w.count - tails; i < w.count && ok; ++i) {
            // both tails at most: the ring holds them side by side
            const uint32_t at = v_at(ring, i, w.count);
            ok = __all_sync(~0u, lpc::mbar_wait(full(at), slot_parity(at), st));
            if (!ok) break;
            // A row is LANES 16-byte pieces, one a lane.  Rows behind the nodes are overwritten
            // unread, nodes are looked at four rows at a time: the last product of an item
            // and its epilogue wait for this (6000 cycles a row after a row, of the 8800
            // from the last softmax to the next item's).
            const int first = (w.j0 + i) * KEYS - w.s.n;  // row 0 as a node
            uint8_t* tile = smem_raw + (slot(at) - raw);
            constexpr int LANES = HD / 8, AT_ONCE = 32 / LANES, BATCH = 4;
            const int sub = lane / LANES, part = lane % LANES;
            const int mine = (warp - 10) * AT_ONCE + sub;
            auto piece = [&](int q) {
              return reinterpret_cast<uint4*>(tile + (part / 8) * HALF_BYTES + q * 128) + part % 8;
            };
            const int from = max(0, -first);                     // the first node's row
            const int to = min(KEYS, w.s.end - w.s.n - first);   // behind the last one's
#pragma unroll 8
            for (int q = max(from, to) + mine; q < KEYS; q += 2 * AT_ONCE)
              *piece(q) = make_uint4(0, 0, 0, 0);
            for (int q0 = from; q0 < to; q0 += 2 * AT_ONCE * BATCH) {
              uint4 v[BATCH];
              bool clear[BATCH];
#pragma unroll
              for (int u = 0; u < BATCH; ++u) {
                const int q = q0 + mine + 2 * AT_ONCE * u;
                v[u] = make_uint4(0, 0, 0, 0);
                clear[u] = q < to && !(seen >> (first + q) & 1);  // nobody sees it
                if (q < to) v[u] = *piece(q);
              }
#pragma unroll
              for (int u = 0; u < BATCH; ++u) {
                const int q = q0 + mine + 2 * AT_ONCE * u;
                constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7c007c00u : 0x7f807f80u;
                auto inf = [&](uint32_t x) {
                  const uint32_t m = x & e;
                  return (m & 0xffffu) == (e & 0xffffu) || (m >> 16) == (e >> 16);
                };
                const bool odd = !clear[u] && (inf(v[u].x) || inf(v[u].y) || inf(v[u].z) || inf(v[u].w));
                // the whole row goes by any of its pieces
                const unsigned row = (LANES == 32 ? ~0u : ((1u << LANES) - 1u)) << (sub * LANES);
                if (__ballot_sync(~0u, odd) & row) {
                  clear[u] = true;
                  bad |= 1ull << (first + q);
                }
                if (clear[u]) *piece(q) = make_uint4(0, 0, 0, 0);
              }
            }
          }
          lpc::fence_proxy_async_smem();
#pragma unroll
          for (int m = 16; m; m >>= 1) bad |= __shfl_xor_sync(~0u, bad, m);
          if (lane == 0) sh.bad[warp - 10] = bad;
          __syncwarp();
          if (lane == 0) lpc::mbar_arrive(fixed);
        }
        ring += 2u * (uint32_t)w.count;
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;\n" ::: "memory");
    // ---------------- softmax and epilogue of stream t ----------------
    const int t = warp >> 2;
    const int rr = (warp & 3) * 32 + lane;  // row of the tile = TMEM lane
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + 128u * t + lane_off;
    bool ok = true;
    uint32_t tiles_done = 0, fixes = 0, twos = 0;  // tiles; segments with tails, of both streams
    int r = 0;
    auto wait_warp = [&](uint32_t bar, uint32_t parity) -> bool {  // the same for the warp
      return __all_sync(~0u, lpc::mbar_wait(bar, parity, st));
    };
    const int all_rows = p.group * p.nodes;
    Walk w(p, sh, pos, stop, seq_first, seq);
    while (ok && w.next()) {
      const int n = w.count;
      const int row = w.rb * S::ITEM_ROWS + (WIDE ? t * ROWS : 0) + rr;  // of the KV head's
      const bool valid = row < all_rows;
      const bool busy = __any_sync(~0u, valid);  // warps of padding only keep the barriers going
      const int head = valid ? row / p.nodes : 0, node = valid ? row - head * p.nodes : 0;
      const uint64_t visible =
          valid ? (uint64_t)p.masks[w.b * p.masks_stride + node] & node_bits(w.s.end - w.s.n) : 0;
      float m_used = -INFINITY, l = 0.f;
      const int step = WIDE ? 1 : 2;
      int mine = 0;  // tiles of this stream so far
      for (int i = WIDE ? 0 : t; i < n; i += step, ++mine) {
        const uint32_t ph = (tiles_done + (uint32_t)mine) & 1u;
        if (!(ok = wait_warp(s_full(t), ph))) break;
        if (!busy) {
          if (lane == 0) {
            lpc::mbar_arrive(p_half(t));
            lpc::mbar_arrive(p_full(t));
          }
          continue;
        }
        lpc::tc_fence_after();
        uint32_t sv[KEYS];
#pragma unroll
        for (int cc = 0; cc < KEYS; cc += 32)
          lpc::tmem_ld32(tS + cc, *reinterpret_cast<uint32_t(*)[32]>(&sv[cc]));
        lpc::tmem_wait_ld();
        if (w.tail(w.j0 + i)) {
          // bits of the tile's keys that this row sees: context below `rel`, nodes from it
          const int rel = w.s.n - (w.j0 + i) * KEYS;  // in (-64, 128)
          uint32_t see[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int sh = 32 * x - rel;  // bit 0 of the word is node sh
            uint32_t bits = sh >= 64 ? 0u : sh >= 0 ? (uint32_t)(visible >> sh)
                            : sh > -32 ? (uint32_t)visible << -sh : 0u;
            const int ctx = rel - 32 * x;  // keys of the word that are context
            bits |= ctx >= 32 ? ~0u : ctx > 0 ? (1u << ctx) - 1u : 0u;
            see[x] = bits;
          }
#pragma unroll
          for (int q = 0; q < KEYS; ++q)
            if (!(see[q >> 5] >> (q & 31) & 1u)) sv[q] = 0xff800000u;  // -inf
        }
        float m0 = -INFINITY, m1 = -INFINITY, m2 = -INFINITY, m3 = -INFINITY;
#pragma unroll
        for (int q = 0; q < KEYS; q += 8) {
          m0 = max3(m0, __uint_as_float(sv[q]), __uint_as_float(sv[q + 1]));
          m1 = max3(m1, __uint_as_float(sv[q + 2]), __uint_as_float(sv[q + 3]));
          m2 = max3(m2, __uint_as_float(sv[q + 4]), __uint_as_float(sv[q + 5]));
          m3 = max3(m3, __uint_as_float(sv[q + 6]), __uint_as_float(sv[q + 7]));
        }
        const float top = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3)) * p.scale_log2;  // scale > 0
        // S of this tile was issued after PV of the stream's tile before: O is stable
        const bool grow = top > m_used + (GROWTH + RAISE<T>) || (m_used == -INFINITY && top > -INFINITY);
        if (__any_sync(~0u, grow)) {
          float alpha = 1.f;
          if (grow) {
            const float now = top - RAISE<T>;
            alpha = m_used == -INFINITY ? 0.f : fast_exp2(m_used - now);
            m_used = now;
            l *= alpha;
          }
          if (mine > 0) {
            const uint32_t tO = tmem + 256u + 128u * t + lane_off;
#pragma unroll 1
            for (int cc = 0; cc < HD; cc += 16) {
              uint32_t v[16];
              lpc::tmem_ld16(tO + cc, v);
              lpc::tmem_wait_ld();
#pragma unroll
              for (int q = 0; q < 16; ++q) v[q] = __float_as_uint(__uint_as_float(v[q]) * alpha);
              lpc::tmem_st16(tO + cc, v);
            }
          }
        }
        const float m_use = m_used == -INFINITY ? 0.f : m_used;
        const uint64_t sc2 = pack_f2(p.scale_log2, p.scale_log2), nm2 = pack_f2(-m_use, -m_use);
        uint64_t rsa = 0, rsb = 0;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t pk[KEYS / 4];
#pragma unroll
          for (int q = 0; q < KEYS / 2; q += 2) {
            const int at = half * (KEYS / 2) + q;
            const uint64_t x = fma_f2(pack_f2(__uint_as_float(sv[at]), __uint_as_float(sv[at + 1])),
                                      sc2, nm2);
            const uint64_t e = pack_f2(fast_exp2(lo_f(x)), fast_exp2(hi_f(x)));
            if ((q >> 1) & 1) rsb = add_f2(rsb, e);
            else rsa = add_f2(rsa, e);
            pk[q >> 1] = pack2<T>(lo_f(e), hi_f(e));
          }
#pragma unroll
          for (int cc = 0; cc < KEYS / 4; cc += 16)
            lpc::tmem_st16(tS + (uint32_t)(half * (KEYS / 4) + cc),
                           *reinterpret_cast<uint32_t(*)[16]>(&pk[cc]));
          lpc::tmem_wait_st();
          lpc::tc_fence_before();
          __syncwarp();
          if (lane == 0) lpc::mbar_arrive(half ? p_full(t) : p_half(t));
        }
        const uint64_t rs2 = add_f2(rsa, rsb);
        l += lo_f(rs2) + hi_f(rs2);
      }
      tiles_done += (uint32_t)mine;
      if (!ok) break;

      // ---- epilogue ----
      const bool two = !WIDE && n > 1;  // both streams have part of these rows
      float M = m_used, L = l, a0 = 1.f, a1 = 0.f;
      if constexpr (!WIDE) {
        // the segment before has been read
        if (r > 0 && !(ok = wait_warp(o_free, (uint32_t)(r - 1) & 1u))) break;
        sh.ml[t][rr] = make_float2(m_used, l);
        __syncwarp();
        if (lane == 0) lpc::mbar_arrive(ml_full);
        if (!(ok = wait_warp(ml_full, (uint32_t)r & 1u))) break;
        const float2 x0 = sh.ml[0][rr], x1 = sh.ml[1][rr];
        M = fmaxf(x0.x, x1.x);
        const float mu = M == -INFINITY ? 0.f : M;
        a0 = fast_exp2(x0.x - mu);
        a1 = two ? fast_exp2(x1.x - mu) : 0.f;
        L = x0.y * a0 + (two ? x1.y * a1 : 0.f);
      }
      unsigned long long bad = 0;
      if (w.tails()) {
        if (!(ok = wait_warp(fixed, fixes & 1u))) break;
        ++fixes;
        bad = (*(volatile unsigned long long*)&sh.bad[0] | *(volatile unsigned long long*)&sh.bad[1]) &
              visible;
      }
      // narrow: both streams' O, columns shared out to the two warpgroups
      if (!(ok = wait_warp(o_done(WIDE ? t : 0), (uint32_t)r & 1u))) break;
      if (two) {
        if (!(ok = wait_warp(o_done(1), twos & 1u))) break;
        ++twos;
      }
      // the part goes where the ring was: nothing may still read it
      if (WIDE && joined && !(ok = wait_warp(o_done(1 - t), (uint32_t)r & 1u))) break;
      lpc::tc_fence_after();
      constexpr int COLS = WIDE ? HD : HD / 2;
      const int col0 = WIDE ? 0 : t * COLS;
      if (!busy) {
        if (lane == 0) lpc::mbar_arrive(o_free);
      } else {
        const uint32_t tO0 = tmem + 256u + (WIDE ? 128u * t : 0u) + lane_off + col0;
        const float inv = L > 0.f || L != L ? 1.f / L : 0.f;
        T* orow = static_cast<T*>(p.out) + (((int64_t)w.b * p.nodes + node) * p.heads +
                                            w.kvh * p.group + head) * p.head_dim + col0;
        // parts: [four columns][row], a warp's rows are 512 bytes side by side
        float* part = joined ? reinterpret_cast<float*>(smem_raw + (sRing - raw))
                             : p.parts + (2 * (int64_t)c + (w.j0 == 0 ? 1 : 0)) * S::PART;
        const int prow = (WIDE ? t * ROWS : 0) + rr;
        if (valid && !w.whole && (WIDE || t == 0))
          reinterpret_cast<float2*>(part + (int64_t)S::ITEM_ROWS * HD)[prow] = make_float2(M, L);
#pragma unroll 1
        for (int cc = 0; cc < COLS; cc += 32) {
          uint32_t o[32];
          __syncwarp();  // rows part below; the reads are the whole warp's
          lpc::tmem_ld32(tO0 + cc, o);
          if (two) {
            uint32_t v[32];
            lpc::tmem_ld32(tO0 + 128u + cc, v);
            lpc::tmem_wait_ld();
#pragma unroll
            for (int q = 0; q < 32; ++q)
              o[q] = __float_as_uint(__uint_as_float(o[q]) * a0 + __uint_as_float(v[q]) * a1);
          }
          lpc::tmem_wait_ld();
          if (cc + 32 == COLS) {  // the next segment's first PV may overwrite O
            lpc::tc_fence_before();
            __syncwarp();
            if (lane == 0) lpc::mbar_arrive(o_free);
          }
          if (!valid || col0 + cc >= p.head_dim) continue;
          if (bad) {
            // visible V rows that are not finite: cleared in the tile, added here
            for (unsigned long long left = bad; left; left &= left - 1) {
              const int j = __ffsll((long long)left) - 1;
              const int at = (j + w.s.n) / KEYS;
              if (at < w.j0 || at >= w.j0 + n) continue;  // in another part of the item
              const int64_t head_rows = p.seq_base ? p.total_rows : p.max_seq_len;
              const int64_t krow = (w.s.row0 + w.kvh * head_rows + w.s.n + j) * p.head_dim;
              const T* kr = static_cast<const T*>(p.k) + krow;
              const T* vr = static_cast<const T*>(p.v) + krow + col0 + cc;
              const T* qr = static_cast<const T*>(p.q) +
                            ((int64_t)(w.b * p.kv_heads + w.kvh) * all_rows + row) * p.head_dim;
              float dot = 0.f;
              for (int d = 0; d < p.head_dim; ++d)
                dot = fmaf(Num<T>::to_f(qr[d]), Num<T>::to_f(kr[d]), dot);
              const float pj = fast_exp2(dot * p.scale_log2 - (M == -INFINITY ? 0.f : M));
#pragma unroll
              for (int q = 0; q < 32; ++q)
                o[q] = __float_as_uint(fmaf(pj, Num<T>::to_f(vr[q]), __uint_as_float(o[q])));
            }
          }
          if (w.whole) {
#pragma unroll
            for (int q = 0; q < 32; q += 8) {
              uint32_t pk[4];
#pragma unroll
              for (int x = 0; x < 4; ++x)
                pk[x] = pack2<T>(__uint_as_float(o[q + 2 * x]) * inv, __uint_as_float(o[q + 2 * x + 1]) * inv);
              *reinterpret_cast<uint4*>(orow + cc + q) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
            }
          } else {
            uint4* dst = reinterpret_cast<uint4*>(part) + (col0 + cc) / 4 * S::ITEM_ROWS + prow;
#pragma unroll
            for (int q = 0; q < 8; ++q)
              dst[q * S::ITEM_ROWS] = make_uint4(o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]);
          }
        }
      }
      ++r;
    }
  }
  lpc::tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    lpc::tc_fence_after();
    lpc::tmem_dealloc(tmem, TMEM_COLS);
  }
  if (joined) {
    // every CTA joins its share of the rows
    __syncwarp();
    lpc::cluster_sync();
    const uint32_t n = (uint32_t)p.cluster, tiles = (uint32_t)sh.known[0].tiles;
    const uint32_t item = c / n, rank = c - item * n;
    const int rb = (int)(item % (uint32_t)p.row_blocks);
    const int kvh = (int)(item / (uint32_t)p.row_blocks) - seq * p.kv_heads;
    const int rows = min(S::ITEM_ROWS, p.group * p.nodes - rb * S::ITEM_ROWS);
    const int r0 = rows * (int)rank / (int)n, mine = rows * (int)(rank + 1) / (int)n - r0;
    const uint32_t part = sRing;
    for (int x = (int)threadIdx.x; x < mine * (p.head_dim / 4); x += NTHREADS) {
      const int group = x / mine, prow = r0 + x - group * mine;
      float2 ml[8];
      float4 v[8];
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i) {
        ml[i] = make_float2(-INFINITY, 0.f);
        v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i < n && tiles * i / n < tiles * (i + 1) / n) {  // it has tiles
          const uint32_t from = lpc::mapa_shared(part, i);
          v[i] = ld_remote16(from + 16u * (uint32_t)(group * S::ITEM_ROWS + prow));
          ml[i] = ld_remote8(from + 4u * S::ITEM_ROWS * HD + 8u * (uint32_t)prow);
        }
      }
      float M = ml[0].x;
#pragma unroll
      for (int i = 1; i < 8; ++i) M = fmaxf(M, ml[i].x);
      const float mu = M == -INFINITY ? 0.f : M;
      float L = 0.f;
      float4 all[1] = {make_float4(0.f, 0.f, 0.f, 0.f)};
      float4& o = all[0];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float f = fast_exp2(ml[i].x - mu);
        L = fmaf(f, ml[i].y, L);
        o.x = fmaf(f, v[i].x, o.x);
        o.y = fmaf(f, v[i].y, o.y);
        o.z = fmaf(f, v[i].z, o.z);
        o.w = fmaf(f, v[i].w, o.w);
      }
      store_row<T, 1>(p, seq, kvh, rb * S::ITEM_ROWS + prow, 4 * group, all, L);
    }
    lpc::cluster_sync();  // a CTA's memory stays until all have read it
  }
}

// Joins the parts of an item: the second part of the CTA that began it and the first part of
// each CTA after it up to the last.  blockIdx.x is the item, or, where there are more of them
// than CTAs, the CTA that began it.  A thread has eight or four columns of a row and every
// LANES-th part, two or four of them in flight; a warp reads rows side by side.  It is bound
// by instructions: with four columns a thread throughout, 256 items of 96 rows and two to three
// parts took 6.3 us, so 4.6.
template <int HD, int LANES>
struct Join {
  static constexpr int THREADS = LANES == 1 ? 256 : 512;
  static constexpr int FOURS = LANES == 1 ? 2 : 1;   // four columns each, a thread
  static constexpr int GROUPS = HD / (4 * FOURS);
  static constexpr int ROWS_HERE = THREADS / (GROUPS * LANES);
  static constexpr int BATCH = LANES == 1 ? 2 : 4;   // parts in flight a thread
  static constexpr int BLOCKS = LANES == 1 ? 6 : 2;  // an SM
};
template <typename T, int HD, bool WIDE, int LANES>
__global__ void __launch_bounds__(Join<HD, LANES>::THREADS, Join<HD, LANES>::BLOCKS)
    tree_join_kernel(const Params p, int ctas) {
  using S = Shape<HD, WIDE>;
  using J = Join<HD, LANES>;
  constexpr int GROUPS = J::GROUPS, ROWS_HERE = J::ROWS_HERE, FOURS = J::FOURS, BATCH = J::BATCH;
  lpc::pdl_trigger();
  lpc::pdl_wait();
  int item, c0, last;  // its first and last CTA
  if (p.batch * p.kv_heads * p.row_blocks > ctas) {
    c0 = (int)blockIdx.x;
    const uint2 begun = lpc::ld_dep8(&p.split[c0]);
    item = (int)begun.x;
    last = (int)begun.y;
  } else {
    __shared__ int2 s_split;  // first and last CTA
    if (threadIdx.x == 0) s_split.x = -1;
    __syncthreads();
    for (int c = (int)threadIdx.x; c < ctas; c += (int)blockDim.x) {
      const uint2 begun = lpc::ld_dep8(&p.split[c]);
      if (begun.x == blockIdx.x) s_split = make_int2(c, (int)begun.y);
    }
    __syncthreads();
    c0 = s_split.x;
    last = s_split.y;
    item = c0 < 0 ? -1 : (int)blockIdx.x;
  }
  if (item < 0) return;
  const int rb = item % p.row_blocks, pair = item / p.row_blocks;
  const int b = pair / p.kv_heads, kvh = pair - b * p.kv_heads;
  const int prow = (int)blockIdx.y * ROWS_HERE + (int)threadIdx.x % ROWS_HERE;
  const int group = (int)threadIdx.x / ROWS_HERE % GROUPS;
  const int which = (int)threadIdx.x / (ROWS_HERE * GROUPS);  // of the LANES
  const int row = rb * S::ITEM_ROWS + prow;
  const bool in = prow < S::ITEM_ROWS && row < p.group * p.nodes && 4 * FOURS * group < p.head_dim;
  float M = -INFINITY, L = 0.f;
  float4 o[FOURS];
#pragma unroll
  for (int f = 0; f < FOURS; ++f) o[f] = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](float m, float l, const float4 (&v)[FOURS]) {  // one more part
    const float top = fmaxf(M, m), mu = top == -INFINITY ? 0.f : top;
    const float a = fast_exp2(M - mu), w = fast_exp2(m - mu);
    M = top;
    L = L * a + w * l;
#pragma unroll
    for (int f = 0; f < FOURS; ++f) {
      o[f].x = o[f].x * a + w * v[f].x;
      o[f].y = o[f].y * a + w * v[f].y;
      o[f].z = o[f].z * a + w * v[f].z;
      o[f].w = o[f].w * a + w * v[f].w;
    }
  };
  if (in)
    for (int c = c0 + which; c <= last; c += BATCH * LANES) {
      float2 x[BATCH];
      float4 v[BATCH][FOURS];
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const int at = min(c + i * LANES, last);
        const float* part = p.parts + (2 * (int64_t)at + (at == c0 ? 1 : 0)) * S::PART;
        x[i] = reinterpret_cast<const float2*>(part + (int64_t)S::ITEM_ROWS * HD)[prow];
#pragma unroll
        for (int f = 0; f < FOURS; ++f)
          v[i][f] = reinterpret_cast<const float4*>(part)[(FOURS * group + f) * S::ITEM_ROWS + prow];
      }
#pragma unroll
      for (int i = 0; i < BATCH; ++i)
        if (c + i * LANES <= last) add(x[i].x, x[i].y, v[i]);
    }
  if constexpr (LANES > 1) {
    constexpr int HERE = ROWS_HERE * GROUPS;
    __shared__ float4 s_o[LANES][HERE][FOURS];
    __shared__ float2 s_ml[LANES][HERE];
    const int at = (int)threadIdx.x % HERE;
#pragma unroll
    for (int f = 0; f < FOURS; ++f) s_o[which][at][f] = o[f];
    s_ml[which][at] = make_float2(M, L);
    __syncthreads();
    if (which) return;
#pragma unroll
    for (int i = 1; i < LANES; ++i) add(s_ml[i][at].x, s_ml[i][at].y, s_o[i][at]);
  }
  if (in) store_row<T, FOURS>(p, b, kvh, row, 4 * FOURS * group, o, L);
}

// CTAs of a call: one an SM, no more than there can be tiles.
int64_t grid_of(int64_t batch, int64_t items_a_sequence, int64_t max_seq_len, int64_t total_rows,
                int sms) {
  const int64_t tiles = total_rows > 0 ? total_rows / KEYS + batch
                                       : batch * ((max_seq_len + KEYS - 1) / KEYS);
  return std::min<int64_t>(sms, tiles * items_a_sequence);
}

bool sizes_ok(int64_t batch, int64_t nodes, int heads, int kv_heads, int head_dim,
              int64_t max_seq_len, int64_t total_rows) {
  return batch >= 0 && batch <= 65535 && nodes >= 1 && nodes <= MAX_NODES && heads > 0 &&
         heads <= 65535 && kv_heads > 0 && heads % kv_heads == 0 &&
         (head_dim == 32 || head_dim == 64 || head_dim == 128) &&
         (total_rows > 0 ? total_rows <= 0x7fffffffLL - KEYS
                         : max_seq_len > 0 && max_seq_len <= 0x7fffffffLL - KEYS);
}

// Clusters of 1 << e CTAs that the device runs at once: one CTA an SM, clusters within
// the groups of SMs that the hardware has.
int clusters_at_once(int e, int sms) {
  static std::atomic<int> cache[64][4];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) {
    cudaGetLastError();
    return std::max(1, sms >> e);
  }
  int v = cache[dev][e].load(std::memory_order_relaxed);
  if (v > 0) return v;
  using S = Shape<128, false>;
  static std::atomic<uint64_t> mask{0};
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1u << e;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(1u << e);
  cfg.blockDim = dim3(NTHREADS);
  cfg.dynamicSmemBytes = S::SMEM;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const auto kernel = tree_attention_kernel<__nv_bfloat16, 128, false>;
  if (lpc::once_per_device_smem((const void*)kernel, S::SMEM, mask) != LPC_OK ||
      cudaOccupancyMaxActiveClusters(&v, kernel, &cfg) != cudaSuccess || v <= 0) {
    cudaGetLastError();
    v = std::max(1, sms >> e);
  }
  cache[dev][e].store(v, std::memory_order_relaxed);
  return v;
}

constexpr int SAVED = 5;

struct Plan {
  bool wide;
  int row_blocks;
  int64_t grid, part_floats;
  int cluster; // CTAs an item (0: stretches)
  bool join;   // stretches, and some item may have more than one tile
  bool fits;   // units and items are 31-bit numbers
};
Plan plan_of(int64_t batch, int64_t nodes, int heads, int kv_heads, int head_dim,
             int64_t max_seq_len, int64_t total_rows) {
  Plan x;
  const int64_t rows = (int64_t)(heads / kv_heads) * nodes;
  x.wide = rows > ROWS;
  const int item_rows = x.wide ? 2 * ROWS : ROWS;
  x.row_blocks = (int)((rows + item_rows - 1) / item_rows);
  const int sms = lpc::current_device_sms();
  const int64_t items = batch * kv_heads * x.row_blocks;
  const int64_t tiles = ((total_rows > 0 ? total_rows : max_seq_len) + KEYS - 1) / KEYS;  // an item's, at most
  // A cluster an item, as many CTAs as one wave has; against stretches, of which the second
  // kernel costs about as much as SAVED tiles.  A CTA's own begin costs a tile more than an
  // item's: of 8 KV heads of 64 rows and up to 250 keys, 32 sequences take 18.8 us (stretches
  // 21.9), 64 35.0 (35.9), 128 65.3 (61.6); of up to 120 keys, where nothing is joined, 32
  // take 16.4 (14.6) and 128 56.2 (41.1).
  int e = 0;
  while (e < 3 && (1 << e) < tiles && items <= clusters_at_once(e + 1, sms)) ++e;
  const int64_t at_once = clusters_at_once(e, sms), n = 1 << e;
  const int64_t waves = (items + at_once - 1) / at_once;
  const int64_t of_cluster = waves * ((tiles + n - 1) / n + START + 1) - 1;
  const int64_t of_stretch = (items * (tiles + START) + sms - 1) / sms + (tiles > 1 ? SAVED : 0);
  x.cluster = of_cluster <= of_stretch ? (int)n : 0;
  x.grid = x.cluster ? items * x.cluster
                     : grid_of(batch, (int64_t)kv_heads * x.row_blocks, max_seq_len, total_rows, sms);
  x.part_floats = (int64_t)item_rows * ((head_dim == 128 ? 128 : 64) + 2);
  x.join = !x.cluster && tiles > 1;
  const int64_t per = (int64_t)kv_heads * x.row_blocks;
  x.fits = batch * (tiles + START) <= 0x7fffffffLL / per;
  return x;
}

template <typename T, int HD, bool WIDE>
int launch(const TmaDesc4& tq, const TmaDesc4& tk, const TmaDesc4& tv, const Params& p,
           const Plan& plan, uint32_t id_qk, uint32_t id_pv, cudaStream_t s) {
  using S = Shape<HD, WIDE>;
  static std::atomic<int> regs{0};
  int have = regs.load(std::memory_order_relaxed);
  if (have == 0) {
    cudaFuncAttributes fa;
    have = cudaFuncGetAttributes(&fa, tree_attention_kernel<T, HD, WIDE>) == cudaSuccess ? fa.numRegs
                                                                                         : -1;
    regs.store(have, std::memory_order_relaxed);
  }
  if (have != LAUNCH_REGS) {
    lpc::set_error("tree_attention: kernel built with %d registers per thread, its register split "
                   "needs %d", have, LAUNCH_REGS);
    return LPC_ERR_UNSUPPORTED;
  }
  static std::atomic<uint64_t> mask{0};
  if (int rc = lpc::once_per_device_smem((const void*)tree_attention_kernel<T, HD, WIDE>, S::SMEM, mask))
    return rc;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = lpc::use_pdl() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)plan.cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)plan.grid);
  cfg.blockDim = dim3(NTHREADS);
  cfg.dynamicSmemBytes = S::SMEM;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = plan.cluster > 1 ? 2 : 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, tree_attention_kernel<T, HD, WIDE>, tq, tk, tv, p, id_qk,
                                     id_pv);
  if (e == cudaSuccess && plan.join) {
    // few items have many parts each: eight threads share them (one KV head of 32,000 keys,
    // 148 parts: 28 us in all, 63 by one thread)
    const int64_t items = (int64_t)p.batch * p.kv_heads * p.row_blocks;
    const bool many = plan.grid > 8 * items;
    const int here = many ? Join<HD, 8>::ROWS_HERE : Join<HD, 1>::ROWS_HERE;
    const int rows = std::min(p.group * p.nodes, S::ITEM_ROWS);
    cfg.gridDim = dim3((unsigned)std::min(items, plan.grid), (unsigned)((rows + here - 1) / here));
    cfg.blockDim = dim3(many ? Join<HD, 8>::THREADS : Join<HD, 1>::THREADS);
    cfg.dynamicSmemBytes = 0;
    e = many ? cudaLaunchKernelEx(&cfg, tree_join_kernel<T, HD, WIDE, 8>, p, (int)plan.grid)
             : cudaLaunchKernelEx(&cfg, tree_join_kernel<T, HD, WIDE, 1>, p, (int)plan.grid);
  }
  if (e != cudaSuccess) {
    lpc::set_error("tree_attention: launch failed: %s", cudaGetErrorString(e));
    return LPC_ERR_CUDA;
  }
  return lpc::check_launch("tree_attention");
}

template <typename T>
int launch_t(const TmaDesc4& tq, const TmaDesc4& tk, const TmaDesc4& tv, const Params& p,
             const Plan& plan, uint32_t fmt, cudaStream_t s) {
  const int hd = p.head_dim == 128 ? 128 : 64;
  const uint32_t qk = lpc::idesc_f16(fmt, ROWS, KEYS, 0u, 0u);
  const uint32_t pv = lpc::idesc_f16(fmt, ROWS, (uint32_t)hd, 0u, 1u);
  if (hd == 128)
    return plan.wide ? launch<T, 128, true>(tq, tk, tv, p, plan, qk, pv, s)
                     : launch<T, 128, false>(tq, tk, tv, p, plan, qk, pv, s);
  return plan.wide ? launch<T, 64, true>(tq, tk, tv, p, plan, qk, pv, s)
                   : launch<T, 64, false>(tq, tk, tv, p, plan, qk, pv, s);
}

}  // namespace

extern "C" int64_t lpc_tree_attention_workspace_bytes(int64_t batch, int nodes, int heads,
                                                      int kv_heads, int head_dim,
                                                      int64_t max_seq_len, int64_t total_rows) {
  if (!sizes_ok(batch, nodes, heads, kv_heads, head_dim, max_seq_len, total_rows) || batch == 0)
    return 0;
  const Plan x = plan_of(batch, nodes, heads, kv_heads, head_dim, max_seq_len, total_rows);
  return x.join && x.fits ? x.grid * (2 * x.part_floats * 4 + 16) : 0;
}

extern "C" int lpc_tree_attention(const void* q, const void* key_cache, const void* value_cache,
                                  const int32_t* seq_lens, const int64_t* masks,
                                  int64_t masks_stride, const int64_t* seq_base,
                                  const int32_t* seq_cap, void* out, void* workspace,
                                  int64_t workspace_bytes, int64_t batch, int nodes, int heads,
                                  int kv_heads, int head_dim, int64_t max_batch,
                                  int64_t max_seq_len, int64_t total_rows, float sm_scale,
                                  int dtype, void* stream) {
  using namespace lpc;
  if (dtype != LPC_DTYPE_BF16 && dtype != LPC_DTYPE_F16) {
    set_error("tree_attention: only bf16 and fp16 are supported");
    return LPC_ERR_UNSUPPORTED;
  }
  if (head_dim != 32 && head_dim != 64 && head_dim != 128) {
    set_error("tree_attention: head_dim must be 32, 64 or 128, got %d", head_dim);
    return LPC_ERR_UNSUPPORTED;
  }
  if ((seq_base != nullptr) != (seq_cap != nullptr) || (seq_base != nullptr) != (total_rows > 0)) {
    set_error("tree_attention: a ragged cache has seq_base, seq_cap and total_rows");
    return LPC_ERR_INVALID;
  }
  if (!sizes_ok(batch, nodes, heads, kv_heads, head_dim, max_seq_len, total_rows) ||
      (masks_stride != 0 && masks_stride < nodes) || (!seq_base && batch > max_batch)) {
    set_error("tree_attention: invalid sizes (batch=%lld of %lld, nodes=%d, heads=%d, kv_heads=%d, "
              "max_seq_len=%lld, total_rows=%lld; 1 to %d nodes)", (long long)batch,
              (long long)max_batch, nodes, heads, kv_heads, (long long)max_seq_len,
              (long long)total_rows, MAX_NODES);
    return LPC_ERR_INVALID;
  }
  if (!(sm_scale > 0.f && sm_scale < INFINITY)) {
    set_error("tree_attention: sm_scale must be positive");
    return LPC_ERR_INVALID;
  }
  if (batch == 0) return LPC_OK;
  if (!q || !key_cache || !value_cache || !seq_lens || !masks || !out) {
    set_error("tree_attention: null pointer");
    return LPC_ERR_INVALID;
  }
  if (!aligned16(q) || !aligned16(key_cache) || !aligned16(value_cache) || !aligned16(out)) {
    set_error("tree_attention: tensors must be 16-byte aligned");
    return LPC_ERR_INVALID;
  }
  const Plan plan = plan_of(batch, nodes, heads, kv_heads, head_dim, max_seq_len, total_rows);
  if (!plan.fits) {
    set_error("tree_attention: %lld sequences of these caches are too many tiles", (long long)batch);
    return LPC_ERR_UNSUPPORTED;
  }
  const int64_t need = plan.join ? plan.grid * (2 * plan.part_floats * 4 + 16) : 0;
  if (need && (!workspace || workspace_bytes < need || !aligned16(workspace))) {
    set_error("tree_attention: workspace of %lld bytes required, got %lld", (long long)need,
              (long long)workspace_bytes);
    return LPC_ERR_INVALID;
  }
  Params p;
  p.q = q;
  p.k = key_cache;
  p.v = value_cache;
  p.out = out;
  p.seq_lens = seq_lens;
  p.masks = masks;
  p.masks_stride = masks_stride;
  p.seq_base = seq_base;
  p.seq_cap = seq_cap;
  p.max_seq_len = max_seq_len;
  p.total_rows = total_rows;
  // the parts lie behind 16 bytes a CTA: they are 16-byte vectors
  p.split = plan.join ? static_cast<int2*>(workspace) : nullptr;
  p.parts = plan.join ? reinterpret_cast<float*>(p.split + 2 * plan.grid) : nullptr;
  p.batch = (int)batch;
  p.nodes = nodes;
  p.heads = heads;
  p.kv_heads = kv_heads;
  p.group = heads / kv_heads;
  p.head_dim = head_dim;
  p.row_blocks = plan.row_blocks;
  p.cluster = plan.cluster;
  p.scale_log2 = sm_scale * LOG2E;
  TmaDesc4 tq, tk, tv;
  const uint64_t rowb = (uint64_t)head_dim * 2;
  const uint32_t box[4] = {BOX, 128, 1, 1};
  {
    const uint64_t rows = (uint64_t)p.group * nodes, pairs = (uint64_t)batch * kv_heads;
    const uint64_t dims[4] = {(uint64_t)head_dim, rows, pairs, 1};
    const uint64_t str[3] = {rowb, rowb * rows, rowb * rows * pairs};
    if (int rc = make_tma_nd(reinterpret_cast<TmaDesc*>(&tq), q, dtype, 4, dims, str, box, true))
      return rc;
  }
  {
    const uint64_t rows = (uint64_t)(seq_base ? total_rows : max_seq_len);
    const uint64_t dims[4] = {(uint64_t)head_dim, rows, (uint64_t)kv_heads,
                              (uint64_t)(seq_base ? 1 : max_batch)};
    const uint64_t str[3] = {rowb, rowb * rows, rowb * rows * kv_heads};
    if (int rc = make_tma_nd(reinterpret_cast<TmaDesc*>(&tk), key_cache, dtype, 4, dims, str, box, true))
      return rc;
    if (int rc = make_tma_nd(reinterpret_cast<TmaDesc*>(&tv), value_cache, dtype, 4, dims, str, box, true))
      return rc;
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == LPC_DTYPE_BF16) return launch_t<__nv_bfloat16>(tq, tk, tv, p, plan, 1u, s);
  return launch_t<__half>(tq, tk, tv, p, plan, 0u, s);
}
