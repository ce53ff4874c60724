// Acceptance of a drafted tree: the branch that the samples agree with, and its
// K/V rows moved together in the caches of every layer.
//
// From the root the branch goes on, while it can, to the lowest child whose
// drafted token is the one sampled after the node.  Node path[i] of the branch
// has its K/V at row n + path[i] of its sequence (n keys before the tree); they
// move to row n + i.  Children stand behind their parents, so path rises and
// path[i] >= i: a thread that owns one 16-byte column of one (layer, K or V, KV
// head) and goes up the path never overwrites a row that it still has to read,
// and needs no other thread's.
//
// Every CTA walks the tree again (a warp, two nodes a lane, one ballot a step):
// cheaper than a second launch that waits for the first.  The bound is latency: the
// rows of a branch are a few kilobytes a layer.  One sequence, 16 nodes, 32 layers
// 3.1 us; 64 sequences of 64 nodes, whose branches move 207 rows of 32 layers (54 MB in
// and out, 8.3 us at the copy rate), 12.7 us.
#include "lpc_common.cuh"

LPC_DECLARE_STATUS(g_accept_status)

unsigned int lpc_status_tree_accept(bool clear) {
  unsigned int v = 0;
  cudaMemcpyFromSymbol(&v, g_accept_status, sizeof(v));
  if (clear && v) {
    unsigned int z = 0;
    cudaMemcpyToSymbol(g_accept_status, &z, sizeof(z));
  }
  return v;
}

namespace {

constexpr int MAX_NODES = 64;
constexpr int MAX_LAYERS = 128;  // a launch
constexpr int THREADS = 128;
// Rows in flight a thread, and CTAs an SM: four and twelve take 12.7 us where eight, whose
// registers leave room for seven CTAs, took 13.9 (64 sequences, 207 rows of 32 layers).
constexpr int BATCH = 4;
constexpr int BLOCKS = 12;

template <int LAYERS>
struct Caches {
  uint8_t* at[2 * LAYERS];  // K and V of each
};

struct Args {
  const int64_t *drafted, *sampled;
  const int32_t* parents;
  int64_t parents_stride;  // 0: one tree for all sequences
  const int32_t* seq_lens;
  const int64_t* seq_base;
  const int32_t* seq_cap;
  int32_t* accepted;
  int64_t* tokens;
  int32_t* path;
  int64_t max_seq_len, total_rows;
  int nodes, caches, kv_heads, columns;  // 16-byte columns of a row
  bool report;                           // this launch writes the results
};

template <int LAYERS>
__global__ void __launch_bounds__(THREADS, BLOCKS)
    tree_accept_kernel(const Args a, const __grid_constant__ Caches<LAYERS> caches) {
  __shared__ int32_t s_path[MAX_NODES];
  __shared__ int s_count;
  const int64_t b = blockIdx.y;
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int32_t parent[2];
    int64_t drafted[2], sampled[2];
    bool bad = false;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int t = lane + 32 * j;
      const bool in = t < a.nodes;
      parent[j] = in ? a.parents[b * a.parents_stride + t] : -1;
      drafted[j] = in ? a.drafted[b * a.nodes + t] : 0;
      sampled[j] = in ? a.sampled[b * a.nodes + t] : 0;
      bad |= in && t > 0 && parent[j] >= t;
      if (t == 0 || parent[j] >= t) parent[j] = -1;  // no child of an earlier node
    }
    int here = 0, count = 0;
    while (true) {  // nodes rise along the branch: at most 64 steps
      const int64_t mine = here < 32 ? sampled[0] : sampled[1];
      const int64_t said = (int64_t)__shfl_sync(~0u, (uint32_t)mine, here & 31) |
                           (int64_t)__shfl_sync(~0u, (uint32_t)(mine >> 32), here & 31) << 32;
      if (lane == 0) {
        s_path[count] = here;
        if (a.report && blockIdx.x == 0) {
          a.path[b * a.nodes + count] = here;
          a.tokens[b * a.nodes + count] = said;
        }
      }
      ++count;
      const unsigned lo = __ballot_sync(~0u, parent[0] == here && drafted[0] == said);
      const unsigned hi = __ballot_sync(~0u, parent[1] == here && drafted[1] == said);
      if (lo) here = __ffs(lo) - 1;
      else if (hi) here = 31 + __ffs(hi);
      else break;
    }
    if (lane == 0) s_count = count;
    if (a.report && blockIdx.x == 0) {
      for (int t = count + lane; t < a.nodes; t += 32) {
        a.path[b * a.nodes + t] = -1;
        a.tokens[b * a.nodes + t] = -1;
      }
      if (lane == 0) a.accepted[b] = count;
      if (__any_sync(~0u, bad) && lane == 0) atomicOr(&g_accept_status, LPC_DEV_ERR_BOUNDS);
    }
  }
  __syncthreads();
  const int count = s_count;
  if (a.caches == 0 || s_path[count - 1] == count - 1) return;  // the branch stands where it should
  // the sequence's rows
  const int64_t n = a.seq_lens[b];
  int64_t row, cap, head_rows;
  bool ok = n >= 0;
  if (a.seq_base) {
    const int64_t base = a.seq_base[b];
    cap = a.seq_cap[b];
    ok = ok && base >= 0 && cap >= 0 && base <= a.total_rows - cap;
    row = base + n;
    head_rows = a.total_rows;
  } else {
    cap = a.max_seq_len;
    row = b * a.kv_heads * a.max_seq_len + n;
    head_rows = a.max_seq_len;
  }
  ok = ok && n + s_path[count - 1] < cap;  // the branch's last row is its highest
  if (!ok) {
    if (blockIdx.x == 0 && threadIdx.x == 0) atomicOr(&g_accept_status, LPC_DEV_ERR_BOUNDS);
    return;
  }
  const int per_cache = a.kv_heads * a.columns;
  const int64_t work = (int64_t)a.caches * per_cache;
  for (int64_t w = (int64_t)blockIdx.x * THREADS + threadIdx.x; w < work;
       w += (int64_t)gridDim.x * THREADS) {
    const int c = (int)(w / per_cache), rest = (int)(w - (int64_t)c * per_cache);
    const int head = rest / a.columns, column = rest - head * a.columns;
    uint4* p = reinterpret_cast<uint4*>(caches.at[c]) + (row + head * head_rows) * a.columns + column;
    for (int i0 = 1; i0 < count; i0 += BATCH) {
      uint4 v[BATCH];
#pragma unroll
      for (int j = 0; j < BATCH; ++j)
        if (i0 + j < count) v[j] = p[(int64_t)s_path[i0 + j] * a.columns];
#pragma unroll
      for (int j = 0; j < BATCH; ++j)
        if (i0 + j < count && s_path[i0 + j] != i0 + j) p[(int64_t)(i0 + j) * a.columns] = v[j];
    }
  }
}

template <int LAYERS>
void launch(dim3 grid, cudaStream_t s, const Args& a, void* const* keys, void* const* values) {
  Caches<LAYERS> c;
  for (int l = 0; l < a.caches / 2; ++l) {
    c.at[2 * l] = static_cast<uint8_t*>(keys[l]);
    c.at[2 * l + 1] = static_cast<uint8_t*>(values[l]);
  }
  tree_accept_kernel<LAYERS><<<grid, THREADS, 0, s>>>(a, c);
}

}  // namespace

extern "C" int lpc_tree_accept(const int64_t* drafted, const int32_t* parents,
                               int64_t parents_stride, const int64_t* sampled,
                               const int32_t* seq_lens, void* const* key_caches,
                               void* const* value_caches, int layers, const int64_t* seq_base,
                               const int32_t* seq_cap, int32_t* accepted, int64_t* tokens,
                               int32_t* path, int64_t batch, int nodes, int kv_heads, int head_dim,
                               int64_t max_batch, int64_t max_seq_len, int64_t total_rows,
                               int elem_bytes, void* stream) {
  using namespace lpc;
  if (batch < 0 || nodes < 1 || layers < 0 || (parents_stride != 0 && parents_stride < nodes)) {
    set_error("tree_accept: invalid sizes (batch=%lld nodes=%d layers=%d)", (long long)batch, nodes,
              layers);
    return LPC_ERR_INVALID;
  }
  if (nodes > MAX_NODES || batch > 65535) {
    set_error("tree_accept: at most %d nodes and 65535 sequences", MAX_NODES);
    return LPC_ERR_UNSUPPORTED;
  }
  if (layers > 0) {
    if (kv_heads <= 0 || head_dim <= 0 || (elem_bytes != 2 && elem_bytes != 4) ||
        (!seq_base && (max_seq_len <= 0 || batch > max_batch)) || (seq_base && total_rows <= 0) ||
        (seq_base && !seq_cap)) {
      set_error("tree_accept: invalid cache sizes");
      return LPC_ERR_INVALID;
    }
    if (head_dim * elem_bytes % 16) {
      set_error("tree_accept: rows must be multiples of 16 bytes");
      return LPC_ERR_UNSUPPORTED;
    }
    if (!key_caches || !value_caches || !seq_lens) {
      set_error("tree_accept: null pointer");
      return LPC_ERR_INVALID;
    }
    for (int l = 0; l < layers; ++l)
      if (!key_caches[l] || !value_caches[l] || !aligned16(key_caches[l]) ||
          !aligned16(value_caches[l])) {
        set_error("tree_accept: caches must be 16-byte aligned");
        return LPC_ERR_INVALID;
      }
  }
  if (batch == 0) return LPC_OK;
  if (!drafted || !parents || !sampled || !accepted || !tokens || !path) {
    set_error("tree_accept: null pointer");
    return LPC_ERR_INVALID;
  }
  Args a;
  a.drafted = drafted;
  a.sampled = sampled;
  a.parents = parents;
  a.parents_stride = parents_stride;
  a.seq_lens = seq_lens;
  a.seq_base = seq_base;
  a.seq_cap = seq_cap;
  a.accepted = accepted;
  a.tokens = tokens;
  a.path = path;
  a.max_seq_len = max_seq_len;
  a.total_rows = total_rows;
  a.nodes = nodes;
  a.kv_heads = kv_heads;
  a.columns = layers ? head_dim * elem_bytes / 16 : 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int done = 0;
  do {
    const int now = layers - done < MAX_LAYERS ? layers - done : MAX_LAYERS;
    a.caches = 2 * now;
    a.report = done == 0;
    // a column a thread, until the grid is 16 CTAs an SM deep
    const int64_t work = (int64_t)a.caches * kv_heads * a.columns;
    const int64_t want = now ? (work + THREADS - 1) / THREADS : 1;
    const int64_t most = ((int64_t)current_device_sms() * 16 + batch - 1) / batch;
    const dim3 grid((unsigned)(want < most ? want : most), (unsigned)batch);
    // the addresses travel as kernel parameters: no more of them than there are
    if (now <= 4) launch<4>(grid, s, a, key_caches + done, value_caches + done);
    else if (now <= 32) launch<32>(grid, s, a, key_caches + done, value_caches + done);
    else launch<MAX_LAYERS>(grid, s, a, key_caches + done, value_caches + done);
    if (int rc = check_launch("tree_accept")) return rc;
    done += now;
  } while (done < layers);
  return LPC_OK;
}
