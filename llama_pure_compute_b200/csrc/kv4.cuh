// The 4-bit KV cache: row format and addressing shared by its kernels.
//
// A row holds one position of one KV head, D dims in two groups (the lower and
// the upper half of the dims), each with its own scale s and minimum m:
//   codes   D/2 bytes; byte j = code of dim j | code of dim j + D/2 << 4.  The
//           two partners of a rotation pair share a byte, so the thread that
//           rotates a pair also writes it; and one mask applied to a 32-bit
//           word picks codes of one group only, which is what lets the
//           attention kernel feed codes to the tensor core and apply s and m
//           to whole accumulators.
//   scales  4 numbers of the cache's type: s0, m0, s1, m1.
// A code c of group g stands for s_g * c + m_g.
#pragma once

#include "lpc_common.cuh"

namespace lpc {

// Where a sequence's rows live.
//   dense  (base == nullptr): [max_batch, Hkv, max_seq, .], row (b, h, p) =
//          (b * Hkv + h) * max_seq + p, capacity max_seq;
//   ragged: [Hkv, total_rows, .], sequence b owns rows [base[b], base[b] + cap[b])
//          of every head.
struct Kv4Rows {
  const int64_t* base;
  const int32_t* cap;
  int64_t max_seq;
  int64_t total_rows;
  int kv_heads;

  // Row of (b, head 0, position 0), the distance between heads and the
  // capacity; false when the sequence's rows are not inside the buffer.
  __device__ __forceinline__ bool locate(int64_t b, int64_t* row0, int64_t* head_rows,
                                         int64_t* capacity) const {
    if (base == nullptr) {
      *row0 = b * kv_heads * max_seq;
      *head_rows = max_seq;
      *capacity = max_seq;
      return true;
    }
    const int64_t sb = ld_dep(base + b);
    const int64_t c = ld_dep(cap + b);
    *row0 = sb;
    *head_rows = total_rows;
    *capacity = c;
    return sb >= 0 && c >= 0 && c <= max_seq && sb <= total_rows && c <= total_rows - sb;
  }
};

// Host check of the handle itself; sets the error text and returns a status.
int kv4_check(const lpc_kv4* kv, const char* what);

inline Kv4Rows kv4_rows(const lpc_kv4* kv) {
  return Kv4Rows{kv->seq_base, kv->seq_cap, kv->max_seq_len, kv->total_rows, kv->kv_heads};
}

}  // namespace lpc
