// Packed 4-bit weights: layout shared by their kernels (int4_linear.cu has the
// description of the codes' order).
//   codes    [tile row][k / 64][512 bytes]        tile rows of 16 weight rows
//   numbers  [tile row][k / group][8][4] of T     (s, m) of rows r and r + 8
//   scaled   [tile row][k / group][16][2] fp16    (s 2^e, m 2^e) of each row
//   factors  [tile row][16] fp32                  2^-e of each row
// e is a power per row that brings the largest 15 |s| + |m| to 2^14..2^15: fp16 holds
// its groups' numbers exactly unless they are below 2^-28 of that.
#pragma once

#include "lpc_common.cuh"

namespace lpc {

// Tile rows of 16: of the weight (layout 0), or gate tile i, up tile i, ...
// (layout 1, gate rows first in the source).  A multiple of 8 of them, so that
// no kernel's item reaches past the last.
__host__ __device__ inline int64_t int4_tile_rows(int64_t n_out, int layout) {
  const int64_t t = (n_out + 15) / 16 * (layout == 1 ? 2 : 1);
  return (t + 7) / 8 * 8;
}

struct Int4Parts {
  uint8_t *codes, *numbers, *scaled;
  float* factors;
  int64_t bytes;
};
inline Int4Parts int4_parts(void* base, int64_t n_out, int k, int group, int layout) {
  const int64_t tr = int4_tile_rows(n_out, layout), ng = k / group;
  Int4Parts p;
  p.codes = static_cast<uint8_t*>(base);
  p.numbers = p.codes + tr * 16 * (int64_t)(k / 2);
  p.scaled = p.numbers + tr * ng * 64;
  p.factors = reinterpret_cast<float*>(p.scaled + tr * ng * 64);
  p.bytes = tr * 16 * (int64_t)(k / 2) + tr * ng * 128 + tr * 64;
  return p;
}

// Token counts and weights that the kernels of int4_linear.cu are not for.
int int4_many(const lpc_w4* w, const void* x, void* out, const void* resid, int64_t tokens,
              int epilogue, void* workspace, cudaStream_t s);

}  // namespace lpc
