// Where the paged fp16 KV cache holds a value.  A page has, head by head, page_size * D
// keys' values and as many values' values (P = page_size, D = head_dim):
//   [page][kv_head][2][P D]
//   K  [P / 16][D / 32][64 lanes][8]: lane j + 16 g of record (t, c) holds token 16 t + j,
//      dims 32 c + 8 g .. + 7;
//   V  [P / 32][D / 16][64 lanes][8]: lane j + 16 g of record (t, c) holds dim (D / 16) j + c
//      of tokens 32 t + 4 g .. + 3 and 32 t + 16 + 4 g .. + 3.
// Both are operands of the matrix instruction that multiplies them, one kilobyte per
// instruction: the attention kernel loads 16 bytes per lane, one after another, and moves
// nothing between lanes.  V's dims are dealt so that 8 neighbouring ones of 8 tokens, what a
// lane turns around in registers, fill records of different c at one lane's place.
#pragma once
#include "common.hpp"
#include "kernels.hpp"

namespace tia {

__host__ __device__ __forceinline__ int64_t paged_head_size(const KvPaged& c) { return int64_t(2) * c.page_size * c.head_dim; }

// Of token t of a page.
__device__ __forceinline__ int paged_k_at(int t, int dim, int D) {
  return (t >> 4) * 16 * D + (dim >> 5) * 512 + ((t & 15) + 16 * ((dim >> 3) & 3)) * 8 + (dim & 7);
}
__device__ __forceinline__ int paged_v_at(int t, int dim, int D) {
  const int r = t & 31, per = D / 16;
  return (t >> 5) * 32 * D + (dim % per) * 512 + (dim / per + 16 * ((r >> 2) & 3)) * 8 + 4 * (r >> 4) + (r & 3);
}

}  // namespace tia
