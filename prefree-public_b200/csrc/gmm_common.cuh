// Grouped matrix products: group g owns the rows [ptr[g], ptr[g+1]) of the
// dense arrays (a row_ptr whose "row" is a group), and has a matrix of its own.
//   product:  Y[r, :] = alpha * X[r, :] * op(W_g) + beta * Y[r, :]
//   gradient: dW_g = alpha * sum_{r in g} dY[r, :]^T X[r, :] + beta * dW_g
// This file: the parameters, and the search of a work item's group, which runs
// on the device (the group sizes are never read back to the host).
#pragma once

#include "pf_values.cuh"

namespace pf {

// The rows of group g, empty (and flagged) where the pointers are not
// non-decreasing or leave [0, rows].
template <typename IT>
__device__ __forceinline__ int64_t group_rows(const IT *ptr, int64_t g, int64_t rows,
                                              int64_t *first, unsigned *err) {
  const int64_t s = (int64_t)ptr[g], e = (int64_t)ptr[g + 1];
  *first = s;
  if (s < 0 || e < s || e > rows) {
    atomicOr(err, PF_DEVERR_ROWPTR);
    return 0;
  }
  return e - s;
}

// Walks the row tiles of all groups in order: item t of the sequence "group 0's
// row tiles times `per`, group 1's, ...". All 32 lanes of a warp call seek()
// with the same, non-decreasing t: each step looks at 32 groups at once.
template <typename IT>
struct GroupWalk {
  const IT *ptr;
  int64_t groups, rows;
  unsigned *err;
  int64_t g = 0;       // first group not passed yet
  int64_t before = 0;  // items of the groups before it
  int64_t first = 0;   // group g's first row and number of rows
  int64_t count = 0;
  int64_t items = 0;   // its items, where they are known

  // finds item t; false when there are fewer. Afterwards group g holds it, at
  // place t - before.
  __device__ __forceinline__ bool seek(int64_t t, int tile_rows, int64_t per) {
    const int lane = threadIdx.x & 31;
    if (t < before + items) return true;
    while (g < groups) {
      int64_t f = 0, c = 0;
      if (g + lane < groups) c = group_rows(ptr, g + lane, rows, &f, err);
      const int64_t own = (c + tile_rows - 1) / tile_rows * per;
      int64_t sum = own;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int64_t v = __shfl_up_sync(~0u, sum, d);
        if (lane >= d) sum += v;
      }
      const unsigned past = __ballot_sync(~0u, before + sum > t);
      if (past) {
        const int k = __ffs(past) - 1;
        const int64_t prev = __shfl_sync(~0u, sum, k > 0 ? k - 1 : 0);
        if (k > 0) before += prev;
        g += k;
        first = __shfl_sync(~0u, f, k);
        count = __shfl_sync(~0u, c, k);
        items = __shfl_sync(~0u, own, k);
        return true;
      }
      before += __shfl_sync(~0u, sum, 31);
      items = 0;
      g += 32;
    }
    return false;
  }
};

}  // namespace pf
