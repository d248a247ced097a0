// 16-bit SpMM over wide dense rows, Y = alpha * A * X + beta * Y, and the
// gradient of its values, dval_j = alpha * <dY[row(j), :], X[col_j, :]> +
// beta * dval_j (a dense-dense product sampled at A's non-zeros).
//
// The dense rows are long (hundreds to thousands of 16-bit values) and the
// CSR rows short: the bytes of X and Y bound both, so threads run along the
// dense row. Products of 16-bit values are exact in fp32; sums are in fp32 in
// the row's order (the same bits on every run) and rounded once.
#pragma once

#include "distill.cuh"
#include "pf_common.cuh"

namespace pf {

template <typename VT, typename IT>
struct WideParams {
  int64_t m, n, nnz;
  const IT *row_ptr;
  const int32_t *col;
  const VT *val;
  const VT *X;
  int64_t ldx;
  VT *Y;         // SpMM: written; the sampled product reads dY here
  int64_t ldy;
  VT *dval;
  int64_t k;     // columns of X and Y
  float alpha, beta;
  unsigned *err;
};

template <typename VT, typename IT, int NT>
__global__ void __launch_bounds__(NT) spmm_wide_kernel(const WideParams<VT, IT> P) {
  const int64_t base = (int64_t)P.row_ptr[0];
  for (int64_t r = blockIdx.x; r < P.m; r += gridDim.x) {
    int64_t s = (int64_t)P.row_ptr[r], e = (int64_t)P.row_ptr[r + 1];
    if (s < base || e < s || e > base + P.nnz) {
      if (threadIdx.x == 0) atomicOr(P.err, PF_DEVERR_ROWPTR);
      s = e = 0;
    }
    for (int64_t c = threadIdx.x; c < P.k; c += NT) {
      float acc = 0.0f;
      for (int64_t i = s; i < e; ++i) {
        const uint32_t j = (uint32_t)P.col[i];
        if (j >= (uint64_t)P.n) {
          atomicOr(P.err, PF_DEVERR_BOUNDS);
          continue;
        }
        acc += to_f32(P.val[i]) * to_f32(P.X[j * P.ldx + c]);
      }
      VT *y = P.Y + r * P.ldy + c;
      float out = P.alpha * acc;
      if (P.beta != 0.0f) out += P.beta * to_f32(*y);
      *y = from_f32<VT>(out);
    }
  }
}

// One warp per row, one non-zero at a time.
template <typename VT, typename IT, int NT>
__global__ void __launch_bounds__(NT) sddmm_kernel(const WideParams<VT, IT> P) {
  const int lane = threadIdx.x & 31;
  const int64_t nwarps = ((int64_t)gridDim.x * NT) >> 5;
  const int64_t base = (int64_t)P.row_ptr[0];
  for (int64_t r = ((int64_t)blockIdx.x * NT + threadIdx.x) >> 5; r < P.m; r += nwarps) {
    int64_t s = (int64_t)P.row_ptr[r], e = (int64_t)P.row_ptr[r + 1];
    if (s < base || e < s || e > base + P.nnz) {
      if (lane == 0) atomicOr(P.err, PF_DEVERR_ROWPTR);
      s = e = 0;
    }
    for (int64_t i = s; i < e; ++i) {
      const uint32_t j = (uint32_t)P.col[i];
      if (j >= (uint64_t)P.n) {
        if (lane == 0) atomicOr(P.err, PF_DEVERR_BOUNDS);
        continue;
      }
      float acc = 0.0f;
      for (int64_t c = lane; c < P.k; c += 32)
        acc += to_f32(P.Y[r * P.ldy + c]) * to_f32(P.X[j * P.ldx + c]);
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) acc += __shfl_xor_sync(~0u, acc, d);
      if (lane == 0) {
        float out = P.alpha * acc;
        if (P.beta != 0.0f) out += P.beta * to_f32(P.dval[i]);
        P.dval[i] = from_f32<VT>(out);
      }
    }
  }
}

}  // namespace pf
