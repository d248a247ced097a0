// The grouped products on the CUDA cores: any alignment and any leading
// dimension. 64 x 64 output tiles, 16 of the reduction at a time through
// shared memory, 4 x 4 outputs a thread, sums in fp32 in the reduction's order.
#pragma once

#include "gmm_common.cuh"

namespace pf {

template <typename VT, typename OT, typename IT>
struct GmmSimtParams {
  int64_t groups, rows, n, k;
  const IT *ptr;
  const VT *A;          // product: X; gradient: dY
  int64_t lda;
  const VT *B;          // product: W; gradient: X
  int64_t ldb, stride_b;
  OT *C;                // product: Y; gradient: dW
  int64_t ldc, stride_c;
  float alpha, beta;
  unsigned *err;
};

// MODE 0: Y = X W_g^T (W_g n x k), 1: Y = X W_g (W_g k x n), 2: dW_g = dY^T X
template <typename VT, typename OT, typename IT, int MODE>
__global__ void __launch_bounds__(256) gmm_simt_kernel(const GmmSimtParams<VT, OT, IT> P) {
  constexpr int BM = 64, BN = 64, BK = 16;
  __shared__ float sa[BK][BM + 4], sb[BK][BN + 4];
  const int tid = threadIdx.x, ti = tid / 16, tj = tid % 16;
  // the output's columns, and (gradient) its rows
  const int64_t out_cols = MODE == 2 ? P.k : P.n;
  const int64_t ct = (out_cols + BN - 1) / BN;
  const int64_t per_group = (P.n + BM - 1) / BM * ct;  // gradient: tiles of one dW_g
  GroupWalk<IT> walk{P.ptr, P.groups, P.rows, P.err};
  for (int64_t t = blockIdx.x;; t += gridDim.x) {
    int64_t g, first, count, i0, j0, i_end;
    if (MODE == 2) {
      g = t / per_group;
      if (g >= P.groups) break;
      count = group_rows(P.ptr, g, P.rows, &first, P.err);
      i0 = t % per_group / ct * BM;
      j0 = t % per_group % ct * BN;
      i_end = P.n;
    } else {
      if (!walk.seek(t, BM, ct)) break;
      g = walk.g;
      first = walk.first;
      count = walk.count;
      i0 = (t - walk.before) / ct * BM;
      j0 = (t - walk.before) % ct * BN;
      i_end = count;
    }
    const int64_t depth = MODE == 2 ? count : P.k;
    float acc[4][4] = {};
    for (int64_t p0 = 0; p0 < depth; p0 += BK) {
      for (int x = tid; x < BM * BK; x += 256) {
        float a = 0.0f, b = 0.0f;
        if (MODE == 2) {
          const int p = x / BM, i = x % BM;
          if (p0 + p < depth && i0 + i < i_end)
            a = to_f32(P.A[(first + p0 + p) * P.lda + i0 + i]);
          if (p0 + p < depth && j0 + i < out_cols)
            b = to_f32(P.B[(first + p0 + p) * P.ldb + j0 + i]);
          sa[p][i] = a;
          sb[p][i] = b;
        } else {
          const int p = x % BK, i = x / BK;
          if (p0 + p < depth && i0 + i < i_end)
            a = to_f32(P.A[(first + i0 + i) * P.lda + p0 + p]);
          sa[p][i] = a;
          if (MODE == 0) {
            if (p0 + p < depth && j0 + i < out_cols)
              b = to_f32(P.B[g * P.stride_b + (j0 + i) * P.ldb + p0 + p]);
            sb[p][i] = b;
          } else {
            const int pp = x / BN, j = x % BN;
            if (p0 + pp < depth && j0 + j < out_cols)
              b = to_f32(P.B[g * P.stride_b + (p0 + pp) * P.ldb + j0 + j]);
            sb[pp][j] = b;
          }
        }
      }
      __syncthreads();
#pragma unroll
      for (int p = 0; p < BK; ++p) {
        float a[4], b[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) a[x] = sa[p][ti * 4 + x], b[x] = sb[p][tj + 16 * x];
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
          for (int y = 0; y < 4; ++y) acc[x][y] += a[x] * b[y];
      }
      __syncthreads();
    }
    OT *c = P.C + (MODE == 2 ? g * P.stride_c : first * P.ldc);
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const int64_t i = i0 + ti * 4 + x, j = j0 + tj + 16 * y;
        if (i < i_end && j < out_cols) {
          float out = P.alpha * acc[x][y];
          if (P.beta != 0.0f) out += P.beta * to_f32(c[i * P.ldc + j]);
          c[i * P.ldc + j] = from_f32<OT>(out);
        }
      }
  }
}

}  // namespace pf
