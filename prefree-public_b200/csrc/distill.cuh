// Distillation from a teacher's kept logits: per-row loss of dense student
// logits Z (m x n) against a CSR matrix of teacher logits, and its gradient.
//
// With temperature tau, row r's stored columns S, teacher logits t and student
// logits z:
//   p_j = exp(t_j / tau - Lt),  Lt = log sum_{j in S} exp(t_j / tau)
//   q_i = exp(z_i / tau - Lz),  Lz = log sum_{all i}  exp(z_i / tau)
//   loss = w * sum_{j in S} p_j (log p_j - log q_j)
//        = w * ((sum_j p_j (t_j - z_j) - max t + max z) / tau
//               - log sum_j exp((t_j - max t) / tau)
//               + log sum_i exp((z_i - max z) / tau))
//   dZ_i = (w / tau) * (q_i - sum_{j in S, col_j = i} p_j)
// An entry with p_j = 0 adds nothing whatever z_j is. A row without teacher
// mass (no entry, or all of them -inf) and a row of weight 0 have loss 0 and
// gradient 0; the student's row of the latter is not read.
#pragma once

#include "pf_common.cuh"

namespace pf {

template <typename VT, typename IT>
struct DistillParams {
  int64_t m, n, nnz;
  const IT *row_ptr;
  const int32_t *col;
  const VT *val;       // teacher logits
  const VT *Z;         // student logits; dZ may be the same array
  int64_t ldz;
  const float *weight; // per row, or null (1)
  float *loss;         // per row, or null
  VT *dZ;              // m x n, or null
  int64_t lddz;
  float inv_tau;
  unsigned *err;
};

template <typename VT>
__device__ __forceinline__ float to_f32(VT v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <typename VT>
__device__ __forceinline__ VT from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// A running softmax state: the largest value so far and the sum of
// exp(scale * (value - m)); NaN values make both NaN.
struct SoftmaxState {
  float m, s;
};
__device__ __forceinline__ float nan_max(float a, float b) {
  return (a != a || a > b) ? a : b;  // NaN if either is
}
// exp(scale * (v - m)) for v <= m, 0 when v is -inf (m may be -inf too)
__device__ __forceinline__ float shifted_exp(float v, float m, float scale) {
  return v == -INFINITY ? 0.0f : __expf((v - m) * scale);
}
__device__ __forceinline__ SoftmaxState merge(SoftmaxState a, SoftmaxState b, float scale) {
  SoftmaxState o;
  o.m = nan_max(a.m, b.m);
  o.s = a.s * shifted_exp(a.m, o.m, scale) + b.s * shifted_exp(b.m, o.m, scale);
  return o;
}

// One CTA per row: one pass for the row's softmax statistics, the teacher's
// statistics and sum_j p_j (t_j - z_j), a second one for the gradient.
template <typename VT, typename IT, int NT>
__global__ void __launch_bounds__(NT) distill_kernel(const DistillParams<VT, IT> P) {
  constexpr int NW = NT / 32;
  __shared__ SoftmaxState sh_z[NW], sh_t[NW];
  __shared__ double sh_d[NW];
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const float sc = P.inv_tau;
  const int64_t base = (int64_t)P.row_ptr[0];
  for (int64_t r = blockIdx.x; r < P.m; r += gridDim.x) {
    const float w = P.weight ? P.weight[r] : 1.0f;
    int64_t s = (int64_t)P.row_ptr[r], e = (int64_t)P.row_ptr[r + 1];
    if (s < base || e < s || e > base + P.nnz) {
      if (tid == 0) atomicOr(P.err, PF_DEVERR_ROWPTR);
      s = e = 0;
    }
    const VT *z = P.Z + r * P.ldz;
    VT *dz = P.dZ ? P.dZ + r * P.lddz : nullptr;
    SoftmaxState t{-INFINITY, 0.0f}, q{-INFINITY, 0.0f};
    if (w != 0.0f) {
      for (int64_t i = s + tid; i < e; i += NT)
        if ((uint32_t)P.col[i] < (uint64_t)P.n)
          t = merge(t, SoftmaxState{to_f32(P.val[i]), 1.0f}, sc);
        else atomicOr(P.err, PF_DEVERR_BOUNDS);
      for (int64_t i = tid; i < P.n; i += NT) q = merge(q, SoftmaxState{to_f32(z[i]), 1.0f}, sc);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
      t = merge(t, SoftmaxState{__shfl_xor_sync(~0u, t.m, d), __shfl_xor_sync(~0u, t.s, d)}, sc);
      q = merge(q, SoftmaxState{__shfl_xor_sync(~0u, q.m, d), __shfl_xor_sync(~0u, q.s, d)}, sc);
    }
    if (lane == 0) sh_t[wid] = t, sh_z[wid] = q;
    __syncthreads();
    t = sh_t[0], q = sh_z[0];
    for (int k = 1; k < NW; ++k) t = merge(t, sh_t[k], sc), q = merge(q, sh_z[k], sc);
    const bool mass = w != 0.0f && t.m != -INFINITY;
    double d = 0.0;
    if (mass)
      for (int64_t i = s + tid; i < e; i += NT) {
        const uint32_t c = (uint32_t)P.col[i];
        if (c >= (uint64_t)P.n) continue;
        const float tv = to_f32(P.val[i]);
        const float p = shifted_exp(tv, t.m, sc);
        if (p != 0.0f) d += (double)p * ((double)tv - (double)to_f32(z[c]));
      }
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) d += __shfl_xor_sync(~0u, d, k);
    if (lane == 0) sh_d[wid] = d;
    __syncthreads();
    if (tid == 0 && P.loss) {
      double total = 0.0;
      for (int k = 0; k < NW; ++k) total += sh_d[k];
      double v = 0.0;
      if (mass && q.m == -INFINITY) v = (double)w * INFINITY;
      else if (mass)
        v = (double)w * ((total / (double)t.s - (double)t.m + (double)q.m) * (double)sc +
                         log((double)q.s / (double)t.s));
      P.loss[r] = (float)v;
    }
    if (dz) {
      const float g = mass ? w * sc : 0.0f;
      const float gz = q.m == -INFINITY ? 0.0f : g / q.s, gt = mass ? g / t.s : 0.0f;
      for (int64_t c0 = (int64_t)wid * 32; c0 < P.n; c0 += NT) {
        const int64_t c = c0 + lane;
        float v = 0.0f;
        if (mass) {
          if (c < P.n) v = gz * shifted_exp(to_f32(z[c]), q.m, sc);
          for (int64_t i0 = s; i0 < e; i0 += 32) {
            const int64_t i = i0 + lane;
            const int32_t ci = i < e ? P.col[i] : -1;
            unsigned hits = __ballot_sync(~0u, ci >= c0 && ci < c0 + 32 && ci < P.n);
            while (hits) {
              const int k = __ffs(hits) - 1;
              hits &= hits - 1;
              const int32_t ck = __shfl_sync(~0u, ci, k);
              if (c == ck) v -= gt * shifted_exp(to_f32(P.val[i0 + k]), t.m, sc);
            }
          }
        }
        if (c < P.n) dz[c] = from_f32<VT>(v);
      }
    }
    __syncthreads();
  }
}

}  // namespace pf
