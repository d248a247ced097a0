// C-ABI of the grouped matrix products.
#include <algorithm>

#include "gmm_simt.cuh"
#include "pf_handle.cuh"

namespace pf {

template <typename VT, typename IT>
static pf_status launch_gmm(pf_handle h, int64_t groups, int64_t rows, int64_t n, int64_t k,
                            const IT *ptr, const VT *X, int64_t ldx, const VT *W, int64_t ldw,
                            int64_t stride_w, int trans_w, double alpha, double beta, VT *Y,
                            int64_t ldy, cudaStream_t st) {
  PF_CHECK_ARG(h != nullptr, "null handle");
  PF_CHECK_ARG(groups >= 0 && rows >= 0 && n >= 0 && k >= 0,
               "negative size (groups=%lld rows=%lld n=%lld k=%lld)", (long long)groups,
               (long long)rows, (long long)n, (long long)k);
  if (groups == 0 || rows == 0 || n == 0) return PF_OK;
  PF_CHECK_ARG(groups < INT32_MAX && n <= INT32_MAX && k <= INT32_MAX && rows <= INT32_MAX,
               "groups, rows, n and k must fit 31 bits");
  PF_CHECK_ARG(ptr && Y, "null group_ptr or Y");
  PF_CHECK_ARG(k == 0 || (X && W), "null X/W with k > 0");
  const int64_t wcols = trans_w ? k : n, wrows = trans_w ? n : k;
  PF_CHECK_ARG(ldx >= k && ldw >= wcols && ldy >= n, "leading dimension below the row's length");
  PF_CHECK_ARG(groups == 1 || wrows == 0 || stride_w >= (wrows - 1) * ldw + wcols,
               "stride_w below one matrix");
  PF_CHECK_ARG(((uintptr_t)ptr % sizeof(IT)) == 0 && ((uintptr_t)X % sizeof(VT)) == 0 &&
                   ((uintptr_t)W % sizeof(VT)) == 0 && ((uintptr_t)Y % sizeof(VT)) == 0,
               "arrays must be aligned to their element size");
  int cur = 0;
  PF_CUDA_TRY(cudaGetDevice(&cur));
  PF_CHECK_ARG(cur == h->device, "handle bound to device %d, current device is %d", h->device, cur);
  GmmSimtParams<VT, VT, IT> p{groups, rows, n,   k,   ptr, X,
                              ldx,    W,    ldw, stride_w, Y,   ldy,
                              0,      (float)alpha, (float)beta, h->err};
  // no more tiles than whole ones and one partial one to a group
  const int64_t tiles = (rows / 64 + std::min(groups, rows)) * ceil_div(n, 64);
  const unsigned grid = (unsigned)std::min<int64_t>(tiles, (int64_t)h->num_sms * 8);
  if (trans_w) gmm_simt_kernel<VT, VT, IT, 0><<<grid, 256, 0, st>>>(p);
  else gmm_simt_kernel<VT, VT, IT, 1><<<grid, 256, 0, st>>>(p);
  count_launches(1);
  PF_CUDA_TRY(cudaGetLastError());
  return PF_OK;
}

template <typename VT, typename OT, typename IT>
static pf_status launch_wgrad(pf_handle h, int64_t groups, int64_t rows, int64_t n, int64_t k,
                              const IT *ptr, const VT *dY, int64_t lddy, const VT *X, int64_t ldx,
                              double alpha, double beta, OT *dW, int64_t lddw, int64_t stride_dw,
                              cudaStream_t st) {
  PF_CHECK_ARG(h != nullptr, "null handle");
  PF_CHECK_ARG(groups >= 0 && rows >= 0 && n >= 0 && k >= 0,
               "negative size (groups=%lld rows=%lld n=%lld k=%lld)", (long long)groups,
               (long long)rows, (long long)n, (long long)k);
  if (groups == 0 || n == 0 || k == 0) return PF_OK;
  PF_CHECK_ARG(groups < INT32_MAX && n <= INT32_MAX && k <= INT32_MAX && rows <= INT32_MAX,
               "groups, rows, n and k must fit 31 bits");
  PF_CHECK_ARG(ptr && dW, "null group_ptr or dW");
  PF_CHECK_ARG(rows == 0 || (dY && X), "null dY/X with rows > 0");
  PF_CHECK_ARG((rows == 0 || (lddy >= n && ldx >= k)) && lddw >= k,
               "leading dimension below the row's length");
  PF_CHECK_ARG(groups == 1 || stride_dw >= (n - 1) * lddw + k, "stride_dw below one matrix");
  PF_CHECK_ARG(((uintptr_t)ptr % sizeof(IT)) == 0 && ((uintptr_t)X % sizeof(VT)) == 0 &&
                   ((uintptr_t)dY % sizeof(VT)) == 0 && ((uintptr_t)dW % sizeof(OT)) == 0,
               "arrays must be aligned to their element size");
  int cur = 0;
  PF_CUDA_TRY(cudaGetDevice(&cur));
  PF_CHECK_ARG(cur == h->device, "handle bound to device %d, current device is %d", h->device, cur);
  GmmSimtParams<VT, OT, IT> p{groups, rows, n,   k, ptr, dY,
                              lddy,   X,    ldx, 0, dW,  lddw,
                              stride_dw, (float)alpha, (float)beta, h->err};
  const int64_t per_group = ceil_div(n, 64) * ceil_div(k, 64), cap = (int64_t)h->num_sms * 8;
  const unsigned grid = (unsigned)(per_group >= cap ? cap : std::min(groups * per_group, cap));
  gmm_simt_kernel<VT, OT, IT, 2><<<grid, 256, 0, st>>>(p);
  count_launches(1);
  PF_CUDA_TRY(cudaGetLastError());
  return PF_OK;
}

}  // namespace pf

using namespace pf;

extern "C" {

// 16-bit values cross the C ABI as their raw bit patterns (uint16_t)
#define PF_DEFINE_GMM(SUFFIX, VT, IT)                                                          \
  pf_status pf_gmm_##SUFFIX(pf_handle h, int64_t groups, int64_t rows, int64_t n, int64_t k,   \
                            const IT *group_ptr, const uint16_t *X, int64_t ldx,               \
                            const uint16_t *W, int64_t ldw, int64_t stride_w, int trans_w,     \
                            double alpha, double beta, uint16_t *Y, int64_t ldy,               \
                            void *stream) {                                                    \
    return launch_gmm<VT, IT>(h, groups, rows, n, k, group_ptr,                                \
                              reinterpret_cast<const VT *>(X), ldx,                            \
                              reinterpret_cast<const VT *>(W), ldw, stride_w, trans_w, alpha,  \
                              beta, reinterpret_cast<VT *>(Y), ldy, (cudaStream_t)stream);     \
  }                                                                                            \
  pf_status pf_gmm_wgrad_##SUFFIX(pf_handle h, int64_t groups, int64_t rows, int64_t n,        \
                                  int64_t k, const IT *group_ptr, const uint16_t *dY,          \
                                  int64_t lddy, const uint16_t *X, int64_t ldx, double alpha,  \
                                  double beta, void *dW, int dw_bytes, int64_t lddw,           \
                                  int64_t stride_dw, void *stream) {                           \
    PF_CHECK_ARG(dw_bytes == 2 || dw_bytes == 4, "dw_bytes %d: 2 or 4", dw_bytes);             \
    const VT *dy = reinterpret_cast<const VT *>(dY), *x = reinterpret_cast<const VT *>(X);     \
    if (dw_bytes == 4)                                                                         \
      return launch_wgrad<VT, float, IT>(h, groups, rows, n, k, group_ptr, dy, lddy, x, ldx,   \
                                         alpha, beta, (float *)dW, lddw, stride_dw,            \
                                         (cudaStream_t)stream);                                \
    return launch_wgrad<VT, VT, IT>(h, groups, rows, n, k, group_ptr, dy, lddy, x, ldx, alpha, \
                                    beta, (VT *)dW, lddw, stride_dw, (cudaStream_t)stream);    \
  }

PF_DEFINE_GMM(f16_i32, __half, int32_t)
PF_DEFINE_GMM(f16_i64, __half, int64_t)
PF_DEFINE_GMM(bf16_i32, __nv_bfloat16, int32_t)
PF_DEFINE_GMM(bf16_i64, __nv_bfloat16, int64_t)

}  // extern "C"
