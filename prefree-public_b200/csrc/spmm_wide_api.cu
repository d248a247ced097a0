// C-ABI of the 16-bit SpMM and of the gradient of its values (spmm_wide.cuh).
#include <algorithm>

#include "pf_handle.cuh"
#include "spmm_wide.cuh"

namespace pf {

// What the two calls check alike: sizes, pointers, leading dimensions,
// alignment, device.
template <typename VT, typename IT>
static pf_status check_wide(pf_handle h, int64_t m, int64_t n, int64_t nnz, const IT *row_ptr,
                            const int32_t *col, const VT *val, int k, const VT *X, int64_t ldx,
                            const VT *Y, int64_t ldy) {
  PF_CHECK_ARG(sizeof(IT) == 8 || nnz <= INT32_MAX, "int32 row_ptr cannot index nnz=%lld",
               (long long)nnz);
  PF_CHECK_ARG(n <= (int64_t)INT32_MAX + 1, "n must fit int32 column indices");
  PF_CHECK_ARG(k <= INT32_MAX - 64, "k must be at most 2^31 - 65");
  PF_CHECK_ARG(nnz == 0 || n > 0, "nnz > 0 needs n > 0 (column indices lie in [0, n))");
  PF_CHECK_ARG(row_ptr && (Y || k == 0), "null row_ptr or Y");
  PF_CHECK_ARG(nnz == 0 || (col && val && (X || k == 0)), "null col/val/X with nnz > 0");
  PF_CHECK_ARG(ldy >= k && (nnz == 0 || ldx >= k), "leading dimension below k");
  PF_CHECK_ARG(((uintptr_t)row_ptr % sizeof(IT)) == 0 && ((uintptr_t)Y % sizeof(VT)) == 0 &&
                   (nnz == 0 || (((uintptr_t)col % 4) == 0 && ((uintptr_t)val % sizeof(VT)) == 0 &&
                                 ((uintptr_t)X % sizeof(VT)) == 0)),
               "arrays must be aligned to their element size");
  int cur = 0;
  PF_CUDA_TRY(cudaGetDevice(&cur));
  PF_CHECK_ARG(cur == h->device, "handle bound to device %d, current device is %d", h->device, cur);
  return PF_OK;
}

// whether every row starts on a 16-byte boundary
template <typename VT>
static bool rows16(const VT *p, int64_t ld) {
  return ((uintptr_t)p % 16) == 0 && ld % 8 == 0;
}

template <typename VT, typename IT>
static pf_status launch_spmm16(pf_handle h, int64_t m, int64_t n, int64_t nnz, const IT *row_ptr,
                               const int32_t *col, const VT *val, int k, double alpha, const VT *X,
                               int64_t ldx, double beta, VT *Y, int64_t ldy, cudaStream_t st) {
  PF_CHECK_ARG(h != nullptr, "null handle");
  PF_CHECK_ARG(m >= 0 && n >= 0 && nnz >= 0 && k >= 0, "negative size");
  if (m == 0 || k == 0) return PF_OK;
  pf_status s = check_wide<VT, IT>(h, m, n, nnz, row_ptr, col, val, k, X, ldx, Y, ldy);
  if (s != PF_OK) return s;
  WideParams<VT, IT> p{m, n, nnz, row_ptr, col, val, X, ldx, Y, ldy, nullptr, k,
                       (float)alpha, (float)beta, h->err};
  // rows of one or two non-zeros (a dispatch, or a gradient of the slots) take
  // several pieces of columns at a time instead of several non-zeros
  const bool aligned = rows16(X, ldx) && rows16(Y, ldy);
  const bool few = nnz <= 2 * m;
  const int64_t units = ceil_div(ceil_div((int64_t)k + (aligned ? 0 : 7), 8), few ? (aligned ? 4 : 3) : 1);
  // threads a row: one for every unit of its columns, up to a CTA, the power of
  // two below (the one above leaves up to half of them idle); the columns of few
  // rows are spread over more CTAs
  int tpr_log2 = 0;
  const int most_log2 = few ? 5 : 8;  // (what a row costs besides its pieces counts there)
  while (tpr_log2 < 8 && (2 << tpr_log2) <= units &&
         (tpr_log2 < most_log2 || ceil_div(m, 256 >> tpr_log2) < 4 * h->num_sms))
    ++tpr_log2;
  while (tpr_log2 > 5 && ceil_div(m, 256 >> tpr_log2) < h->num_sms) --tpr_log2;
  const int64_t ctas = ceil_div(m, 256 >> tpr_log2), most = (int64_t)h->num_sms * (aligned ? 4 : 3);
  dim3 grid((unsigned)std::min(ctas, most));
  if (ctas < h->num_sms) grid.y = (unsigned)std::min<int64_t>(64, ceil_div(units, 1 << tpr_log2));
  if (aligned && few) spmm_wide_kernel<VT, IT, 256, true, 1, 4><<<grid, 256, 0, st>>>(p, tpr_log2);
  else if (aligned) spmm_wide_kernel<VT, IT, 256, true, 4, 1><<<grid, 256, 0, st>>>(p, tpr_log2);
  else if (few) spmm_wide_kernel<VT, IT, 256, false, 1, 3><<<grid, 256, 0, st>>>(p, tpr_log2);
  else spmm_wide_kernel<VT, IT, 256, false, 2, 1><<<grid, 256, 0, st>>>(p, tpr_log2);
  count_launches(1);
  PF_CUDA_TRY(cudaGetLastError());
  return PF_OK;
}

template <typename VT, typename IT>
static pf_status launch_sddmm(pf_handle h, int64_t m, int64_t n, int64_t nnz, const IT *row_ptr,
                              const int32_t *col, int k, double alpha, const VT *dY, int64_t lddy,
                              const VT *X, int64_t ldx, double beta, VT *dval, cudaStream_t st) {
  PF_CHECK_ARG(h != nullptr, "null handle");
  PF_CHECK_ARG(m >= 0 && n >= 0 && nnz >= 0 && k >= 0, "negative size");
  if (m == 0 || nnz == 0) return PF_OK;
  PF_CHECK_ARG(dval, "null dval");
  pf_status s = check_wide<VT, IT>(h, m, n, nnz, row_ptr, col, dval, k, X, ldx, dY, lddy);
  if (s != PF_OK) return s;
  WideParams<VT, IT> p{m, n, nnz, row_ptr, col, nullptr, X, ldx, const_cast<VT *>(dY), lddy, dval,
                       k, (float)alpha, (float)beta, h->err};
  // warps a row: as many as it has non-zeros on average
  int wpr_log2 = 0;
  while (wpr_log2 < 3 && ((int64_t)m << wpr_log2) < nnz) ++wpr_log2;
  const unsigned grid =
      (unsigned)std::min<int64_t>(ceil_div(m, 8 >> wpr_log2), (int64_t)h->num_sms * 3);
  if (rows16(X, ldx) && rows16(dY, lddy))
    sddmm_kernel<VT, IT, 256, true><<<grid, 256, 0, st>>>(p, wpr_log2);
  else sddmm_kernel<VT, IT, 256, false><<<grid, 256, 0, st>>>(p, wpr_log2);
  count_launches(1);
  PF_CUDA_TRY(cudaGetLastError());
  return PF_OK;
}

}  // namespace pf

using namespace pf;

extern "C" {

// 16-bit values cross the C ABI as their raw bit patterns (uint16_t)
#define PF_DEFINE_WIDE(SUFFIX, VT, IT)                                                          \
  pf_status pf_spmm_##SUFFIX(pf_handle h, int64_t m, int64_t n, int64_t nnz, const IT *row_ptr, \
                             const int32_t *col_idx, const uint16_t *val, int k, double alpha,  \
                             const uint16_t *X, int64_t ldx, double beta, uint16_t *Y,          \
                             int64_t ldy, void *stream) {                                       \
    return launch_spmm16<VT, IT>(h, m, n, nnz, row_ptr, col_idx,                                \
                                 reinterpret_cast<const VT *>(val), k, alpha,                   \
                                 reinterpret_cast<const VT *>(X), ldx, beta,                    \
                                 reinterpret_cast<VT *>(Y), ldy, (cudaStream_t)stream);         \
  }                                                                                             \
  pf_status pf_sddmm_##SUFFIX(pf_handle h, int64_t m, int64_t n, int64_t nnz,                   \
                              const IT *row_ptr, const int32_t *col_idx, int k, double alpha,   \
                              const uint16_t *dY, int64_t lddy, const uint16_t *X, int64_t ldx, \
                              double beta, uint16_t *dval, void *stream) {                      \
    return launch_sddmm<VT, IT>(h, m, n, nnz, row_ptr, col_idx, k, alpha,                       \
                                reinterpret_cast<const VT *>(dY), lddy,                         \
                                reinterpret_cast<const VT *>(X), ldx, beta,                     \
                                reinterpret_cast<VT *>(dval), (cudaStream_t)stream);            \
  }

PF_DEFINE_WIDE(f16_i32, __half, int32_t)
PF_DEFINE_WIDE(f16_i64, __half, int64_t)
PF_DEFINE_WIDE(bf16_i32, __nv_bfloat16, int32_t)
PF_DEFINE_WIDE(bf16_i64, __nv_bfloat16, int64_t)

}  // extern "C"
