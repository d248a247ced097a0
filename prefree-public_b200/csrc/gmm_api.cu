// C-ABI of the grouped matrix products.
#include <algorithm>
#include <type_traits>

#include "gmm_simt.cuh"
#include "gmm_tc.cuh"
#include "pf_handle.cuh"

namespace pf {

// largest size: the kernels' 32-bit coordinates run up to a tile past the end
constexpr int64_t kMost = INT32_MAX - 1024;

// cuTensorMapEncodeTiled, looked up at run time (the library does not link
// against the driver); null where there is none
typedef CUresult (*EncodeFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *,
                             const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                             const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeFn encode_fn() {
  static EncodeFn fn = [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &r) !=
            cudaSuccess || r != cudaDriverEntryPointSuccess)
      p = nullptr;
    return (EncodeFn)p;
  }();
  return fn;
}

// A map of `planes` row-major matrices (rows x cols, leading dimension ld,
// `plane` elements apart; planes = 0: one matrix, a 2-d map) for boxes of 64
// columns x box_rows rows, 128-byte swizzle, zeros outside.
template <typename VT>
static pf_status encode(CUtensorMap *map, const VT *base, int64_t cols, int64_t rows, int64_t ld,
                        int64_t planes, int64_t plane, int box_rows) {
  const EncodeFn fn = encode_fn();
  if (!fn) {
    set_error("cuTensorMapEncodeTiled is not available");
    return PF_ERR_CUDA;
  }
  const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)planes};
  const cuuint64_t strides[2] = {(cuuint64_t)ld * sizeof(VT), (cuuint64_t)plane * sizeof(VT)};
  const cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1}, one[3] = {1, 1, 1};
  const CUtensorMapDataType type = std::is_same<VT, __half>::value
                                       ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                       : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const CUresult r = fn(map, type, planes ? 3 : 2, const_cast<VT *>(base), dims, strides, box, one,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled: error %d", (int)r);
    return PF_ERR_CUDA;
  }
  return PF_OK;
}

// what a tensor map takes: 16-byte aligned base and strides
template <typename VT>
static bool tma_ready(const VT *base, int64_t ld, int64_t plane = 0) {
  return ((uintptr_t)base % 16) == 0 && ld % 8 == 0 && plane % 8 == 0 && ld < (1LL << 38) &&
         plane < (1LL << 38);
}

template <typename OT>
static bool rows_aligned(const OT *c, int64_t ld, int64_t plane) {
  return ((uintptr_t)c % 16) == 0 && ld * sizeof(OT) % 16 == 0 && plane * sizeof(OT) % 16 == 0;
}

// no more row tiles than whole ones and one partial one to a group
static int64_t most_tiles(int64_t groups, int64_t rows, int bn) {
  return rows / bn + std::min(groups, rows);
}

// Scratch for split sums: tiles x parts are at most the SMs (parts_for), so one
// size serves every call. Made by the handle's first such call and kept as
// long as the handle: graphs captured since hold its address.
template <typename IT, typename OT>
static pf_status split_scratch(pf_handle h, int64_t tiles, GmmTcParams<IT, OT> *p,
                               cudaStream_t st) {
  if (!h->gmm_partial) {
    // (a captured clearing would leave the counters as they are until a replay)
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    PF_CUDA_TRY(cudaStreamIsCapturing(st, &capture));
    if (capture != cudaStreamCaptureStatusNone) {
      set_error("the handle's first grouped product with split sums allocates: "
                "make one before the stream capture");
      return PF_ERR_UNSUPPORTED;
    }
    const size_t sums = sizeof(float) * 128 * 128 * h->num_sms;
    float *partial = nullptr;
    PF_CUDA_TRY(cudaMalloc(&partial, sums + h->gmm_counters() * sizeof(unsigned)));
    h->gmm_arrived = reinterpret_cast<unsigned *>(reinterpret_cast<char *>(partial) + sums);
    const cudaError_t e =
        cudaMemsetAsync(h->gmm_arrived, 0, h->gmm_counters() * sizeof(unsigned), st);
    if (e != cudaSuccess) {
      cudaFree(partial);
      h->gmm_arrived = nullptr;
      PF_CUDA_TRY(e);
    }
    h->gmm_partial = partial;
  }
  p->most = tiles;
  p->partial = h->gmm_partial;
  p->arrived = h->gmm_arrived;
  return PF_OK;
}

template <int MODE, int CG, int BN, bool BF16, bool SPLIT, typename IT, typename OT>
static pf_status launch_tc(pf_handle h, const GmmMaps &maps, GmmTcParams<IT, OT> p,
                           cudaStream_t st) {
  using Cfg = GmmCfg<MODE, CG, BN>;
  auto kern = gmm_tc_kernel<MODE, CG, BN, BF16, SPLIT, IT, OT>;
  static bool ready[64] = {};  // the attribute is set once per device
  bool &done = ready[h->device % 64];
  if (!done) {
    PF_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM));
    done = true;
  }
  const int64_t ti = ceil_div(p.ni, Cfg::TI);
  int64_t tiles = MODE == GMM_DW ? p.groups * ti * ceil_div(p.nj, BN)
                                 : most_tiles(p.groups, p.rows, BN) * ti;
  if (SPLIT) {
    pf_status s = split_scratch(h, tiles, &p, st);
    if (s != PF_OK) return s;
    tiles *= p.parts;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(std::min<int64_t>(tiles, h->num_sms / CG) * CG));
  cfg.blockDim = dim3(Cfg::NT);
  cfg.dynamicSmemBytes = Cfg::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = CG;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  PF_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, maps, p));
  count_launches(1);
  return PF_OK;
}

// Parts of each sum (of `blocks` blocks of 64): as many as there are CTAs to a
// tile (tiles x parts are at most the SMs: split_scratch relies on it), of
// `least` blocks at least, eight parts at most. A join costs about what
// 16 blocks do, more where all 128 x 128 sums of the tile exist (a weight
// gradient); with more items than CTAs the joins come one after another (256
// tiles in 4 parts: 82 us instead of 42). 17 rows, n 512, k 4096: 23.0 -> 11.9
// us; gradient of 256 x 512 over 10000 rows: 49.7 -> 28.0.
static int parts_for(pf_handle h, int64_t tiles, int64_t blocks, int64_t least) {
  return (int)std::max<int64_t>(1, std::min<int64_t>({h->num_sms / tiles, blocks / least, 8}));
}

template <int MODE, typename VT, typename IT>
static pf_status product_tc(pf_handle h, const VT *X, int64_t ldx, const VT *W, int64_t ldw,
                            int64_t stride_w, int64_t k, GmmTcParams<IT, VT> p, cudaStream_t st) {
  constexpr bool BF16 = std::is_same<VT, __nv_bfloat16>::value;
  // 256 x 256 by CTA pairs where the groups fill more than a quarter of that;
  // 128 x 128 below, where the weights' bytes bound it and tiles are few (the
  // instruction's N follows the rows in either)
  const int64_t avg = p.rows / std::min(p.groups, p.rows);
  const bool pairs = avg > 64 && p.ni > 128;
  const bool fwd = MODE == GMM_FWD;
  GmmMaps maps = {};
  p.group_step = stride_w != 0 || p.groups == 1;
  const int64_t planes = p.group_step ? p.groups : 1;
  const int64_t plane = p.groups == 1 || !p.group_step ? (fwd ? p.ni : k) * ldw : stride_w;
  pf_status s = encode(&maps.a, W, fwd ? k : p.ni, fwd ? p.ni : k, ldw, planes, plane,
                       fwd ? 128 : 64);
  if (s != PF_OK) return s;
  s = encode(&maps.b, X, k, p.rows, ldx, 0, 0, 32);
  if (s != PF_OK) return s;
  if (pairs) return launch_tc<MODE, 2, 256, BF16, false>(h, maps, p, st);
  p.parts = parts_for(h, most_tiles(p.groups, p.rows, 128) * ceil_div(p.ni, 128),
                      ceil_div(k, 64), 8);
  if (p.parts > 1) return launch_tc<MODE, 1, 128, BF16, true>(h, maps, p, st);
  return launch_tc<MODE, 1, 128, BF16, false>(h, maps, p, st);
}

template <typename VT, typename OT, typename IT>
static pf_status wgrad_tc(pf_handle h, const VT *dY, int64_t lddy, const VT *X, int64_t ldx,
                          GmmTcParams<IT, OT> p, cudaStream_t st) {
  constexpr bool BF16 = std::is_same<VT, __nv_bfloat16>::value;
  GmmMaps maps = {};
  pf_status s = encode(&maps.a, X, p.ni, p.rows, ldx, 0, 0, 64);
  if (s != PF_OK) return s;
  s = encode(&maps.b, dY, p.nj, p.rows, lddy, 0, 0, 64);
  if (s != PF_OK) return s;
  const int64_t blocks = p.rows / p.groups / 64;
  p.parts = parts_for(h, p.groups * ceil_div(p.ni, 128) * ceil_div(p.nj, 128), blocks, 16);
  if (p.parts > 1) return launch_tc<GMM_DW, 1, 128, BF16, true>(h, maps, p, st);
  if (p.ni > 128 && p.nj > 128) return launch_tc<GMM_DW, 2, 256, BF16, false>(h, maps, p, st);
  return launch_tc<GMM_DW, 1, 128, BF16, false>(h, maps, p, st);
}

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
  PF_CHECK_ARG(groups <= kMost && n <= kMost && k <= kMost && rows <= kMost,
               "groups, rows, n and k must be at most 2^31 - 1025");
  PF_CHECK_ARG(ptr && Y, "null group_ptr or Y");
  PF_CHECK_ARG(k == 0 || (X && W), "null X/W with k > 0");
  const int64_t wcols = trans_w ? k : n, wrows = trans_w ? n : k;
  PF_CHECK_ARG(ldx >= k && ldw >= wcols && ldy >= n, "leading dimension below the row's length");
  PF_CHECK_ARG(groups == 1 || wrows == 0 || stride_w == 0 ||
                   stride_w >= (wrows - 1) * ldw + wcols,
               "stride_w below one matrix");
  PF_CHECK_ARG(((uintptr_t)ptr % sizeof(IT)) == 0 && ((uintptr_t)X % sizeof(VT)) == 0 &&
                   ((uintptr_t)W % sizeof(VT)) == 0 && ((uintptr_t)Y % sizeof(VT)) == 0,
               "arrays must be aligned to their element size");
  int cur = 0;
  PF_CUDA_TRY(cudaGetDevice(&cur));
  PF_CHECK_ARG(cur == h->device, "handle bound to device %d, current device is %d", h->device, cur);
  if (k > 0 && tma_ready(X, ldx) && tma_ready(W, ldw, groups > 1 ? stride_w : 0)) {
    GmmTcParams<IT, VT> p{groups, rows, (int)n, 0, (int)k, 1, ptr, Y, ldy, 0,
                          (float)alpha, (float)beta, 1, 0, nullptr, nullptr, rows_aligned(Y, ldy, 0),
                          beta == 0.0 && rows_aligned(Y, ldy, 0), h->err};
    return trans_w ? product_tc<GMM_FWD>(h, X, ldx, W, ldw, stride_w, k, p, st)
                   : product_tc<GMM_DX>(h, X, ldx, W, ldw, stride_w, k, p, st);
  }
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
  PF_CHECK_ARG(groups <= kMost && n <= kMost && k <= kMost && rows <= kMost,
               "groups, rows, n and k must be at most 2^31 - 1025");
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
  if (rows > 0 && tma_ready(X, ldx) && tma_ready(dY, lddy)) {
    GmmTcParams<IT, OT> p{groups, rows, (int)k, (int)n, 0, 1, ptr, dW, lddw, stride_dw,
                          (float)alpha, (float)beta, 1, 0, nullptr, nullptr, rows_aligned(dW, lddw, stride_dw),
                          beta == 0.0 && rows_aligned(dW, lddw, stride_dw), h->err};
    return wgrad_tc<VT>(h, dY, lddy, X, ldx, p, st);
  }
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
