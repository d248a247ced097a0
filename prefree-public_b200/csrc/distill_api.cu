// C-ABI of the distillation loss (distill.cuh).
#include <algorithm>

#include "distill.cuh"
#include "pf_handle.cuh"

namespace pf {

constexpr int kMaxDevices = 64;

template <typename VT, typename IT, int NT, bool GRAD>
static pf_status launch_kernel(pf_handle h, const DistillParams<VT, IT> &p, int C,
                               cudaStream_t st) {
  using Cfg = DistillCfg<VT, NT>;
  auto kern = distill_kernel<VT, IT, NT, GRAD>;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(NT + 64);
  cfg.dynamicSmemBytes = Cfg::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = C;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  // clusters that the device holds at once, per device and size (0 = not yet)
  static int held[kMaxDevices][DISTILL_MAX_C + 1] = {};
  int &most = held[h->device % kMaxDevices][C];
  if (most == 0) {
    PF_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM));
    cfg.gridDim = dim3(C);
    int v = 0;
    PF_CUDA_TRY(cudaOccupancyMaxActiveClusters(&v, kern, &cfg));
    most = std::max(1, v);
  }
  cfg.gridDim = dim3((unsigned)(std::min<int64_t>(p.m, most) * C));
  PF_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, p));
  count_launches(1);
  return PF_OK;
}

// CTAs a row and threads a CTA. One CTA a row, of the fewest threads that take
// it at once; few rows are spread over more CTAs, until they fill the GPU, and
// so are rows whose gradient is to find them in L2 (kRowsInHand bytes at most
// in hand on the whole GPU).
constexpr int64_t kRowsInHand = 40 << 20;

template <typename VT, typename IT, bool GRAD>
static pf_status launch_rows(pf_handle h, const DistillParams<VT, IT> &p, cudaStream_t st) {
  constexpr int64_t SMALL = DistillCfg<VT, 64>::PIECE;
  const int64_t need = ceil_div(p.n, DistillCfg<VT, 64>::VE) + 1;  // pieces
  int C = 1;
  while (GRAD && C < DISTILL_MAX_C && need > C * 4 * SMALL &&
         need * 16 * (2 * h->num_sms / C) > kRowsInHand)
    C *= 2;
  while (C < DISTILL_MAX_C && p.m * C * 2 <= h->num_sms && need > C * SMALL) C *= 2;
  if (need <= C * SMALL) return launch_kernel<VT, IT, 64, GRAD>(h, p, C, st);
  if (need <= C * 2 * SMALL) return launch_kernel<VT, IT, 128, GRAD>(h, p, C, st);
  return launch_kernel<VT, IT, 256, GRAD>(h, p, C, st);
}

template <typename VT, typename IT>
static pf_status launch_distill(pf_handle h, int64_t m, int64_t n, int64_t nnz, const IT *row_ptr,
                                const int32_t *col, const VT *val, double temperature, const VT *Z,
                                int64_t ldz, const float *weight, float *loss, VT *dZ,
                                int64_t lddz, cudaStream_t st) {
  PF_CHECK_ARG(h != nullptr, "null handle");
  PF_CHECK_ARG(m >= 0 && n >= 0 && nnz >= 0, "negative size (m=%lld n=%lld nnz=%lld)",
               (long long)m, (long long)n, (long long)nnz);
  PF_CHECK_ARG(temperature > 0.0 && temperature <= 1e30 && temperature >= 1e-30,
               "temperature %g outside [1e-30, 1e30]", temperature);
  if (m == 0) return PF_OK;
  PF_CHECK_ARG(n <= (int64_t)INT32_MAX - 16, "n must be at most 2^31 - 17");
  PF_CHECK_ARG(loss || dZ, "neither loss nor dZ is asked for");
  PF_CHECK_ARG(row_ptr, "null row_ptr");
  PF_CHECK_ARG(nnz == 0 || (col && val), "null col/val with nnz > 0");
  PF_CHECK_ARG(nnz == 0 || n > 0, "nnz > 0 needs n > 0 (column indices lie in [0, n))");
  PF_CHECK_ARG(n == 0 || Z, "null Z");
  PF_CHECK_ARG(sizeof(IT) == 8 || nnz <= INT32_MAX, "int32 row_ptr cannot index nnz=%lld",
               (long long)nnz);
  PF_CHECK_ARG(ldz >= n && (!dZ || lddz >= n), "leading dimension below n");
  PF_CHECK_ARG(!dZ || (const void *)dZ != (const void *)Z || lddz == ldz,
               "dZ in Z's place needs lddz == ldz");
  PF_CHECK_ARG(((uintptr_t)row_ptr % sizeof(IT)) == 0 && ((uintptr_t)col % 4) == 0 &&
                   ((uintptr_t)val % sizeof(VT)) == 0 && ((uintptr_t)Z % sizeof(VT)) == 0 &&
                   ((uintptr_t)dZ % sizeof(VT)) == 0 && ((uintptr_t)weight % 4) == 0 &&
                   ((uintptr_t)loss % 4) == 0,
               "arrays must be aligned to their element size");
  int cur = 0;
  PF_CUDA_TRY(cudaGetDevice(&cur));
  PF_CHECK_ARG(cur == h->device, "handle bound to device %d, current device is %d", h->device, cur);
  if (n == 0) {
    // no entries, no gradient; and no slots, by whose release the kernel keeps
    // its warps within DISTILL_RING rows of one another
    if (loss) PF_CUDA_TRY(cudaMemsetAsync(loss, 0, m * sizeof(float), st));
    return PF_OK;
  }
  DistillParams<VT, IT> p;
  p.m = m;
  p.n = n;
  p.nnz = nnz;
  p.row_ptr = p.row_ptr0 = row_ptr;
  p.col = col;
  p.val = val;
  p.Z = Z;
  p.ldz = ldz;
  p.weight = weight;
  p.loss = loss;
  p.dZ = dZ;
  p.lddz = lddz;
  p.inv_tau = (float)(1.0 / temperature);
  p.err = h->err;
  return dZ ? launch_rows<VT, IT, true>(h, p, st) : launch_rows<VT, IT, false>(h, p, st);
}

}  // namespace pf

using namespace pf;

extern "C" {

// 16-bit values cross the C ABI as their raw bit patterns (uint16_t)
#define PF_DEFINE_DISTILL(SUFFIX, VT, CT, IT)                                              \
  pf_status pf_distill_##SUFFIX(pf_handle h, int64_t m, int64_t n, int64_t nnz,            \
                                const IT *row_ptr, const int32_t *col_idx, const CT *val,  \
                                double temperature, const CT *Z, int64_t ldz,              \
                                const float *weight, float *loss, CT *dZ, int64_t lddz,    \
                                void *stream) {                                            \
    return launch_distill<VT, IT>(h, m, n, nnz, row_ptr, col_idx,                          \
                                  reinterpret_cast<const VT *>(val), temperature,          \
                                  reinterpret_cast<const VT *>(Z), ldz, weight, loss,      \
                                  reinterpret_cast<VT *>(dZ), lddz, (cudaStream_t)stream); \
  }

PF_DEFINE_DISTILL(f32_i32, float, float, int32_t)
PF_DEFINE_DISTILL(f32_i64, float, float, int64_t)
PF_DEFINE_DISTILL(f16_i32, __half, uint16_t, int32_t)
PF_DEFINE_DISTILL(f16_i64, __half, uint16_t, int64_t)
PF_DEFINE_DISTILL(bf16_i32, __nv_bfloat16, uint16_t, int32_t)
PF_DEFINE_DISTILL(bf16_i64, __nv_bfloat16, uint16_t, int64_t)

}  // extern "C"
