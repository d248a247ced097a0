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

// Dense rows start anywhere. A row is cut into the 16-byte pieces of memory that
// it lies in; Y's pieces give the columns that a thread holds, and X's columns
// for one of them lie in two of X's pieces, `d` elements further. The second
// piece is the neighbour thread's first (a hit in L1), and the shift is the same
// for a whole row: eight cases with fixed registers. (Elements one by one, or
// pairs in 4-byte words, took 127 and 142 us instead of 33 for the gradients of
// 3001 tokens of four slots, 1531 columns.) Elements of neighbours are never
// stored, and masked where they would be summed.
template <typename VT>
struct DenseRow {
  const uint4 *piece;  // its first 16-byte piece
  int shift;           // elements before the row in it
  int count;           // pieces
  __device__ __forceinline__ DenseRow(const VT *row, int64_t k) {
    shift = (int)(((uintptr_t)row & 15) / sizeof(VT));
    piece = reinterpret_cast<const uint4 *>(row - shift);
    count = (int)((k + shift + 7) / 8);
  }
};

// elements d .. d + 7 of two pieces
__device__ __forceinline__ uint4 shifted(const uint4 &a, const uint4 &b, int d) {
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#define PF_EVEN(i) make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3])
#define PF_ODD(i)                                                                         \
  make_uint4(__funnelshift_r(w[i], w[i + 1], 16), __funnelshift_r(w[i + 1], w[i + 2], 16), \
             __funnelshift_r(w[i + 2], w[i + 3], 16), __funnelshift_r(w[i + 3], w[i + 4], 16))
  switch (d) {
    case 0: return PF_EVEN(0);
    case 1: return PF_ODD(0);
    case 2: return PF_EVEN(1);
    case 3: return PF_ODD(1);
    case 4: return PF_EVEN(2);
    case 5: return PF_ODD(2);
    case 6: return PF_EVEN(3);
    default: return PF_ODD(3);
  }
#undef PF_EVEN
#undef PF_ODD
}

// The columns of X's row that lie at piece v of a row that starts `shift`
// elements into its first piece: load() the pieces, get() the elements.
template <typename VT, bool ALIGNED>
struct Gather {
  uint4 a, b;
  __device__ __forceinline__ void load(const DenseRow<VT> &x, int v, int shift) {
    if (ALIGNED) {
      a = __ldg(x.piece + v);
      return;
    }
    const int delta = x.shift - shift, p = v + (delta >> 3), d = delta & 7;
    a = b = make_uint4(0, 0, 0, 0);
    if (p >= 0 && p < x.count) a = __ldg(x.piece + p);
    if (d != 0 && p + 1 < x.count) b = __ldg(x.piece + p + 1);
  }
  __device__ __forceinline__ void get(int delta, float (&out)[8]) const {
    unpack<VT>(ALIGNED ? a : shifted(a, b, delta & 7), out);
  }
};

// The bounds of the CSR's rows, checked: empty and flagged where the pointers are
// not non-decreasing within [row_ptr[0], row_ptr[0] + nnz].
template <typename VT, typename IT>
struct RowWalk {
  const WideParams<VT, IT> &P;
  int64_t base, s = 0, e = 0;
  __device__ __forceinline__ RowWalk(const WideParams<VT, IT> &p)
      : P(p), base((int64_t)p.row_ptr[0]) {}
  __device__ __forceinline__ void fetch(int64_t r) {  // nothing is waited for
    if (r < P.m) s = (int64_t)P.row_ptr[r], e = (int64_t)P.row_ptr[r + 1];
    else s = e = base;
  }
  __device__ __forceinline__ void check(bool flag) {
    if (s < base || e < s || e > base + P.nnz) {
      if (flag) atomicOr(P.err, PF_DEVERR_ROWPTR);
      s = e = base;
    }
  }
};

// 2^tpr_log2 threads a row, each Q pieces of columns at a time; B non-zeros are
// gathered before the first is used: 64 bytes on their way to a thread. While a
// row is worked on, the next one's first columns and values and the bounds of
// the one after that are fetched: a row costs one latency instead of three
// (62259 rows of one non-zero, 2048 columns: 109 us without).
template <typename VT, typename IT, int NT, bool ALIGNED, int B, int Q>
__global__ void __launch_bounds__(NT, ALIGNED ? 4 : 3)
spmm_wide_kernel(const WideParams<VT, IT> P, int tpr_log2) {
  const int tpr = 1 << tpr_log2;
  const int sub = threadIdx.x & (tpr - 1);
  const int64_t step = (int64_t)gridDim.x * (NT >> tpr_log2);
  const int64_t r0 = (int64_t)blockIdx.x * (NT >> tpr_log2) + (threadIdx.x >> tpr_log2);
  const bool flag = sub == 0 && blockIdx.y == 0;
  RowWalk<VT, IT> next(P);
  next.fetch(r0);
  int64_t s = 0, e = 0;
  uint32_t col[B];
  VT val[B];
  auto entries = [&](int64_t i, int64_t end) {
#pragma unroll
    for (int b = 0; b < B; ++b) {
      col[b] = 0xffffffffu;
      if (i + b < end) col[b] = (uint32_t)P.col[i + b], val[b] = P.val[i + b];
    }
  };
  next.check(flag && r0 < P.m);
  s = next.s, e = next.e;
  entries(s, e);
  next.fetch(r0 + step);
  for (int64_t r = r0; r < P.m; r += step) {
    VT *y = P.Y + r * P.ldy;
    const DenseRow<VT> Y(y, P.k);
    const int shift = ALIGNED ? 0 : Y.shift;
    bool fetched = true;  // whether col and val are the row's first
    for (int v = blockIdx.y * tpr * Q + sub; v < Y.count; v += gridDim.y * tpr * Q) {
      float acc[Q][8] = {};
      for (int64_t i = s; i < e; i += B) {
        if (!fetched) entries(i, e);
        fetched = false;
        Gather<VT, ALIGNED> x[B][Q];
        int delta[B];
#pragma unroll
        for (int b = 0; b < B; ++b) {
          if (col[b] >= (uint64_t)P.n) {
            if (i + b < e) atomicOr(P.err, PF_DEVERR_BOUNDS);
            col[b] = 0xffffffffu;
            continue;
          }
          const DenseRow<VT> X(P.X + (int64_t)col[b] * P.ldx, P.k);
          delta[b] = X.shift - shift;
#pragma unroll
          for (int q = 0; q < Q; ++q)
            if (v + q * tpr < Y.count) x[b][q].load(X, v + q * tpr, shift);
        }
#pragma unroll
        for (int b = 0; b < B; ++b) {
          if (col[b] == 0xffffffffu) continue;
          const float a = to_f32(val[b]);
#pragma unroll
          for (int q = 0; q < Q; ++q)
            if (v + q * tpr < Y.count) {
              float f[8];
              x[b][q].get(delta[b], f);
#pragma unroll
              for (int z = 0; z < 8; ++z) acc[q][z] = fmaf(a, f[z], acc[q][z]);
            }
        }
      }
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const int p = v + q * tpr;
        if (p >= Y.count) continue;
        VT *to = y - shift + (int64_t)p * 8;
        const int lo = p == 0 ? shift : 0;
        const int hi = (int)min((int64_t)8, P.k + shift - (int64_t)p * 8);
        const bool whole = lo == 0 && hi == 8;
        if (P.beta != 0.0f) {
          float old[8] = {};
          if (whole) unpack<VT>(*reinterpret_cast<const uint4 *>(to), old);
          else
#pragma unroll
            for (int z = 0; z < 8; ++z)
              if (z >= lo && z < hi) old[z] = to_f32(to[z]);
#pragma unroll
          for (int z = 0; z < 8; ++z) acc[q][z] = P.alpha * acc[q][z] + P.beta * old[z];
        } else {
#pragma unroll
          for (int z = 0; z < 8; ++z) acc[q][z] *= P.alpha;
        }
        if (whole) {
          __stcs(reinterpret_cast<uint4 *>(to), pack<VT>(acc[q]));
        } else {
#pragma unroll
          for (int z = 0; z < 8; ++z)
            if (z >= lo && z < hi) to[z] = from_f32<VT>(acc[q][z]);
        }
      }
    }
    next.check(flag && r + step < P.m);
    s = next.s, e = next.e;
    entries(s, e);
    next.fetch(r + 2 * step);
  }
}

// 2^wpr_log2 warps a row; a warp takes one non-zero at a time, Q pieces of both
// dense rows on their way to a lane. The next row's bounds and first column are
// fetched ahead, as above.
template <typename VT, typename IT, int NT, bool ALIGNED>
__global__ void __launch_bounds__(NT, 4)
sddmm_kernel(const WideParams<VT, IT> P, int wpr_log2) {
  constexpr int Q = ALIGNED ? 4 : 2;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int wpr = 1 << wpr_log2, mine = warp & (wpr - 1);
  const int64_t step = (int64_t)gridDim.x * ((NT / 32) >> wpr_log2);
  const int64_t r0 = (int64_t)blockIdx.x * ((NT / 32) >> wpr_log2) + (warp >> wpr_log2);
  const bool flag = lane == 0 && mine == 0;
  RowWalk<VT, IT> next(P);
  next.fetch(r0);
  next.check(flag && r0 < P.m);
  int64_t s = next.s, e = next.e;
  uint32_t first = s + mine < e ? (uint32_t)P.col[s + mine] : 0;
  next.fetch(r0 + step);
  for (int64_t r = r0; r < P.m; r += step) {
    const DenseRow<VT> Y(P.Y + r * P.ldy, P.k);
    const int shift = ALIGNED ? 0 : Y.shift;
    for (int64_t i = s + mine; i < e; i += wpr) {
      const uint32_t col = i == s + mine ? first : (uint32_t)P.col[i];
      if (col >= (uint64_t)P.n) {
        if (lane == 0) atomicOr(P.err, PF_DEVERR_BOUNDS);
        continue;
      }
      const DenseRow<VT> X(P.X + (int64_t)col * P.ldx, P.k);
      float acc[8] = {};
      for (int v = lane; v < Y.count; v += 32 * Q) {
        Gather<VT, ALIGNED> x[Q];
        uint4 y[Q];
#pragma unroll
        for (int q = 0; q < Q; ++q)
          if (v + 32 * q < Y.count) {
            x[q].load(X, v + 32 * q, shift);
            y[q] = __ldg(Y.piece + v + 32 * q);
          }
#pragma unroll
        for (int q = 0; q < Q; ++q) {
          const int p = v + 32 * q;
          if (p >= Y.count) continue;
          float f[8], g[8];
          x[q].get(X.shift - shift, f);
          unpack<VT>(y[q], g);
          const int lo = p == 0 ? shift : 0;
          const int hi = (int)min((int64_t)8, P.k + shift - (int64_t)p * 8);
          if (lo == 0 && hi == 8) {
#pragma unroll
            for (int z = 0; z < 8; ++z) acc[z] = fmaf(f[z], g[z], acc[z]);
          } else {
#pragma unroll
            for (int z = 0; z < 8; ++z)
              if (z >= lo && z < hi) acc[z] = fmaf(f[z], g[z], acc[z]);
          }
        }
      }
      float sum = ((acc[0] + acc[1]) + (acc[2] + acc[3])) + ((acc[4] + acc[5]) + (acc[6] + acc[7]));
      sum = warp_sum(sum);
      if (lane == 0) {
        float out = P.alpha * sum;
        if (P.beta != 0.0f) out += P.beta * to_f32(P.dval[i]);
        P.dval[i] = from_f32<VT>(out);
      }
    }
    next.check(flag && r + step < P.m);
    s = next.s, e = next.e;
    first = s + mine < e ? (uint32_t)P.col[s + mine] : 0;
    next.fetch(r + 2 * step);
  }
}

}  // namespace pf
