// 16-bit SpMM over wide dense rows, Y = alpha * A * X + beta * Y, and the
// gradient of its values, dval_j = alpha * <dY[row(j), :], X[col_j, :]> +
// beta * dval_j (a dense-dense product sampled at A's non-zeros).
//
// The dense rows are long (hundreds to thousands of 16-bit values) and the
// CSR rows short: the bytes of X and Y bound both, so threads run along the
// dense row. Products of 16-bit values are exact in fp32 (alpha is multiplied
// into the SpMM's values first); sums are in fp32 in the row's order (the same
// bits on every run) and rounded once. Measured: 8192 rows of eight non-zeros,
// 2048 columns, 57 us (5.3 TB/s, 80 % of the copy rate); 62259 rows of one
// non-zero 79 us; the values' gradient of the former 56 us.
#pragma once

#include "pf_values.cuh"

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
// piece is the neighbour thread's first (a hit in L1). (Elements one by one, or
// pairs in 4-byte words, took 127 and 142 us instead of 41-43 for the gradients of
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
    count = k > 0 ? (int)((k + shift + 7) / 8) : 0;
  }
};

// elements d .. d + 7 of two pieces: by 4, 2 and 1 elements, in registers
__device__ __forceinline__ uint4 shifted(const uint4 &a, const uint4 &b, int d) {
  const bool four = (d & 4) != 0, two = (d & 2) != 0;
  const uint32_t u0 = four ? a.z : a.x, u1 = four ? a.w : a.y, u2 = four ? b.x : a.z,
                 u3 = four ? b.y : a.w, u4 = four ? b.z : b.x, u5 = four ? b.w : b.y;
  const uint32_t v0 = two ? u1 : u0, v1 = two ? u2 : u1, v2 = two ? u3 : u2, v3 = two ? u4 : u3,
                 v4 = two ? u5 : u4;
  const int by = (d & 1) * 16;
  return make_uint4(__funnelshift_r(v0, v1, by), __funnelshift_r(v1, v2, by),
                    __funnelshift_r(v2, v3, by), __funnelshift_r(v3, v4, by));
}

// The columns of X's row that lie at piece v of a row that starts `shift`
// elements into its first piece: load() the pieces, get() the elements.
template <typename VT, bool ALIGNED>
struct Gather {
  uint4 a, b;
  __device__ __forceinline__ void load(const DenseRow<VT> &x, int v, int delta) {
    if (ALIGNED) {
      a = __ldg(x.piece + v);
      return;
    }
    const int p = v + (delta >> 3);
    a = b = make_uint4(0, 0, 0, 0);
    if ((uint32_t)p < (uint32_t)x.count) a = __ldg(x.piece + p);
    if ((delta & 7) != 0 && p + 1 < x.count) b = __ldg(x.piece + p + 1);
  }
  __device__ __forceinline__ void get(int delta, float (&out)[8]) const {
    unpack<VT>(ALIGNED ? a : shifted(a, b, delta & 7), out);
  }
};

// Places within a row, counted from its first entry: unsigned, so that steps
// past the end of a row that ends at the largest signed index do not wrap.
template <typename IT>
using Place = typename std::make_unsigned<IT>::type;

// The bounds of the CSR's rows, checked: empty and flagged where the pointers are
// not non-decreasing within [row_ptr[0], row_ptr[0] + nnz].
template <typename VT, typename IT>
struct RowWalk {
  const IT *ptr;
  int64_t m;
  IT base, last, s, e;
  __device__ __forceinline__ RowWalk(const WideParams<VT, IT> &p)
      : ptr(p.row_ptr), m(p.m), base(p.row_ptr[0]) {
    const int64_t end = (int64_t)base + p.nnz;
    last = sizeof(IT) == 4 && end > INT32_MAX ? (IT)INT32_MAX : (IT)end;
  }
  __device__ __forceinline__ void fetch(int64_t r) {  // nothing is waited for
    s = e = base;
    if (r < m) s = ptr[r], e = ptr[r + 1];
  }
  __device__ __forceinline__ void check(bool flag, unsigned *err) {
    if (s < base || e < s || e > last) {
      if (flag) atomicOr(err, PF_DEVERR_ROWPTR);
      s = e = base;
    }
  }
};

// 2^tpr_log2 threads a row, each Q pieces of columns at a time; B non-zeros are
// gathered before the first is used: 64 bytes on their way to a thread. While a
// row is worked on, the next one's first columns and values and the bounds of
// the one after that are fetched: a row costs one latency instead of three.
// What bounds it besides DRAM is the number of instructions, so alpha goes into
// the values, and whole pieces take a path without masks.
template <typename VT, typename IT, int NT, bool ALIGNED, int B, int Q>
__global__ void __launch_bounds__(NT, ALIGNED ? 4 : 3)
spmm_wide_kernel(const WideParams<VT, IT> P, int tpr_log2) {
  const int tpr = 1 << tpr_log2;
  const int sub = threadIdx.x & (tpr - 1);
  const int64_t step = (int64_t)gridDim.x * (NT >> tpr_log2);
  const int64_t r0 = (int64_t)blockIdx.x * (NT >> tpr_log2) + (threadIdx.x >> tpr_log2);
  const bool flag = sub == 0 && blockIdx.y == 0;
  const uint32_t n = (uint32_t)min(P.n, (int64_t)0xffffffff);
  const int k = (int)P.k;
  RowWalk<VT, IT> next(P);
  next.fetch(r0);
  uint32_t col[B];
  VT val[B];
  auto entries = [&](IT i, IT end) {
#pragma unroll
    for (int b = 0; b < B; ++b) {
      col[b] = 0xffffffffu;
      if (end - i > b) col[b] = (uint32_t)P.col[i + b], val[b] = P.val[i + b];
    }
  };
  next.check(flag && r0 < P.m, P.err);
  IT s = next.s, e = next.e;
  entries(s, e);
  next.fetch(r0 + step);
  for (int64_t r = r0; r < P.m; r += step) {
    VT *y = P.Y + r * P.ldy;
    const DenseRow<VT> Y(y, k);
    const int shift = ALIGNED ? 0 : Y.shift, count = Y.count;
    // pieces first_whole .. last_whole are all the row's
    const int first_whole = shift > 0, last_whole = count - 1 - ((k + shift) % 8 != 0);
    bool fetched = true;  // whether col and val are the row's first
    for (int v = blockIdx.y * tpr * Q + sub; v < count; v += gridDim.y * tpr * Q) {
      float acc[Q][8] = {};
      const Place<IT> left = (Place<IT>)e - (Place<IT>)s;
      for (Place<IT> i = 0; i < left; i += B) {
        if (!fetched) entries(s + (IT)i, e);
        fetched = false;
        Gather<VT, ALIGNED> x[B][Q];
        int delta[B];
#pragma unroll
        for (int b = 0; b < B; ++b) {
          if (col[b] >= n) {
            if (left - i > b) atomicOr(P.err, PF_DEVERR_BOUNDS);
            col[b] = 0xffffffffu;
            continue;
          }
          const DenseRow<VT> X(P.X + (int64_t)col[b] * P.ldx, k);
          delta[b] = ALIGNED ? 0 : X.shift - shift;
#pragma unroll
          for (int q = 0; q < Q; ++q)
            if (v + q * tpr < count) x[b][q].load(X, v + q * tpr, delta[b]);
        }
#pragma unroll
        for (int b = 0; b < B; ++b) {
          if (col[b] == 0xffffffffu) continue;
          const float a = P.alpha * to_f32(val[b]);
#pragma unroll
          for (int q = 0; q < Q; ++q) {
            float f[8];
            x[b][q].get(delta[b], f);  // (past the row: not stored)
#pragma unroll
            for (int z = 0; z < 8; ++z) acc[q][z] = fmaf(a, f[z], acc[q][z]);
          }
        }
      }
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const int p = v + q * tpr;
        VT *to = y - shift + (int64_t)p * 8;
        if (p >= first_whole && p <= last_whole) {
          if (P.beta != 0.0f) {
            float old[8];
            unpack<VT>(*reinterpret_cast<const uint4 *>(to), old);
#pragma unroll
            for (int z = 0; z < 8; ++z) acc[q][z] = fmaf(P.beta, old[z], acc[q][z]);
          }
          __stcs(reinterpret_cast<uint4 *>(to), pack<VT>(acc[q]));
        } else if (p < count) {
          const int lo = p == 0 ? shift : 0, hi = min(8, k + shift - p * 8);
#pragma unroll
          for (int z = 0; z < 8; ++z)
            if (z >= lo && z < hi) {
              float o = acc[q][z];
              if (P.beta != 0.0f) o = fmaf(P.beta, to_f32(to[z]), o);
              to[z] = from_f32<VT>(o);
            }
        }
      }
    }
    next.check(flag && r + step < P.m, P.err);
    s = next.s, e = next.e;
    entries(s, e);
    next.fetch(r + 2 * step);
  }
}

// 2^wpr_log2 warps a row; a warp takes one non-zero at a time, Q pieces of both
// dense rows on their way to a lane. The next row's bounds and first column are
// fetched ahead, as above.
template <typename VT, typename IT, int NT, bool ALIGNED>
__global__ void __launch_bounds__(NT, 3)
sddmm_kernel(const WideParams<VT, IT> P, int wpr_log2) {
  constexpr int Q = ALIGNED ? 4 : 3;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int wpr = 1 << wpr_log2, mine = warp & (wpr - 1);
  const int64_t step = (int64_t)gridDim.x * ((NT / 32) >> wpr_log2);
  const int64_t r0 = (int64_t)blockIdx.x * ((NT / 32) >> wpr_log2) + (warp >> wpr_log2);
  const bool flag = lane == 0 && mine == 0;
  const int k = (int)P.k;
  RowWalk<VT, IT> next(P);
  next.fetch(r0);
  next.check(flag && r0 < P.m, P.err);
  IT s = next.s, e = next.e;
  const uint32_t n = (uint32_t)min(P.n, (int64_t)0xffffffff);
  uint32_t first = e - s > mine ? (uint32_t)P.col[s + mine] : 0;
  next.fetch(r0 + step);
  for (int64_t r = r0; r < P.m; r += step) {
    const DenseRow<VT> Y(P.Y + r * P.ldy, k);
    const int shift = ALIGNED ? 0 : Y.shift, count = Y.count;
    const int first_whole = shift > 0, last_whole = count - 1 - ((k + shift) % 8 != 0);
    const Place<IT> left = (Place<IT>)e - (Place<IT>)s;
    for (Place<IT> at = mine; at < left; at += wpr) {
      const IT i = s + (IT)at;
      const uint32_t col = at == (Place<IT>)mine ? first : (uint32_t)P.col[i];
      if (col >= n) {
        if (lane == 0) atomicOr(P.err, PF_DEVERR_BOUNDS);
        continue;
      }
      const DenseRow<VT> X(P.X + (int64_t)col * P.ldx, k);
      const int delta = ALIGNED ? 0 : X.shift - shift;
      float acc[8] = {};
      for (int v = lane; v < count; v += 32 * Q) {
        Gather<VT, ALIGNED> x[Q];
        uint4 y[Q];
#pragma unroll
        for (int q = 0; q < Q; ++q)
          if (v + 32 * q < count) {
            x[q].load(X, v + 32 * q, delta);
            y[q] = __ldg(Y.piece + v + 32 * q);
          }
#pragma unroll
        for (int q = 0; q < Q; ++q) {
          const int p = v + 32 * q;
          if (p >= count) continue;
          float f[8], g[8];
          x[q].get(delta, f);
          unpack<VT>(y[q], g);
          if (p >= first_whole && p <= last_whole) {
#pragma unroll
            for (int z = 0; z < 8; ++z) acc[z] = fmaf(f[z], g[z], acc[z]);
          } else {
            const int lo = p == 0 ? shift : 0, hi = min(8, k + shift - p * 8);
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
    next.check(flag && r + step < P.m, P.err);
    s = next.s, e = next.e;
    first = e - s > mine ? (uint32_t)P.col[s + mine] : 0;
    next.fetch(r + 2 * step);
  }
}

}  // namespace pf
