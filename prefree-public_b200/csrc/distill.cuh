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

#include <type_traits>

#include "pf_common.cuh"

namespace pf {

template <typename VT, typename IT>
struct DistillParams {
  int64_t m, n, nnz;
  const IT *row_ptr;
  const IT *row_ptr0;  // the whole matrix's (its first entry starts col and val)
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

// A row's softmax statistics: largest value and sum of 2^(scale (v - m)) of the
// student (z) and of the teacher (t), and the sum of 2^(scale (t - tm)) (t - z).
// A sum of 0 means that nothing above -inf was met; NaN shows in the sums.
struct alignas(16) RowState {
  float zm, zs, tm, ts;
  double td;
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 2^(scale (a - b)), 0 for a = -inf, which b may be too
__device__ __forceinline__ float rescale(float a, float b, float scale) {
  return a == -INFINITY ? 0.0f : exp2_fast((a - b) * scale);
}
__device__ __forceinline__ float warp_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
template <typename T>
__device__ __forceinline__ T warp_sum(T v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
  return v;
}
__device__ __forceinline__ void warp_student(RowState &s, float scale) {
  const float m = warp_max(s.zm);
  s.zs = warp_sum(s.zm == -INFINITY ? s.zs : s.zs * rescale(s.zm, m, scale));
  s.zm = m;
}
template <bool DOT>
__device__ __forceinline__ void warp_teacher(RowState &s, float scale) {
  const float m = warp_max(s.tm);
  const float f = s.tm == -INFINITY ? 1.0f : rescale(s.tm, m, scale);
  s.ts = warp_sum(s.ts * f);
  // a factor of 0: the terms have p = 0 and add nothing, infinite or not
  if (DOT) s.td = warp_sum(f == 0.0f ? 0.0 : s.td * (double)f);
  s.tm = m;
}

template <typename VT>
__device__ __forceinline__ void unpack(const uint4 &r, float *x);
template <>
__device__ __forceinline__ void unpack<float>(const uint4 &r, float *x) {
  x[0] = __uint_as_float(r.x), x[1] = __uint_as_float(r.y);
  x[2] = __uint_as_float(r.z), x[3] = __uint_as_float(r.w);
}
template <>
__device__ __forceinline__ void unpack<__nv_bfloat16>(const uint4 &r, float *x) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
template <>
__device__ __forceinline__ void unpack<__half>(const uint4 &r, float *x) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
    x[2 * i] = f.x, x[2 * i + 1] = f.y;
  }
}
template <typename VT>
__device__ __forceinline__ uint4 pack(const float *x) {
  uint4 r;
  if constexpr (sizeof(VT) == 4) {
    r = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]),
                   __float_as_uint(x[3]));
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<VT, __half>::value) {
        const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t *>(&h);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t *>(&h);
      }
    }
    r = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return r;
}

// Elements that one thread holds of its row at a time.
constexpr int DISTILL_EPT = 32;

// One cluster of C = 1, 2, 4 or 8 CTAs per row; CTA `rank` takes the rank-th
// NT * 32 elements of it (LOOP: of every piece of C * NT * 32). A row is cut
// into the 16-byte pieces of memory that it lies in, so that every load is one
// of 16 bytes whatever the row's alignment; elements of neighbours in the first
// and the last piece are masked (and not written).
//
// Without LOOP the row's exponentials stay in registers between the statistics
// and the gradient: Z is read once, and each element costs one exponential.
// They are taken relative to the thread's own maximum, and one factor per
// thread turns them into q.
//
// The teacher's entries of a row are spread over the cluster's warps, 32 to a
// warp, for the statistics. For the gradient every warp looks through all of
// them for columns that its lanes hold; the lane concerned subtracts p in its
// register. Repeated columns are subtracted one by one in the entries' order.
template <typename VT, typename IT, int NT, bool GRAD, bool LOOP>
__global__ void __launch_bounds__(NT, 1024 / NT) distill_kernel(const DistillParams<VT, IT> P) {
  constexpr int NW = NT / 32, VE = 16 / (int)sizeof(VT), NV = DISTILL_EPT / VE;
  __shared__ RowState sh_warp[NW], sh_cta[8];
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  uint32_t rank, C;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(C));
  const int64_t r = blockIdx.x / C;
  const float scale = P.inv_tau * 1.4426950408889634f;

  const VT *z = P.Z + r * P.ldz;
  VT *dz = GRAD ? P.dZ + r * P.lddz : nullptr;
  const int shift = (int)(((uintptr_t)z & 15) / sizeof(VT));  // elements before the row
  const uint4 *zv = reinterpret_cast<const uint4 *>(z - shift);
  const int n = (int)P.n, nvec = (int)(((int64_t)n + shift + VE - 1) / VE);
  const bool same = ((uintptr_t)dz & 15) == ((uintptr_t)z & 15);  // dZ's pieces lie alike
  constexpr int PIECE = NT * NV;
  const int chunks = LOOP ? (nvec + (int)C * PIECE - 1) / ((int)C * PIECE) : 1;

  // `lo`, `hi`: the elements of piece v that belong to the row
  auto lo_of = [&](int v) { return v == 0 ? shift : 0; };
  auto hi_of = [&](int v) { return v == nvec - 1 ? n + shift - v * VE : VE; };
  auto store = [&](int v, const float *g) {
    const int lo = lo_of(v), hi = hi_of(v);
    if (same && lo == 0 && hi == VE) {
      __stcs(reinterpret_cast<uint4 *>(dz - shift) + v, pack<VT>(g));
    } else {
#pragma unroll
      for (int e = 0; e < VE; ++e)
        if (e >= lo && e < hi) dz[(int64_t)v * VE + e - shift] = from_f32<VT>(g[e]);
    }
  };
  auto zero_row = [&] {
    const float g[VE] = {};
    for (int v = (int)rank * NT + tid; v < nvec; v += (int)C * NT) store(v, g);
  };

  const float w = P.weight ? P.weight[r] : 1.0f;
  if (w == 0.0f) {  // the same for all of the cluster
    if (P.loss && rank == 0 && tid == 0) P.loss[r] = 0.0f;
    if (GRAD) zero_row();
    return;
  }

  // ---- this thread's elements: x, relative to their maximum as exponentials
  float x[NV][VE];
  auto load = [&](int v0) {  // raw values, -inf where there is none; their maximum
    uint4 raw[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int v = v0 + j * NT;
      // not a read-only load: dZ may be Z
      if (v < nvec)
        asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(raw[j].x), "=r"(raw[j].y), "=r"(raw[j].z), "=r"(raw[j].w)
                     : "l"(zv + v));
    }
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int v = v0 + j * NT;
      if (v < nvec) {
        unpack<VT>(raw[j], x[j]);
        const int lo = lo_of(v), hi = hi_of(v);
        if (lo != 0 || hi != VE) {
#pragma unroll
          for (int e = 0; e < VE; ++e)
            if (e < lo || e >= hi) x[j][e] = -INFINITY;
        }
      } else {
#pragma unroll
        for (int e = 0; e < VE; ++e) x[j][e] = -INFINITY;
      }
#pragma unroll
      for (int e = 0; e < VE; ++e) m = fmaxf(m, x[j][e]);
    }
    return m;
  };
  // x <- 2^(scale (x - m)); returns what one more factor 2^result corrects: the
  // rounding of scale * m, which all of x share
  auto exponentials = [&](float m) {
    const float ms = m * scale;
    if (fabsf(ms) <= 1e30f) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < VE; ++e) x[j][e] = exp2_fast(fmaf(x[j][e], scale, -ms));
      return -fmaf(m, scale, -ms);
    }
    // the type's lowest values, or infinities: no product may overflow
    const float b = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < VE; ++e) x[j][e] = exp2_fast((x[j][e] - b) * scale);
    return 0.0f;
  };
  auto total = [&] {
    float s[4] = {};
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < VE; ++e) s[e & 3] += x[j][e];
    return (s[0] + s[1]) + (s[2] + s[3]);
  };

  // the teacher's entries
  int64_t first = (int64_t)P.row_ptr[r], end = (int64_t)P.row_ptr[r + 1];
  {
    const int64_t base = (int64_t)*P.row_ptr0;
    if (first < base || end < first || end > base + P.nnz) {
      if (tid == 0 && rank == 0) atomicOr(P.err, PF_DEVERR_ROWPTR);
      first = end = 0;
    }
  }

  RowState st{-INFINITY, 0.0f, -INFINITY, 0.0f, 0.0};
  float own_m = -INFINITY, own_adjust = 0.0f;
  for (int c = 0; c < chunks; ++c) {
    const float m = load((c * (int)C + (int)rank) * PIECE + tid);
    const float adjust = exponentials(m);
    const float sum = total() * exp2_fast(adjust);
    if (!LOOP) {
      st.zm = own_m = m, st.zs = sum, own_adjust = adjust;
    } else {
      const float b = fmaxf(st.zm, m);
      st.zs = (st.zm == -INFINITY ? st.zs : st.zs * rescale(st.zm, b, scale)) +
              (m == -INFINITY ? sum : sum * rescale(m, b, scale));
      st.zm = b;
    }
  }

  // teacher statistics: 32 entries to a warp
  const int64_t stride = (int64_t)C * NT;
  const bool has_entries = first + ((int64_t)rank * NW + wid) * 32 < end;
  if (has_entries) {
    for (int64_t i = first + (int64_t)rank * NT + tid; i < end; i += stride) {
      const uint32_t c = (uint32_t)P.col[i];
      if (c >= (uint32_t)n) {
        atomicOr(P.err, PF_DEVERR_BOUNDS);
        continue;
      }
      const float t = to_f32(P.val[i]);
      if (t == -INFINITY) continue;
      const double d = (double)t - (double)to_f32(z[c]);
      const float b = fmaxf(st.tm, t);
      const float fo = st.tm == -INFINITY ? 1.0f : rescale(st.tm, b, scale);
      const float fn = t != t ? t : rescale(t, b, scale);
      st.ts = st.ts * fo + fn;
      st.td = (fo == 0.0f ? 0.0 : st.td * (double)fo) + (fn == 0.0f ? 0.0 : d * (double)fn);
      st.tm = b;
    }
    __syncwarp();
    warp_teacher<true>(st, scale);
  }
  warp_student(st, scale);
  if (lane == 0) sh_warp[wid] = st;
  __syncthreads();
  const RowState none{-INFINITY, 0.0f, -INFINITY, 0.0f, 0.0};
  if (C == 1) {
    st = lane < NW ? sh_warp[lane] : none;
  } else {
    if (wid == 0) {
      st = lane < NW ? sh_warp[lane] : none;
      warp_student(st, scale);
      warp_teacher<true>(st, scale);
      if (lane < (int)C) {  // to every CTA of the cluster
        uint32_t to;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
                     : "=r"(to)
                     : "r"((uint32_t)__cvta_generic_to_shared(&sh_cta[rank])), "r"(lane));
        asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to), "f"(st.zm),
                     "f"(st.zs), "f"(st.tm), "f"(st.ts)
                     : "memory");
        asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(to + 16), "d"(st.td) : "memory");
      }
      __syncwarp();
    }
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;"
                 ::: "memory");
    st = lane < (int)C ? sh_cta[lane] : none;
  }
  warp_student(st, scale);
  if (wid == 0) warp_teacher<true>(st, scale);
  else warp_teacher<false>(st, scale);
  const bool mass = !(st.ts == 0.0f);

  if (P.loss && rank == 0 && tid == 0) {
    double v = 0.0;
    if (mass && st.zs == 0.0f) v = (double)w * INFINITY;
    else if (mass)
      v = (double)w * ((st.td / (double)st.ts - (double)st.tm + (double)st.zm) *
                           (double)P.inv_tau + log((double)st.zs / (double)st.ts));
    P.loss[r] = (float)v;
  }
  if constexpr (GRAD) {
    if (!mass) {
      zero_row();
      return;
    }
    const float g = w * P.inv_tau;
    const float gz = st.zs == 0.0f ? 0.0f : g / st.zs, gt = g / st.ts;
    for (int c = 0; c < chunks; ++c) {
      const int v0 = (c * (int)C + (int)rank) * PIECE;
      if (LOOP) {
        own_m = load(v0 + tid);
        own_adjust = exponentials(own_m);
      }
      const float f = own_m == -INFINITY
                          ? gz
                          : gz * exp2_fast((own_m - st.zm) * scale + own_adjust);
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < VE; ++e) x[j][e] *= f;
      for (int64_t i0 = first; i0 < end; i0 += 32) {
        const int64_t i = i0 + lane;
        const uint32_t cc = i < end ? (uint32_t)P.col[i] : 0xffffffffu;
        const uint32_t at = cc + (uint32_t)shift;            // element, counted in pieces
        const uint32_t vv = at / VE - (uint32_t)v0;          // piece of this CTA
        const bool mine = cc < (uint32_t)n && vv < (uint32_t)PIECE && vv % NT / 32 == (uint32_t)wid;
        unsigned hits = __ballot_sync(~0u, mine);
        if (hits == 0) continue;
        float p = 0.0f;
        if (mine) {
          const float t = to_f32(P.val[i]);
          p = t != t ? t : gt * rescale(t, st.tm, scale);
        }
        const int slot = (int)(vv / NT * VE + at % VE);      // which of the lane's elements
        const int owner = (int)(vv % 32);
        while (hits) {
          const int k = __ffs(hits) - 1;
          hits &= hits - 1;
          const float pk = __shfl_sync(~0u, p, k);
          const int sk = __shfl_sync(~0u, slot, k), ok = __shfl_sync(~0u, owner, k);
          if (lane == ok) {
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
              for (int e = 0; e < VE; ++e)
                if (j * VE + e == sk) x[j][e] -= pk;
          }
        }
      }
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int v = v0 + j * NT + tid;
        if (v < nvec) store(v, x[j]);
      }
    }
  }
}

}  // namespace pf
