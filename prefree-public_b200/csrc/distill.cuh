// Distillation from a teacher's kept logits: per-row loss of dense student
// logits Z (m x n) against a CSR matrix of teacher logits, and its gradient.
//
// With temperature tau, row r's stored columns S, teacher logits t and student
// logits z:
//   p_j = exp(t_j / tau - Lt),  Lt = log sum_{j in S} exp(t_j / tau)
//   q_i = exp(z_i / tau - Lz),  Lz = log sum_{all i}  exp(z_i / tau)
//   loss = w * sum_{j in S} p_j (log p_j - log q_j)
//        = w * (sum_j p_j ((t_j - max t) + (max z - z_j)) / tau
//               - log sum_j exp((t_j - max t) / tau)
//               + log sum_i exp((z_i - max z) / tau))
// (in differences of the row's own values: what all of a row is moved by, a
// mask's -1e20 for one, leaves no rounding)
//   dZ_i = (w / tau) * (q_i - sum_{j in S, col_j = i} p_j)
// An entry with p_j = 0 adds nothing whatever z_j is. A row without teacher
// mass (no entry, or all of them -inf) and a row of weight 0 have loss 0 and
// gradient 0; the student's row of the latter is not read.
//
// What bounds it: the bytes of Z (and dZ); the exponentials, one an element for
// the loss and two with the gradient, at 16 a clock and SM, come next (60 % of
// that rate with bf16 and the gradient). Measured: 4096 x 131072 bf16 with the
// gradient 425-439 us (4.9 TB/s of Z and dZ, 75 % of the copy rate), 2048 x 128000
// fp32 358 us (89 %), 2048 x 65536 fp32 loss alone 85 us (95 %).
#pragma once

#include "pf_ptx.cuh"
#include "pf_values.cuh"

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

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 2^(scale (a - b)), 0 for a = -inf, which b may be too
__device__ __forceinline__ float rescale(float a, float b, float scale) {
  return a == -INFINITY ? 0.0f : exp2_fast((a - b) * scale);
}
// A running softmax: the largest value and the sum of 2^(scale (v - m)). A sum
// of 0 means that nothing above -inf was met; NaN and +inf show as NaN sums.
struct SoftmaxState {
  float m, s;
};
// what a state's sum is multiplied with when its maximum becomes b; an empty
// state's sum (0, or NaN alone) stays
__device__ __forceinline__ float state_factor(float m, float b, float scale) {
  return m == -INFINITY ? 1.0f : rescale(m, b, scale);
}
__device__ __forceinline__ SoftmaxState join(SoftmaxState a, SoftmaxState b, float scale) {
  const float m = fmaxf(a.m, b.m);
  return SoftmaxState{m, a.s * state_factor(a.m, m, scale) + b.s * state_factor(b.m, m, scale)};
}
__device__ __forceinline__ SoftmaxState warp_join(SoftmaxState a, float scale) {
  const float m = warp_max(a.m);
  return SoftmaxState{m, warp_sum(a.s * state_factor(a.m, m, scale))};
}

// One 8-byte value to the same place of CTA `rank`, counted on its barrier.
__device__ __forceinline__ void send8(const void *to, const void *bar, uint32_t rank, uint32_t a,
                                      uint32_t b) {
  uint32_t t, m;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(t) : "r"(ptx::smem_addr(to)), "r"(rank));
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(m) : "r"(ptx::smem_addr(bar)), "r"(rank));
  asm volatile(
      "st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.b32 [%0], {%1, %2}, [%3];" ::"r"(t),
      "r"(a), "r"(b), "r"(m)
      : "memory");
}

constexpr uint64_t DISTILL_WAIT_NS = 4000000000ull;
constexpr int DISTILL_MAX_C = 8;    // CTAs of a cluster
constexpr int DISTILL_LIST = 64;    // entries of a row that the teacher's warp lists
constexpr int DISTILL_RING = 16;    // rows whose barriers and results are kept apart
// What the entries of a lane or CTA add to the loss's sum: p times (t - max t) +
// (ref - z), ref the largest z met so far. A larger ref adds the sum of p times
// the difference, so that no term but the teacher's, which is small, is negative.
struct EntrySum {
  float v, p, ref;
};
__device__ __forceinline__ float raised(const EntrySum &s, float ref) {
  return s.p == 0.0f || ref == s.ref ? s.v : s.v + s.p * (ref - s.ref);
}
// p, t - max t and z of one entry
__device__ __forceinline__ float entry_term(float p, float t, float z, float ref) {
  return z == -INFINITY ? INFINITY : p * (t + (ref - z));
}
// the warp's sums of a (in lane 0) and b (in lane 16)
__device__ __forceinline__ float warp_sum2(float a, float b) {
  const bool low = (threadIdx.x & 16) == 0;
  float v = (low ? a : b) + __shfl_xor_sync(~0u, low ? b : a, 16);
#pragma unroll
  for (int d = 8; d > 0; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
  return v;
}

// 2^(scale (x - m)) is taken as 2^(scale x - ms), ms = scale m rounded, and one
// more factor corrects that rounding, which a whole sum shares: a power within
// 1/2 of 0 as long as |ms| is at most 2^24. (From 2^31 on the power leaves fp32's
// range: inf * 0.) Above, the difference is taken first.
constexpr float DISTILL_FOLDED = 16777216.0f;

template <typename VT, int NT>
struct DistillCfg {
  static constexpr int VE = 16 / (int)sizeof(VT);  // elements of a 16-byte piece
  static constexpr int NV = 8;                     // pieces that a thread holds
  static constexpr int PIECE = NT * NV;            // pieces of a slot
  static constexpr int NW = NT / 32;
  static constexpr int STAGES = 3;
  // per SM (64 threads: 6 instead of 4 took 15-20 % off vocabularies up to 4000)
  static constexpr int CTAS = NT >= 256 ? 2 : NT >= 128 ? 4 : 6;
  static constexpr int SMEM = STAGES * PIECE * 16;
};

// A row cut into pieces of 16 bytes of memory: its element 0 is element `shift`
// of piece 0, and it lies in nvec pieces.
struct RowCut {
  int n, shift, nvec;
  template <int VE>
  __device__ __forceinline__ int lo(int v) const { return v == 0 ? shift : 0; }
  template <int VE>
  __device__ __forceinline__ int hi(int v) const {
    return v == nvec - 1 ? n + shift - v * VE : VE;
  }
};
// piece v of the gradient: whole where the piece is all the row's and dZ's
// pieces lie as Z's do (`same`), else by elements
template <typename VT>
__device__ __forceinline__ void store_piece(const RowCut &R, VT *dz, bool same, int v,
                                            const float *g) {
  constexpr int VE = 16 / (int)sizeof(VT);
  const int lo = R.lo<VE>(v), hi = R.hi<VE>(v);
  if (same && lo == 0 && hi == VE) {
    __stcs(reinterpret_cast<uint4 *>(dz - R.shift) + v, pack<VT>(g));
  } else {
#pragma unroll
    for (int e = 0; e < VE; ++e)
      if (e >= lo && e < hi) dz[(int64_t)v * VE + e - R.shift] = from_f32<VT>(g[e]);
  }
}

// Subtracts p from the values x of this lane's piece (piece `piece0` of the row
// is lane 0's), for rows of many entries: the warp looks through all of them.
// Seldom called, so small rather than fast.
template <typename VT, typename IT>
__device__ __forceinline__ void subtract_many(const DistillParams<VT, IT> &P, const RowCut &R,
                                              int piece0, float scale, float2 told, int64_t first,
                                              int64_t end, float *x) {
  constexpr int VE = 16 / (int)sizeof(VT);
  const int lane = threadIdx.x & 31;
#pragma unroll 1
  for (int64_t i0 = first; i0 < end; i0 += 32) {
    const uint32_t cc = i0 + lane < end ? (uint32_t)P.col[i0 + lane] : 0xffffffffu;
    const uint32_t at = cc + (uint32_t)R.shift - (uint32_t)piece0 * VE;  // element of the warp's
    const bool here = cc < (uint32_t)R.n && at < 32 * VE;
    unsigned hits = __ballot_sync(~0u, here);
    if (hits == 0) continue;
    float p = 0.0f;
    if (here) {
      const float t = to_f32(P.val[i0 + lane]);
      p = t != t ? t : told.y * rescale(t, told.x, scale);
    }
#pragma unroll 1
    while (hits) {
      const int k = __ffs(hits) - 1;
      hits &= hits - 1;
      const float pk = __shfl_sync(~0u, p, k);
      const uint32_t ak = __shfl_sync(~0u, at, k);
#pragma unroll
      for (int e = 0; e < VE; ++e)
        if ((uint32_t)(lane * VE + e) == ak) x[e] -= pk;
    }
  }
}

// Persistent clusters of C = 1, 2, 4 or 8 CTAs; a cluster takes every
// (clusters)-th row, the CTAs a slice of NT * 8 pieces of 16 bytes each (and
// of every further C * NT * 8 pieces of a longer row). A row is cut into the
// 16-byte pieces of memory that it lies in, so that every access is aligned
// whatever the row's alignment; elements of neighbours in the first and the
// last piece are masked, and not written.
//
// A warp of its own keeps bulk copies of the next slices on their way into
// shared memory. The gradient takes the exponentials a second time, from the
// slot where the row fits one, else from a second copy, which comes out of L2:
// the rows in hand on the whole GPU are kept well below its size. (Keeping a
// row's values or exponentials in registers in between cost spills or resident
// warps, and 2 to 3 times the time.)
//
// NT threads deal with the student alone and store weight / tau * q. Each warp
// sends its part of the row's statistics to every CTA of the cluster (st.async,
// counted on a barrier there), and each warp joins all parts, in the same
// order: no barrier of the whole CTA or cluster in the loop. The parts of two
// rows have places of their own, which is enough: a warp sends its part of row
// i + 2 after it has joined row i + 1, to which every reader of row i has sent.
//
// A second warp of its own deals with the teacher: the softmax of the row's
// entries, the loss's sum over those of the CTA's slice (whose z is in
// shared memory), and, one row behind, the loss and the gradient q - p at the
// entries' columns, written over what the others stored. Nothing in the common
// case waits for it but the release of the slots, which also keeps it within
// STAGES + 2 rows of the others: the DISTILL_RING rows kept apart are enough.
// Of rows of more than DISTILL_LIST entries the others wait to be told the
// teacher's statistics; they look through the entries for columns that they hold
// and subtract p (subtract_many). Repeated columns add up in the entries' order.
template <typename VT, typename IT, int NT, bool GRAD>
__global__ void __launch_bounds__(NT + 64, DistillCfg<VT, NT>::CTAS)
distill_kernel(const DistillParams<VT, IT> P) {
  using Cfg = DistillCfg<VT, NT>;
  constexpr int VE = Cfg::VE, NV = Cfg::NV, PIECE = Cfg::PIECE, NW = Cfg::NW;
  constexpr int STAGES = Cfg::STAGES;
  extern __shared__ __align__(128) uint8_t slots[];
  __shared__ SoftmaxState parts[2][DISTILL_MAX_C * NW];
  __shared__ SoftmaxState student[DISTILL_RING];  // a row's joined statistics
  __shared__ float2 told_as[DISTILL_RING];        // tm; weight / tau / sum of exponentials
  __shared__ float2 dots[DISTILL_RING][DISTILL_MAX_C][2];  // v and ref; p
  __shared__ uint32_t seen[GRAD ? 512 : 1];  // the teacher's warp's: columns met
  __shared__ uint64_t full[STAGES], empty[STAGES], joined[2];
  __shared__ uint64_t told[DISTILL_RING], heard[DISTILL_RING], dotted[DISTILL_RING];
  __shared__ volatile int dead;
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  uint32_t rank, C, cluster, clusters;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(C));
  asm volatile("mov.u32 %0, %%clusterid.x;" : "=r"(cluster));
  asm volatile("mov.u32 %0, %%nclusterid.x;" : "=r"(clusters));
  const float scale = P.inv_tau * 1.4426950408889634f;
  const int n = (int)P.n;

  if (tid == 0) {
    dead = 0;
    for (int s = 0; s < STAGES; ++s) {
      ptx::mbar_init(&full[s], 1);
      ptx::mbar_init(&empty[s], NW + 1);
    }
    ptx::mbar_init(&joined[0], 1);
    ptx::mbar_init(&joined[1], 1);
    for (int s = 0; s < DISTILL_RING; ++s) {
      ptx::mbar_init(&told[s], 1);
      ptx::mbar_init(&heard[s], GRAD ? NW : 1);
      ptx::mbar_init(&dotted[s], 1);
    }
    ptx::fence_mbar_init();
  }
  __syncthreads();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;"
               ::: "memory");

  // called by whole warps
  auto wait = [&](uint64_t *bar, uint32_t parity) -> bool {
    if (__all_sync(~0u, ptx::mbar_wait_bounded(bar, parity, DISTILL_WAIT_NS))) return true;
    atomicOr(P.err, PF_DEVERR_WAIT_TIMEOUT);
    dead = 1;
    return false;
  };
  // a row's pieces: elements of memory before the row in its first piece, pieces
  auto shift_of = [&](int64_t r) {
    return (int)(((uintptr_t)(P.Z + r * P.ldz) & 15) / sizeof(VT));
  };
  auto pieces_of = [&](int shift) { return (int)(((int64_t)n + shift + VE - 1) / VE); };
  auto chunks_of = [&](int nvec) { return (nvec + (int)C * PIECE - 1) / ((int)C * PIECE); };

  bool ok = true;
  uint32_t it = 0;       // slots used so far
  uint32_t rows_in = 0;  // rows (of weight other than 0) begun so far
  if (wid == NW) {  // ---- copies
    // what is copied twice is to stay in L2 until then
    const uint64_t keep = ptx::policy_evict_last(), once = ptx::policy_evict_first();
    for (int64_t r = cluster; ok && r < P.m; r += clusters) {
      if (P.weight && P.weight[r] == 0.0f) continue;
      const int shift = shift_of(r), nvec = pieces_of(shift), chunks = chunks_of(nvec);
      const uint4 *from = reinterpret_cast<const uint4 *>(P.Z + r * P.ldz - shift);
      const int items = GRAD && chunks > 1 ? 2 * chunks : chunks;
      for (int k = 0; k < items; ++k, ++it) {
        const uint32_t s = it % STAGES;
        if (!wait(&empty[s], (it / STAGES & 1) ^ 1)) {
          ok = false;
          break;
        }
        if (lane == 0) {
          const int v0 = ((k < chunks ? k : k - chunks) * (int)C + (int)rank) * PIECE;
          const int count = max(0, min(PIECE, nvec - v0));
          if (count > 0) {
            ptx::mbar_arrive_expect_tx(&full[s], (uint32_t)count * 16);
            for (int x = 0; x < count; x += 1024)
              ptx::bulk_g2s(slots + ((size_t)s * PIECE + x) * 16, from + v0 + x,
                            (uint32_t)min(1024, count - x) * 16, &full[s],
                            GRAD && k + chunks < items ? keep : once);
          } else {
            ptx::mbar_arrive(&full[s]);
          }
        }
        __syncwarp();
      }
    }
  } else if (wid == NW + 1) {  // ---- the teacher and the loss
    constexpr int U = DISTILL_LIST / 32;  // entries that a lane fetches ahead
    const int64_t entry0 = (int64_t)*P.row_ptr0;
    // the rows' bounds two ahead, the entries one ahead: no load is waited for
    int64_t far_s = 0, far_e = 0, near_s = 0, near_e = 0;
    uint32_t near_c[U];
    float near_t[U], near_w = 1.0f, far_w = 1.0f;
    auto fetch_bounds = [&](int64_t r) {
      if (r < P.m) {
        far_s = (int64_t)P.row_ptr[r];
        far_e = (int64_t)P.row_ptr[r + 1];
        if (P.weight) far_w = P.weight[r];
      }
    };
    auto fetch_entries = [&] {  // of the row whose bounds were fetched last
      near_s = far_s, near_e = far_e, near_w = far_w;
      if (near_s < entry0 || near_e < near_s || near_e > entry0 + P.nnz) {
        if (lane == 0 && rank == 0) atomicOr(P.err, PF_DEVERR_ROWPTR);
        near_s = near_e = 0;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t i = near_s + u * 32 + lane;
        near_c[u] = 0xffffffffu;
        near_t[u] = -INFINITY;
        if (i < near_e) {
          near_c[u] = (uint32_t)P.col[i];
          near_t[u] = to_f32(P.val[i]);
        }
      }
    };
    fetch_bounds(cluster);
    fetch_entries();
    fetch_bounds((int64_t)cluster + clusters);
    if (GRAD) {
      for (int k = lane; k < 512; k += 32) seen[k] = 0;
      __syncwarp();
    }
    // the row behind, still to be finished: its entries (p: weight / tau * p)
    struct Row {
      int64_t r;
      SoftmaxState a;
      float w;
      int pieces;
      uint32_t index;
      bool repeats;  // a column may occur twice
      uint32_t c[U]; // 0xffffffff: not in this CTA's slices, or p = 0
      float p[U], z[U];
    } last;
    // one row's terms of the loss in each lane, finished 32 rows at a time: the
    // closing arithmetic is in double
    struct {
      int64_t r = -1;
      float w, d, as, qs;
    } term;
    int terms = 0;
    auto flush_terms = [&] {
      if (term.r >= 0) {
        double v = 0.0;
        if (term.as != 0.0f && term.qs == 0.0f) v = (double)term.w * INFINITY;
        else if (term.as != 0.0f)
          v = (double)term.w *
              ((double)term.d * (double)P.inv_tau +
               log((double)term.qs / (double)term.as));
        P.loss[term.r] = (float)v;
      }
      term.r = -1;
      terms = 0;
    };
    auto finish = [&]() -> bool {
      const uint32_t ring = last.index % DISTILL_RING, phase = last.index / DISTILL_RING & 1;
      const bool mass = !(last.a.s == 0.0f), lossy = rank == 0 && P.loss;
      if (!GRAD && !lossy) return true;
      // after the others' stores, which these take the place of
      if (!wait(&heard[ring], phase)) return false;
      const SoftmaxState q = student[ring];
      if constexpr (GRAD) {
        const int64_t r = last.r;
        VT *dz = P.dZ + r * P.lddz;
        if (!mass) {
          for (int v0 = (int)rank * PIECE; v0 < last.pieces; v0 += (int)C * PIECE) {
            const int64_t lo = max((int64_t)0, (int64_t)v0 * VE - shift_of(r));
            const int64_t hi = min((int64_t)n, (int64_t)(v0 + PIECE) * VE - shift_of(r));
            for (int64_t c = lo + lane; c < hi; c += 32) dz[c] = from_f32<VT>(0.0f);
          }
        } else {
          const float gz = q.s == 0.0f ? 0.0f : last.w * P.inv_tau / q.s;
          if (last.repeats) {  // each one's p becomes the sum over its column's
            float total[U] = {};
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll 1
              for (int k = 0; k < 32; ++k) {
                const uint32_t c = __shfl_sync(~0u, last.c[u], k);
                const float p = __shfl_sync(~0u, last.p[u], k);
#pragma unroll
                for (int o = 0; o < U; ++o) total[o] += last.c[o] == c ? p : 0.0f;
              }
#pragma unroll
            for (int u = 0; u < U; ++u) last.p[u] = total[u];
          }
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (last.c[u] != 0xffffffffu) {
              const float zc = last.z[u];
              const float g = zc != zc ? zc : gz * rescale(zc, q.m, scale) - last.p[u];
              dz[last.c[u]] = from_f32<VT>(g);
            }
        }
        __syncwarp();
      }
      if (lossy) {
        if (!wait(&dotted[ring], phase)) return false;
        float d = 0.0f;
        for (int k = 0; k < (int)C; ++k) {
          const float2 v = dots[ring][k][0];
          d += raised(EntrySum{v.x, dots[ring][k][1].x, v.y}, q.m);
        }
        if (lane == terms) {
          term.r = last.r;
          term.w = last.w;
          term.d = d;
          term.as = last.a.s;
          term.qs = q.s;
        }
        if (++terms == 32) flush_terms();
      }
      return true;
    };
    for (int64_t r = cluster; ok && r < P.m; r += clusters) {
      const int64_t first = near_s, end = near_e;
      const float w = near_w;
      uint32_t c_[U];
      float t_[U], p_[U];
#pragma unroll
      for (int u = 0; u < U; ++u) c_[u] = near_c[u], t_[u] = near_t[u];
      fetch_entries();
      fetch_bounds(r + 2 * (int64_t)clusters);
      if (w == 0.0f) continue;
      const int shift = shift_of(r), nvec = pieces_of(shift), chunks = chunks_of(nvec);
      const uint32_t ring = rows_in % DISTILL_RING;
      const bool listing = GRAD && end - first <= DISTILL_LIST;
      // the softmax over the entries with a valid column (the others count as -inf)
      SoftmaxState a{-INFINITY, 0.0f};
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (c_[u] >= (uint32_t)n) {
          if (first + u * 32 + lane < end && rank == 0) atomicOr(P.err, PF_DEVERR_BOUNDS);
          t_[u] = -INFINITY;
        }
        a.m = fmaxf(a.m, t_[u]);
      }
      // an entry after the fetched ones
      auto entry = [&](int64_t i, uint32_t *c, float *t) {
        *c = (uint32_t)P.col[i];
        *t = *c < (uint32_t)n ? to_f32(P.val[i]) : -INFINITY;
      };
      for (int64_t i = first + DISTILL_LIST + lane; i < end; i += 32) {
        uint32_t c;
        float t;
        entry(i, &c, &t);
        if (c >= (uint32_t)n && rank == 0) atomicOr(P.err, PF_DEVERR_BOUNDS);
        a.m = fmaxf(a.m, t);
      }
      a.m = warp_max(a.m);
      auto power = [&](float t) { return t != t ? t : rescale(t, a.m, scale); };
#pragma unroll
      for (int u = 0; u < U; ++u) a.s += p_[u] = power(t_[u]);
      for (int64_t i = first + DISTILL_LIST + lane; i < end; i += 32) {
        uint32_t c;
        float t;
        entry(i, &c, &t);
        a.s += power(t);
      }
      a.s = warp_sum(a.s);
      const float gt = w * P.inv_tau / a.s;  // not used without mass
      if (GRAD) {  // for every row: the barrier's phase counts them
        if (lane == 0) {
          told_as[ring] = make_float2(a.m, a.s == 0.0f ? 0.0f : gt);
          ptx::mbar_arrive(&told[ring]);
        }
        __syncwarp();
      }

      // the sum over the entries of this CTA's slices. p = 0 adds nothing, infinite
      // or not.
      const float one = 1.0f / a.s;
      EntrySum sum{0.0f, 0.0f, -INFINITY};
      float z_[U];
      bool own[U] = {};
      for (int c = 0; c < chunks; ++c, ++it) {
        const uint32_t s = it % STAGES;
        if (!wait(&full[s], it / STAGES & 1)) {
          ok = false;
          break;
        }
        const VT *slot = reinterpret_cast<const VT *>(slots + (size_t)s * PIECE * 16);
        const uint32_t v0 = (uint32_t)(c * (int)C + (int)rank) * PIECE;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const uint32_t at = c_[u] + (uint32_t)shift, vv = at / VE - v0;
          if (t_[u] != -INFINITY && vv < (uint32_t)PIECE) {
            z_[u] = to_f32(slot[vv * VE + at % VE]);
            own[u] = true;
          }
        }
        if (P.loss && end - first > DISTILL_LIST)
          for (int64_t i = first + DISTILL_LIST + lane; i < end; i += 32) {
            uint32_t cc;
            float t;
            entry(i, &cc, &t);
            const uint32_t at = cc + (uint32_t)shift, vv = at / VE - v0;
            const float p = power(t) * one;
            if (t != -INFINITY && vv < (uint32_t)PIECE && p != 0.0f) {
              const float z = to_f32(slot[vv * VE + at % VE]), ref = fmaxf(sum.ref, z);
              sum = EntrySum{raised(sum, ref) + entry_term(p, t - a.m, z, ref), sum.p + p, ref};
            }
          }
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&empty[s]);
      }
      if (GRAD && chunks > 1)  // the gradient's slots are not looked at here
        for (int c = 0; ok && c < chunks; ++c, ++it) {
          // (an arrival before the slot's turn would count for the turn before)
          ok = wait(&full[it % STAGES], it / STAGES & 1);
          if (ok && lane == 0) ptx::mbar_arrive(&empty[it % STAGES]);
        }
      if (!ok) break;
      if (P.loss) {
        float ref = sum.ref;
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (own[u] && p_[u] * one != 0.0f) ref = fmaxf(ref, z_[u]);
        ref = warp_max(ref);
        float v = raised(sum, ref);
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (own[u] && p_[u] * one != 0.0f) {
            v += entry_term(p_[u] * one, t_[u] - a.m, z_[u], ref);
            sum.p += p_[u] * one;
          }
        v = warp_sum2(v, sum.p);
        if (rank == 0 && lane == 0) ptx::mbar_arrive_expect_tx(&dotted[ring], C * 16);
        if (lane % 16 == 0)
          send8(&dots[ring][rank][lane / 16], &dotted[ring], 0, __float_as_uint(v),
                __float_as_uint(ref));
        __syncwarp();
      }
      if (rows_in > 0) ok = finish();
      if (!ok) break;
      last.r = r;
      last.a = a;
      last.w = w;
      last.pieces = nvec;
      last.index = rows_in;
      last.repeats = false;
      if (GRAD) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const bool mine = listing && own[u];
          last.c[u] = mine ? c_[u] : 0xffffffffu;
          last.p[u] = gt * p_[u];
          last.z[u] = z_[u];
          // columns by their last 14 bits: two that agree there may be equal
          const uint32_t bit = 1u << (c_[u] & 31);
          if (mine) last.repeats |= (atomicOr(&seen[c_[u] / 32 % 512], bit) & bit) != 0;
        }
        last.repeats = __any_sync(~0u, last.repeats);
        __syncwarp();
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (last.c[u] != 0xffffffffu) seen[c_[u] / 32 % 512] = 0;
        __syncwarp();
      }
      ++rows_in;
    }
    if (ok && rows_in > 0) ok = finish();
    if (P.loss) flush_terms();
  } else {  // ---- statistics and gradient
    // joins the parts of the row that was begun as number `index`; warp 0 leaves
    // the result to the teacher's warp
    auto join_row = [&](uint32_t index, SoftmaxState *o) -> bool {
      const uint32_t side = index & 1;
      if (!wait(&joined[side], index >> 1 & 1)) return false;
      SoftmaxState q{-INFINITY, 0.0f};
      for (int k = lane; k < (int)C * NW; k += 32) q = join(q, parts[side][k], scale);
      *o = q = warp_join(q, scale);
      if (wid == 0 && lane == 0) student[index % DISTILL_RING] = q;
      return true;
    };
    // the next row's weight and bounds are fetched while a row is worked on
    float next_w = 1.0f;
    int64_t next_s = 0, next_e = 0;
    auto fetch = [&](int64_t r) {
      if (r >= P.m) return;
      if (P.weight) next_w = P.weight[r];
      if (GRAD) {
        next_s = (int64_t)P.row_ptr[r];
        next_e = (int64_t)P.row_ptr[r + 1];
      }
    };
    const int64_t entry0 = GRAD ? (int64_t)*P.row_ptr0 : 0;
    fetch(cluster);
    for (int64_t r = cluster; ok && r < P.m; r += clusters) {
      const float w = next_w;
      int64_t first = next_s, end = next_e;
      fetch(r + clusters);
      const VT *z = P.Z + r * P.ldz;
      VT *dz = GRAD ? P.dZ + r * P.lddz : nullptr;
      const int shift = shift_of(r), nvec = pieces_of(shift), chunks = chunks_of(nvec);
      const bool same = ((uintptr_t)dz & 15) == ((uintptr_t)z & 15);  // dZ's pieces lie alike
      const RowCut R{n, shift, nvec};
      if (w == 0.0f) {  // the same for all of the cluster
        if (P.loss && rank == 0 && tid == 0) P.loss[r] = 0.0f;
        if (GRAD) {
          const float g[VE] = {};
#pragma unroll 1
          for (int v = (int)rank * NT + tid; v < nvec; v += (int)C * NT)
            store_piece<VT>(R, dz, same, v, g);
        }
        continue;
      }
      if (GRAD && (first < entry0 || end < first || end > entry0 + P.nnz)) first = end = 0;
      const bool many = GRAD && end - first > DISTILL_LIST;
      const uint32_t index = rows_in++, side = index & 1, ring = index % DISTILL_RING;

      // body(j, v, cut) for this thread's pieces v = v0 + j NT + tid of the row; cut:
      // not all of the piece is the row's. The common case, all pieces of the
      // warp there and whole, is unrolled.
      const int whole0 = shift > 0 ? 1 : 0, whole1 = nvec - ((n + shift) % VE != 0 ? 1 : 0);
      auto pieces = [&](int v0, auto &&body) {
        const int base = v0 + wid * 32;
        if (base >= whole0 && base + (NV - 1) * NT + 32 <= whole1) {
#pragma unroll
          for (int j = 0; j < NV; ++j) body(j, base + j * NT + lane, false);
        } else {
#pragma unroll 1
          for (int j = 0; j < NV; ++j) {
            const int v = base + j * NT + lane;
            if (v < nvec) body(j, v, v < whole0 || v >= whole1);
          }
        }
      };
      // the values of piece v, -inf in place of neighbours
      auto values = [&](const uint4 &raw, int v, bool cut, float *x) {
        unpack<VT>(raw, x);
        if (cut) {
          const int lo = R.lo<VE>(v), hi = R.hi<VE>(v);
#pragma unroll
          for (int e = 0; e < VE; ++e)
            if (e < lo || e >= hi) x[e] = -INFINITY;
        }
      };
      SoftmaxState st{-INFINITY, 0.0f};  // of this thread
      for (int c = 0; c < chunks; ++c, ++it) {
        const uint32_t s = it % STAGES;
        if (!wait(&full[s], it / STAGES & 1)) {
          ok = false;
          break;
        }
        const uint4 *slot = reinterpret_cast<const uint4 *>(slots) + (size_t)s * PIECE + tid;
        const int v0 = (c * (int)C + (int)rank) * PIECE;
        float m = st.m, sum[4] = {};
        pieces(v0, [&](int j, int v, bool cut) {
          float x[VE];
          values(slot[j * NT], v, cut, x);
#pragma unroll
          for (int e = 0; e < VE; ++e) m = fmaxf(m, x[e]);
        });
        const float ms = m * scale;
        if (fabsf(ms) <= DISTILL_FOLDED) {
          pieces(v0, [&](int j, int v, bool cut) {
            float x[VE];
            values(slot[j * NT], v, cut, x);
#pragma unroll
            for (int e = 0; e < VE; ++e) sum[e & 3] += exp2_fast(fmaf(x[e], scale, -ms));
          });
          sum[0] = ((sum[0] + sum[1]) + (sum[2] + sum[3])) * exp2_fast(-fmaf(m, scale, -ms));
        } else {
          // masks (finite ones of any size too) and infinities
          const float b = m == -INFINITY ? 0.0f : m;
#pragma unroll 1
          for (int j = 0; j < NV; ++j) {
            const int v = v0 + j * NT + tid;
            if (v >= nvec) break;
            float x[VE];
            values(slot[j * NT], v, v < whole0 || v >= whole1, x);
#pragma unroll
            for (int e = 0; e < VE; ++e) sum[0] += exp2_fast((x[e] - b) * scale);
          }
        }
        if (!GRAD || chunks > 1) {  // the slot has been read
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(&empty[s]);
        }
        st.s = st.s * state_factor(st.m, m, scale) + sum[0];
        st.m = m;
      }
      if (!ok) break;
      st = warp_join(st, scale);

      // ---- this warp's part to every CTA, after the last row was joined
      if (!GRAD && index > 0) {
        SoftmaxState before;
        if (!join_row(index - 1, &before)) break;
        if (wid == 0 && lane == 0) ptx::mbar_arrive(&heard[(index - 1) % DISTILL_RING]);
      }
      if (tid == 0) ptx::mbar_arrive_expect_tx(&joined[side], C * NW * 8);
      if (lane < (int)C)
        send8(&parts[side][rank * NW + wid], &joined[side], lane, __float_as_uint(st.m),
              __float_as_uint(st.s));
      __syncwarp();

      if constexpr (GRAD) {
        if (!join_row(index, &st)) break;
        const float gz = st.s == 0.0f ? 0.0f : w * P.inv_tau / st.s;
        const float ms = st.m * scale;
        const float f = sizeof(VT) == 4 ? gz : gz * exp2_fast(-fmaf(st.m, scale, -ms));
        if (many && !wait(&told[ring], index / DISTILL_RING & 1)) break;
        for (int c = 0; c < chunks; ++c) {
          uint32_t s = (it - 1) % STAGES;  // one chunk: the slot is still held
          if (chunks > 1) {
            s = it % STAGES;
            if (!wait(&full[s], it / STAGES & 1)) {
              ok = false;
              break;
            }
            ++it;
          }
          const uint4 *slot = reinterpret_cast<const uint4 *>(slots) + (size_t)s * PIECE;
          const int v0 = (c * (int)C + (int)rank) * PIECE;
          if (!many && fabsf(ms) <= DISTILL_FOLDED && same) {
            uint4 *to = reinterpret_cast<uint4 *>(dz - shift);
            pieces(v0, [&](int j, int v, bool cut) {
              float x[VE];
              unpack<VT>(slot[j * NT + tid], x);
#pragma unroll
              for (int e = 0; e < VE; ++e)
                // fp32 results: the difference first, which rounds less
                x[e] = f * (sizeof(VT) == 4 ? exp2_fast((x[e] - st.m) * scale)
                                            : exp2_fast(fmaf(x[e], scale, -ms)));
              if (cut) store_piece<VT>(R, dz, same, v, x);
              else __stcs(to + v, pack<VT>(x));
            });
          } else {
            const float b = st.m == -INFINITY ? 0.0f : st.m;
#pragma unroll 1
            for (int j = 0; j < NV; ++j) {
              const int v = v0 + j * NT + tid;
              if (v - lane >= nvec) break;
              float x[VE];
              unpack<VT>(slot[j * NT + tid], x);
#pragma unroll
              for (int e = 0; e < VE; ++e) x[e] = gz * exp2_fast((x[e] - b) * scale);
              if (many) subtract_many<VT>(P, R, v - lane, scale, told_as[ring], first, end, x);
              if (v < nvec) store_piece<VT>(R, dz, same, v, x);
            }
          }
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(&empty[s]);
        }
        if (!ok) break;
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&heard[ring]);
      }
    }
    if (!GRAD && ok && rows_in > 0) {
      SoftmaxState before;
      if (join_row(rows_in - 1, &before) && wid == 0 && lane == 0)
        ptx::mbar_arrive(&heard[(rows_in - 1) % DISTILL_RING]);
    }
  }
  __syncwarp();
  __syncthreads();
  if (dead && tid == 0) {  // copies may still be on their way into this CTA
    for (int s = 0; s < STAGES; ++s) ptx::mbar_drain(&full[s], 50000000ull);
  }
  __syncthreads();
  // no CTA ends while another one may still send to it
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;"
               ::: "memory");
}

}  // namespace pf
