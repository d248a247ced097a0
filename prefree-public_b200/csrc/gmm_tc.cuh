// The grouped products on the tensor cores (tcgen05, TMA, tensor memory).
//
// Every direction is C[j, i] = alpha * sum_p A[i, p] B[j, p] + beta * C[j, i]
// with the ragged dimension away from the matrix instruction's M:
//   FWD  i = W's rows (n),    j = the group's rows, p = k    W, X: p contiguous
//   DX   i = W's columns (n), j = the group's rows, p = k    W: i contiguous
//   DW   i = X's columns (k), j = dY's columns (n), p = the group's rows,
//        both with p the slow dimension
// The instruction's N takes any multiple of 16, so a group's last tile of j
// costs what its rows need, where rows on M would cost 128 (a decoding step's
// one or two rows would waste 98 % of the tensor time and load 128 rows).
//
// One persistent CTA (CG = 1, 128 x BN tiles) or CTA pair (CG = 2, 256 x BN,
// each CTA loads half of A and half of B) per SM, in roles: warp 0 copies
// tiles of 64 along p with TMA into a ring of stages, warp 1 of the (leading)
// CTA issues the matrix instructions, warps 2-5 move the finished accumulator
// from tensor memory to C while the next tile is computed into the other half.
// Tiles are found on the device from group_ptr (GroupWalk), by each role for
// itself.
//
// DW: rows past a group's end belong to the next group and must not meet the
// sum (0 * NaN is NaN). The group's last block is copied in boxes of 8 rows
// and single rows, and filled up to a multiple of 16 by boxes that lie wholly
// outside of the array, which TMA fills with zeros.
#pragma once

#include "gmm_common.cuh"
#include "tc_ptx.cuh"

namespace pf {

enum GmmMode { GMM_FWD = 0, GMM_DX = 1, GMM_DW = 2 };

struct GmmMaps {
  CUtensorMap a, b;       // boxes of 64 along p (DW: 64 rows)
  CUtensorMap a8, b8;     // DW: boxes of 8 rows
  CUtensorMap a1, b1;     // DW: single rows
};

template <typename IT, typename OT>
struct GmmTcParams {
  int64_t groups, rows;
  int ni, nj, np;          // extents of i, j (DW), p (FWD, DX)
  int group_step;          // 1, or 0 where one W serves all groups
  const IT *ptr;
  OT *C;
  int64_t ldc, stride_c;
  float alpha, beta;
  unsigned *err;
};

template <int MODE, int CG, int BN>
struct GmmCfg {
  static constexpr int TI = 128 * CG;           // i of a tile
  static constexpr int BH = BN / CG;            // B rows that one CTA loads
  static constexpr int BOX = BH < 32 ? BH : 32; // rows of one B box (FWD, DX)
  static constexpr int A_BYTES = 128 * 128;
  static constexpr int B_BYTES = BH * 128;
  static constexpr int STAGE = A_BYTES + B_BYTES;
  static constexpr int STAGES = 200 * 1024 / STAGE > 10 ? 10 : 200 * 1024 / STAGE;
  static constexpr int COLS = 2 * BN < 32 ? 32 : 2 * BN;  // tensor memory columns
  static constexpr int NT = 192;
  static constexpr int SMEM = STAGES * STAGE + 1024;      // and alignment
};

constexpr uint64_t GMM_WAIT_NS = 4000000000ull;

// One tile: where it lies and how long its sum is.
struct GmmTile {
  int64_t g;
  int i0;          // first i of the CTA (pair)
  int64_t j0;      // first j: an absolute row (FWD, DX) or a column of dY (DW)
  int jn;          // number of j
  int64_t p0;      // DW: first row of the group
  int np;          // length of the sum
};

template <int MODE, int CG, int BN, typename IT, typename OT>
struct GmmTiles {
  using Cfg = GmmCfg<MODE, CG, BN>;
  const GmmTcParams<IT, OT> &P;
  GroupWalk<IT> walk;
  int ti, tj;
  int64_t t, step;

  __device__ GmmTiles(const GmmTcParams<IT, OT> &p)
      : P(p), walk{p.ptr, p.groups, p.rows, p.err}, ti((p.ni + Cfg::TI - 1) / Cfg::TI),
        tj(MODE == GMM_DW ? (p.nj + BN - 1) / BN : 0), t(blockIdx.x / CG), step(gridDim.x / CG) {}

  // the next tile of this CTA (all lanes of a warp together)
  __device__ __forceinline__ bool next(GmmTile *o) {
    if constexpr (MODE == GMM_DW) {
      const int64_t per = (int64_t)ti * tj;
      o->g = t / per;
      if (o->g >= P.groups) return false;
      const int l = (int)(t - o->g * per);
      o->np = (int)group_rows(P.ptr, o->g, P.rows, &o->p0, P.err);
      o->i0 = l % ti * Cfg::TI;
      o->j0 = (int64_t)(l / ti) * BN;
      o->jn = min(BN, P.nj - (int)o->j0);
    } else {
      if (!walk.seek(t, BN, ti)) return false;
      const int64_t l = t - walk.before;
      const int64_t jt = l / ti;
      o->g = walk.g;
      o->i0 = (int)(l - jt * ti) * Cfg::TI;
      o->j0 = walk.first + jt * BN;
      o->jn = (int)min((int64_t)BN, walk.count - jt * BN);
      o->np = P.np;
      o->p0 = 0;
    }
    t += step;
    return true;
  }
};

// columns that the matrix instruction computes for jn outputs
template <int CG>
__device__ __forceinline__ int instr_cols(int jn) {
  return (jn + 16 * CG - 1) / (16 * CG) * (16 * CG);
}

template <int MODE, int CG, int BN, bool BF16, typename IT, typename OT>
__global__ void __launch_bounds__(192, 1)
gmm_tc_kernel(const __grid_constant__ GmmMaps M, const GmmTcParams<IT, OT> P) {
  using Cfg = GmmCfg<MODE, CG, BN>;
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t full[Cfg::STAGES], empty[Cfg::STAGES], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_base;
  __shared__ volatile int dead;
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const uint32_t rank = CG == 2 ? tc::cluster_rank() : 0;
  const uint32_t stage0 = (tc::smem_addr(raw) + 1023) & ~1023u;

  if (tid == 0) {
    dead = 0;
    for (int s = 0; s < Cfg::STAGES; ++s) {
      ptx::mbar_init(&full[s], 1);
      ptx::mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      ptx::mbar_init(&acc_full[s], 1);
      ptx::mbar_init(&acc_empty[s], 4 * CG);
    }
    ptx::fence_mbar_init();
    tc::prefetch_map(&M.a);
    tc::prefetch_map(&M.b);
  }
  if (wid == 1) tc::tmem_alloc<CG>(&tmem_base, Cfg::COLS);
  tc::fence_before_sync();
  __syncthreads();
  if (CG == 2) tc::cluster_sync();
  tc::fence_after_sync();
  const uint32_t tmem = tmem_base;

  auto wait = [&](uint64_t *bar, uint32_t parity) {
    if (ptx::mbar_wait_bounded(bar, parity, GMM_WAIT_NS)) return true;
    atomicOr(P.err, PF_DEVERR_WAIT_TIMEOUT);
    dead = 1;
    return false;
  };

  GmmTiles<MODE, CG, BN, IT, OT> tiles(P);
  GmmTile t;
  if (wid == 0) {  // ---- copies
    uint32_t it = 0;
    bool ok = true;
    while (ok && tiles.next(&t)) {
      const int nb = (t.np + 63) / 64;
      const int ncols = instr_cols<CG>(t.jn), half = ncols / CG;
      const int gw = (int)t.g * P.group_step;
      const int ia = t.i0 + (int)rank * 128;
      if (lane == 0) {
        for (int kb = 0; kb < nb; ++kb, ++it) {
          const uint32_t s = it % Cfg::STAGES, ph = it / Cfg::STAGES & 1;
          if (!wait(&empty[s], ph ^ 1)) {
            ok = false;
            break;
          }
          const uint32_t sa = stage0 + s * Cfg::STAGE, sb = sa + Cfg::A_BYTES;
          const uint32_t bar = CG == 2 ? tc::map_rank(tc::smem_addr(&full[s]), 0)
                                       : tc::smem_addr(&full[s]);
          if constexpr (MODE == GMM_DW) {
            const int left = t.np - kb * 64;
            const int valid = left < 64 ? left : 64, r16 = (valid + 15) / 16 * 16;
            const int panels_b = (half + 63) / 64;
            if (rank == 0)
              ptx::mbar_arrive_expect_tx(&full[s], (uint32_t)(CG * (2 + panels_b) * r16 * 128));
            const int row = (int)t.p0 + kb * 64, outside = (int)P.rows;
            const int jb = (int)t.j0 + (int)rank * half;
            for (int x = 0; x < 2 + panels_b; ++x) {
              const bool is_a = x < 2;
              const uint32_t dst = is_a ? sa + x * 8192 : sb + (x - 2) * 8192;
              const int c = is_a ? ia + x * 64 : jb + (x - 2) * 64;
              if (valid == 64) {
                tc::load_2d<CG>(dst, is_a ? &M.a : &M.b, bar, c, row);
                continue;
              }
              for (int r = 0; r < r16; r += 8) {
                if (r + 8 <= valid || r >= valid)
                  tc::load_2d<CG>(dst + r * 128, is_a ? &M.a8 : &M.b8, bar, c,
                                  r < valid ? row + r : outside);
                else
                  for (int q = r; q < r + 8; ++q)
                    tc::load_2d<CG>(dst + q * 128, is_a ? &M.a1 : &M.b1, bar, c,
                                    q < valid ? row + q : outside);
              }
            }
          } else {
            const int boxes = (half + Cfg::BOX - 1) / Cfg::BOX;
            if (rank == 0)
              ptx::mbar_arrive_expect_tx(
                  &full[s], (uint32_t)(CG * (Cfg::A_BYTES + boxes * Cfg::BOX * 128)));
            if constexpr (MODE == GMM_FWD) {
              tc::load_3d<CG>(sa, &M.a, bar, kb * 64, ia, gw);
            } else {
              tc::load_3d<CG>(sa, &M.a, bar, ia, kb * 64, gw);
              tc::load_3d<CG>(sa + 8192, &M.a, bar, ia + 64, kb * 64, gw);
            }
            const int row = (int)t.j0 + (int)rank * half;
            for (int x = 0; x < boxes; ++x)
              tc::load_2d<CG>(sb + x * Cfg::BOX * 128, &M.b, bar, kb * 64, row + x * Cfg::BOX);
          }
        }
      }
      ok = __shfl_sync(~0u, (int)ok, 0);
      it = __shfl_sync(~0u, it, 0);
    }
    // every stage read: no completion is on its way to a CTA that has ended
    if (lane == 0)
      for (int x = 0; ok && x < Cfg::STAGES; ++x, ++it)
        ok = wait(&empty[it % Cfg::STAGES], (it / Cfg::STAGES & 1) ^ 1);
  } else if (wid == 1 && rank == 0) {  // ---- matrix instructions
    uint32_t it = 0, tile = 0;
    bool ok = true;
    while (ok && tiles.next(&t)) {
      const int nb = (t.np + 63) / 64;
      if (nb == 0) continue;
      const uint32_t buf = tile & 1, aph = tile >> 1 & 1;
      ++tile;
      if (lane == 0) {
        const uint32_t idesc = tc::instr_desc(BF16, MODE != GMM_FWD, MODE == GMM_DW, 128 * CG,
                                              (uint32_t)instr_cols<CG>(t.jn));
        ok = wait(&acc_empty[buf], aph ^ 1);
        tc::fence_after_sync();
        const uint32_t d = tmem + buf * BN;
        for (int kb = 0; ok && kb < nb; ++kb, ++it) {
          const uint32_t s = it % Cfg::STAGES, ph = it / Cfg::STAGES & 1;
          if (!wait(&full[s], ph)) {
            ok = false;
            break;
          }
          tc::fence_after_sync();
          const uint32_t sa = stage0 + s * Cfg::STAGE, sb = sa + Cfg::A_BYTES;
          const uint64_t da = tc::operand_desc(sa, 8192), db = tc::operand_desc(sb, 8192);
          const int left = t.np - kb * 64, steps = left < 64 ? (left + 15) / 16 : 4;
          // 16 along p: 32 bytes of a line, or two atoms of eight lines
          constexpr int STEP_A = MODE == GMM_FWD ? 2 : 128, STEP_B = MODE == GMM_DW ? 128 : 2;
          for (int q = 0; q < steps; ++q)
            tc::mma<CG>(d, da + q * STEP_A, db + q * STEP_B, idesc, kb + q > 0);
          tc::commit<CG>(&empty[s]);
        }
        if (ok) tc::commit<CG>(&acc_full[buf]);
      }
      ok = __shfl_sync(~0u, (int)ok, 0);
      it = __shfl_sync(~0u, it, 0);
    }
  } else if (wid >= 2) {  // ---- accumulator to C
    const int quad = wid & 3;  // the tensor memory lanes that this warp may read
    uint32_t tile = 0;
    bool ok = true;
    while (ok && tiles.next(&t)) {
      const bool sum = t.np > 0;
      const uint32_t buf = tile & 1, aph = tile >> 1 & 1;
      if (sum) {
        ++tile;
        ok = wait(&acc_full[buf], aph);
        ok = __all_sync(~0u, ok);
        if (!ok) break;
        tc::fence_after_sync();
      }
      OT *c = P.C + (MODE == GMM_DW ? t.g * P.stride_c : 0) + t.j0 * P.ldc;
      const int i = t.i0 + (int)rank * 128 + quad * 32 + lane;
      for (int j = 0; j < t.jn; j += 32) {
        float v[32];
        if (sum) {
          tc::tmem_load32(tmem + ((uint32_t)quad << 21) + buf * BN + j, v);
          if (j + 32 >= t.jn) {  // the accumulator is in registers: free it
            tc::fence_before_sync();
            if (lane == 0) {
              if (CG == 2) tc::mbar_arrive_cluster(tc::map_rank(tc::smem_addr(&acc_empty[buf]), 0));
              else ptx::mbar_arrive(&acc_empty[buf]);
            }
          }
        } else {
#pragma unroll
          for (int x = 0; x < 32; ++x) v[x] = 0.0f;
        }
        const int lim = t.jn - j;
#pragma unroll
        for (int x = 0; x < 32; ++x) {
          if (x < lim && i < P.ni) {
            OT *p = c + (int64_t)(j + x) * P.ldc + i;
            float o = P.alpha * v[x];
            if (P.beta != 0.0f) o += P.beta * to_f32(*p);
            *p = from_f32<OT>(o);
          }
        }
      }
    }
  }
  __syncwarp();
  tc::fence_before_sync();
  __syncthreads();
  if (dead && tid == 0 && rank == 0) {
    // copies may still be on their way into this CTA pair's shared memory
    for (int s = 0; s < Cfg::STAGES; ++s)
      if (!ptx::mbar_wait_bounded(&full[s], 0, 50000000ull))
        ptx::mbar_wait_bounded(&full[s], 1, 50000000ull);
  }
  if (CG == 2) tc::cluster_sync();
  tc::fence_after_sync();
  if (wid == 1) tc::tmem_free<CG>(tmem, Cfg::COLS);
}

}  // namespace pf
