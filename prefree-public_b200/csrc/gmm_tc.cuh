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
// Measured: 16384 rows, one group, n 4096, k 2048, bf16: 160-183 us in short
// bursts (cuBLAS's product of the same size 1-2 % less in the same call), 207-213
// us in a long run under the power cap (cuBLAS 201-211); 16 groups of 1024 rows
// 170-203 and 230-236 us, 16 uneven ones 252-259; 64 groups of 128 rows, 2048 x
// 2048: 102-113 us, 82 us of it the weights' bytes. Large products are bound by
// the tensor cores and the power cap (what uneven groups cost beyond is open),
// products of few rows by the weights' bytes, gradients of few rows by their own:
// 64 of 2048 x 2048 over 64 rows each take 140-148 us, setting those bytes to
// zero 140.
//
// DW: rows past a group's end belong to the next group and must not meet the
// sum (0 * NaN is NaN). A group's last, partial block is announced to a warp of
// its own, which clears the rows up to the next multiple of 16 (what the matrix
// instruction reads) in both operands before it passes the stage on. That takes
// about as long as the ring looks ahead, so the block is loaded first and used
// two blocks later. (Copied in boxes of 8 rows and single rows, filled up by
// boxes outside of the array, it cost 3 us a tile.)
#pragma once

#include "gmm_common.cuh"
#include "tc_ptx.cuh"

namespace pf {

enum GmmMode { GMM_FWD = 0, GMM_DX = 1, GMM_DW = 2 };

struct GmmMaps {
  CUtensorMap a, b;
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
  int parts;               // SPLIT: parts of each sum, at least 2
  int64_t most;            // SPLIT: tiles that there is scratch for
  float *partial;          // SPLIT: 128 * BN floats for each tile and part
  unsigned *arrived;       // SPLIT: 4 counters for each tile, 0 between calls
  bool aligned;            // C's rows start on 16-byte boundaries
  bool plain;              // 16-bit C, aligned, beta = 0
  unsigned *err;
};

// The accumulator holds i along its lanes and j along its columns, C the other
// way round. Each epilogue warp turns 32 x 32 of it in shared memory: 16-bit
// results as pairs of columns through transposing matrix stores (lines of 64
// bytes), everything else as floats (lines of 128 bytes); 16 bytes of padding
// to a line keep the banks apart. Storing straight from the registers, 2 bytes
// a lane and 64 bytes an instruction, bound the kernel: 790 us instead of 140
// for 64 gradients of 2048 x 2048. (Rows of 256 bytes put together by all four
// warps take 140 too.)
constexpr int GMM_STAGING = 64 * (64 + 16);  // and 32 * (128 + 16) is less

template <typename OT>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<float>(float, float) { return 0; }  // not called

// 32 lanes x 64 columns of tensor memory -> alpha * v, rounded, [column][lane]
// in two areas of 32 columns, 32 * 80 bytes each
template <typename OT>
__device__ __forceinline__ void stage_pairs(uint8_t *stage, uint32_t src, float alpha) {
  const int lane = threadIdx.x & 31;
  float v[4][16];  // lanes 0-15 and 16-31 of two times 32 columns: fragments of 8 x 8
  tc::tmem_load16x256b_x4(src, v[0]);
  tc::tmem_load16x256b_x4(src + (16u << 16), v[1]);
  tc::tmem_load16x256b_x4(src + 32, v[2]);
  tc::tmem_load16x256b_x4(src + 32 + (16u << 16), v[3]);
  tc::tmem_load_wait();
  const uint32_t at = ptx::smem_addr(stage) + (lane & 7) * 80 + (lane >> 3) * 16;
#pragma unroll
  for (int b = 0; b < 8; ++b) {  // eight columns
    const float *lo = v[b / 4 * 2] + b % 4 * 4, *hi = v[b / 4 * 2 + 1] + b % 4 * 4;
    tc::store_matrices_t(at + b * 8 * 80, pack2<OT>(alpha * lo[0], alpha * lo[1]),
                         pack2<OT>(alpha * lo[2], alpha * lo[3]),
                         pack2<OT>(alpha * hi[0], alpha * hi[1]),
                         pack2<OT>(alpha * hi[2], alpha * hi[3]));
  }
}
// ... to C (zeros where `stage` is null), whose rows are 16-byte aligned; ni of 32
// i and nj of 64 j exist
template <typename OT>
__device__ __forceinline__ void store_pairs(const uint8_t *stage, OT *c, int64_t ldc, int ni,
                                            int nj) {
  const int lane = threadIdx.x & 31, x = lane & 3;
  const uint8_t *from = stage + (lane >> 2) * 80 + x * 16;
  OT *p = c + (lane >> 2) * ldc + x * 8;
  if (ni == 32 && nj == 64) {
    uint4 v[8];
#pragma unroll
    for (int q = 0; q < 8; ++q)
      v[q] = stage ? *reinterpret_cast<const uint4 *>(from + q * 640) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int q = 0; q < 8; ++q) *reinterpret_cast<uint4 *>(p + q * 8 * ldc) = v[q];
    return;
  }
#pragma unroll 1
  for (int j = lane >> 2; j < nj; j += 8, from += 640, p += 8 * ldc) {
    const uint4 v = stage ? *reinterpret_cast<const uint4 *>(from) : make_uint4(0, 0, 0, 0);
    if (x * 8 + 8 <= ni) {
      *reinterpret_cast<uint4 *>(p) = v;
    } else {
      alignas(16) OT e[8];
      *reinterpret_cast<uint4 *>(e) = v;
      for (int y = 0; y < ni - x * 8; ++y) p[y] = e[y];
    }
  }
}
__device__ __forceinline__ void stage_floats(uint8_t *stage, uint32_t src, bool sum) {
  const int lane = threadIdx.x & 31;
  float v[32];
  if (sum) {
    tc::tmem_load32(src, v);
  } else {
#pragma unroll
    for (int x = 0; x < 32; ++x) v[x] = 0.0f;
  }
#pragma unroll
  for (int x = 0; x < 32; ++x) *reinterpret_cast<float *>(stage + x * 144 + lane * 4) = v[x];
}
// alpha * staged + beta * C; `aligned`: C's rows are 16-byte aligned
template <typename OT>
__device__ __forceinline__ void store_floats(const uint8_t *stage, OT *c, int64_t ldc, int ni,
                                             int nj, float alpha, float beta, bool aligned) {
  constexpr int E = 16 / (int)sizeof(OT), LPR = 32 / E;  // elements a lane, lanes a row
  const int lane = threadIdx.x & 31, x = lane % LPR * E;
  if (!aligned) {
    if (lane < ni)
      for (int j = 0; j < nj; ++j) {
        float o = alpha * *reinterpret_cast<const float *>(stage + j * 144 + lane * 4);
        if (beta != 0.0f) o += beta * to_f32(c[j * ldc + lane]);
        c[j * ldc + lane] = from_f32<OT>(o);
      }
    return;
  }
  for (int j = lane / LPR; j < nj; j += E) {
    OT *p = c + j * ldc + x;
    const bool whole = x + E <= ni;
    alignas(16) OT e[E];
    if (beta != 0.0f) {
      if (whole) *reinterpret_cast<uint4 *>(e) = *reinterpret_cast<const uint4 *>(p);
      else
        for (int y = 0; y < E; ++y) e[y] = x + y < ni ? p[y] : from_f32<OT>(0.0f);
    }
#pragma unroll
    for (int y = 0; y < E; ++y) {
      float o = alpha * *reinterpret_cast<const float *>(stage + j * 144 + (x + y) * 4);
      if (beta != 0.0f) o += beta * to_f32(e[y]);
      e[y] = from_f32<OT>(o);
    }
    if (whole) *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(e);
    else
      for (int y = 0; y < E; ++y)
        if (x + y < ni) p[y] = e[y];
  }
}

template <int MODE, int CG, int BN>
struct GmmCfg {
  static constexpr int TI = 128 * CG;           // i of a tile
  static constexpr int BH = BN / CG;            // B rows that one CTA loads
  static constexpr int BOX = 32;                // rows of one B box (FWD, DX)
  static constexpr int A_BYTES = 128 * 128;
  static constexpr int B_BYTES = BH * 128;
  static constexpr int STAGE = A_BYTES + B_BYTES;
  static constexpr int STAGES = 200 * 1024 / STAGE;
  static constexpr int COLS = 2 * BN;           // tensor memory columns
  static constexpr int NT = MODE == GMM_DW ? 224 : 192;
  static constexpr int SMEM = STAGES * STAGE + 4 * GMM_STAGING + 1024;  // and alignment
};

// SPLIT: a tile's sum is cut into parts where there are too few tiles to fill the
// GPU (a decoding step, a narrow layer): see the epilogue. 17 rows, n 512, k
// 2048, one group: 4 tiles of 32 blocks each become 32 parts.
constexpr uint64_t GMM_WAIT_NS = 4000000000ull;

// columns that the matrix instruction computes for jn outputs
template <int CG>
__device__ __forceinline__ int instr_cols(int jn) {
  return (jn + 16 * CG - 1) / (16 * CG) * (16 * CG);
}

// One tile: where it lies and how long its sum is.
struct GmmTile {
  int64_t g;
  int i0;          // first i of the CTA (pair)
  int64_t j0;      // first j: an absolute row (FWD, DX) or a column of dY (DW)
  int jn;          // number of j
  int64_t p0;      // first of p (DW: a row)
  int np;          // length of the sum
  int64_t tile;    // SPLIT: the tile's number
  int part;        // SPLIT: which part of its sum
};

template <int MODE, int CG, int BN, bool SPLIT, typename IT, typename OT>
struct GmmTiles {
  using Cfg = GmmCfg<MODE, CG, BN>;
  const GmmTcParams<IT, OT> &P;
  GroupWalk<IT> walk;
  int ti, tj;
  int64_t t, step;         // items: tiles, or (SPLIT) parts of tiles
  int64_t g = 0;           // DW: the next item's group and place in it
  int l = 0, step_l = 0;
  int64_t step_g = 0;

  __device__ GmmTiles(const GmmTcParams<IT, OT> &p)
      : P(p), walk{p.ptr, p.groups, p.rows, p.err}, ti((p.ni + Cfg::TI - 1) / Cfg::TI),
        tj(MODE == GMM_DW ? (p.nj + BN - 1) / BN : 0), t(blockIdx.x / CG), step(gridDim.x / CG) {
    if constexpr (MODE == GMM_DW) {
      const int64_t per = (int64_t)ti * tj * (SPLIT ? P.parts : 1);
      g = t / per;
      l = (int)(t - g * per);
      step_g = step / per;
      step_l = (int)(step - step_g * per);
    }
  }

  // the next tile of this CTA (all lanes of a warp together)
  __device__ __forceinline__ bool next(GmmTile *o) {
    if constexpr (MODE == GMM_DW) {
      if (g >= P.groups) return false;
      const int parts = SPLIT ? P.parts : 1;
      const int l = this->l / parts;
      if (SPLIT) o->tile = t / parts, o->part = this->l - l * parts;
      o->g = g;
      o->np = (int)group_rows(P.ptr, o->g, P.rows, &o->p0, P.err);
      o->i0 = l % ti * Cfg::TI;
      o->j0 = (int64_t)(l / ti) * BN;
      o->jn = min(BN, P.nj - (int)o->j0);
      g += step_g;
      this->l += step_l;
      if (this->l >= ti * tj * parts) this->l -= ti * tj * parts, ++g;
    } else {
      const int64_t t = SPLIT ? this->t / P.parts : this->t;
      if (!walk.seek(t, BN, ti)) return false;
      if (SPLIT) o->tile = t, o->part = (int)(this->t - t * P.parts);
      // rows and n fit 31 bits, and so do a group's row tiles; its tiles may not
      const int64_t l = t - walk.before;
      const int jt = l <= INT32_MAX ? (int)l / ti : (int)(l / ti);
      o->g = walk.g;
      o->i0 = (int)(l - (int64_t)jt * ti) * Cfg::TI;
      // the group's tiles are of equal size, up to the instruction's step: full
      // ones and a remainder would leave some CTAs with more to do than others
      const int nt = (int)((walk.count + BN - 1) / BN);
      const int each = instr_cols<CG>((int)((walk.count + nt - 1) / nt));
      o->j0 = walk.first + (int64_t)jt * each;
      o->jn = (int)min((int64_t)each, walk.count - (int64_t)jt * each);
      o->np = P.np;
      o->p0 = 0;
    }
    this->t += step;
    if (SPLIT && o->tile >= P.most) {  // groups that overlap: no valid pointers
      atomicOr(P.err, PF_DEVERR_ROWPTR);
      return false;
    }
    if (SPLIT) {  // whole blocks of 64; a part of a short sum can be empty
      const int64_t nb = (o->np + 63) / 64;
      const int b0 = (int)(nb * o->part / P.parts), b1 = (int)(nb * (o->part + 1) / P.parts);
      o->np = min(o->np, b1 * 64) - b0 * 64;
      if (o->np < 0) o->np = 0;
      o->p0 += b0 * 64;
    }
    return true;
  }
};

template <int MODE, int CG, int BN, bool BF16, bool SPLIT, typename IT, typename OT>
__global__ void __launch_bounds__(GmmCfg<MODE, CG, BN>::NT, 1)
gmm_tc_kernel(const __grid_constant__ GmmMaps M, const GmmTcParams<IT, OT> P) {
  using Cfg = GmmCfg<MODE, CG, BN>;
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t full[Cfg::STAGES], empty[Cfg::STAGES], acc_full[2], acc_empty[2];
  __shared__ uint64_t tail[Cfg::STAGES], cleared[Cfg::STAGES];  // DW
  __shared__ uint32_t tmem_base;
  __shared__ volatile int dead;
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const uint32_t rank = CG == 2 ? tc::cluster_rank() : 0;
  const uint32_t stage0 = (tc::smem_addr(raw) + 1023) & ~1023u;

  if (tid == 0) {
    dead = 0;
    for (int s = 0; s < Cfg::STAGES; ++s) {
      ptx::mbar_init(&full[s], CG);
      ptx::mbar_init(&empty[s], 1);
      ptx::mbar_init(&tail[s], 1);
      ptx::mbar_init(&cleared[s], 1);
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

  // called by whole warps
  auto wait = [&](uint64_t *bar, uint32_t parity) -> bool {
    if (__all_sync(~0u, ptx::mbar_wait_bounded(bar, parity, GMM_WAIT_NS))) return true;
    atomicOr(P.err, PF_DEVERR_WAIT_TIMEOUT);
    dead = 1;
    return false;
  };

  GmmTiles<MODE, CG, BN, SPLIT, IT, OT> tiles(P);
  GmmTile t;
  if (wid == 0) {  // ---- copies
    const uint32_t full_at = CG == 2 ? tc::map_rank(tc::smem_addr(&full[0]), 0)
                                     : tc::smem_addr(&full[0]);
    uint32_t it = 0;
    bool ok = true;
    while (ok && tiles.next(&t)) {
      const int nb = (t.np + 63) / 64;
      const int ncols = instr_cols<CG>(t.jn), half = ncols / CG;
      const int gw = (int)t.g * P.group_step;
      const int ia = t.i0 + (int)rank * 128;
      const int p_first = SPLIT ? (int)t.p0 : 0;  // (DW reads t.p0)
      for (int kb = 0; kb < nb; ++kb, ++it) {
        const uint32_t s = it % Cfg::STAGES, ph = it / Cfg::STAGES & 1;
        if (!wait(&empty[s], ph ^ 1)) {
          ok = false;
          break;
        }
        if (tc::elect()) {
          const uint32_t sa = stage0 + s * Cfg::STAGE, sb = sa + Cfg::A_BYTES;
          const uint32_t bar = full_at + s * 8;
          if constexpr (MODE == GMM_DW) {
            const int panels_b = (half + 63) / 64;
            const uint32_t bytes = (uint32_t)(2 + panels_b) * 8192;
            // the partial block goes first
            const bool ragged = (t.np & 63) != 0, whole = !ragged || kb > 0;
            const int block = ragged ? (kb > 0 ? kb - 1 : nb - 1) : kb;
            const uint32_t to = whole ? bar : tc::smem_addr(&tail[s]);
            if (!whole) {
              ptx::mbar_arrive_expect_tx(&tail[s], bytes);
            } else if (rank == 0) {
              ptx::mbar_arrive_expect_tx(&full[s], CG * bytes);
              if (CG == 2) ptx::mbar_arrive(&full[s]);
            }
            const int row = (int)t.p0 + block * 64, jb = (int)t.j0 + (int)rank * half;
            tc::load_2d<CG>(sa, &M.a, to, ia, row);
            tc::load_2d<CG>(sa + 8192, &M.a, to, ia + 64, row);
            for (int x = 0; x < panels_b; ++x)
              tc::load_2d<CG>(sb + x * 8192, &M.b, to, jb + x * 64, row);
          } else {
            const int boxes = (half + Cfg::BOX - 1) / Cfg::BOX;
            if (rank == 0) {
              ptx::mbar_arrive_expect_tx(
                  &full[s], (uint32_t)(CG * (Cfg::A_BYTES + boxes * Cfg::BOX * 128)));
              if (CG == 2) ptx::mbar_arrive(&full[s]);
            }
            const int p = p_first + kb * 64;
            if constexpr (MODE == GMM_FWD) {
              tc::load_3d<CG>(sa, &M.a, bar, p, ia, gw);
            } else {
              tc::load_3d<CG>(sa, &M.a, bar, ia, p, gw);
              tc::load_3d<CG>(sa + 8192, &M.a, bar, ia + 64, p, gw);
            }
            const int row = (int)t.j0 + (int)rank * half;
            for (int x = 0; x < boxes; ++x)
              tc::load_2d<CG>(sb + x * Cfg::BOX * 128, &M.b, bar, p, row + x * Cfg::BOX);
          }
        }
        __syncwarp();
      }
    }
    // every stage read: no completion is on its way to a CTA that has ended
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
      const uint32_t idesc = tc::instr_desc(BF16, MODE != GMM_FWD, MODE == GMM_DW, 128 * CG,
                                            (uint32_t)instr_cols<CG>(t.jn));
      ok = wait(&acc_empty[buf], aph ^ 1);
      tc::fence_after_sync();
      const uint32_t d = tmem + buf * BN;
      // DW: a partial block is loaded first and used after the next `late` ones, by
      // when its rows are cleared
      const bool ragged = MODE == GMM_DW && (t.np & 63) != 0;
      const int late = min(nb - 1, 2);
      for (int c = 0; ok && c < nb; ++c) {
        const int kb = !ragged || c > late ? c : c < late ? c + 1 : 0;  // as loaded
        const uint32_t n = it + kb, s = n % Cfg::STAGES, ph = n / Cfg::STAGES & 1;
        if (!wait(&full[s], ph)) {
          ok = false;
          break;
        }
        tc::fence_after_sync();
        if (tc::elect()) {
          const uint32_t sa = stage0 + s * Cfg::STAGE, sb = sa + Cfg::A_BYTES;
          const uint64_t da = tc::operand_desc(sa, 8192), db = tc::operand_desc(sb, 8192);
          const int left = ragged ? (kb > 0 ? 64 : t.np & 63) : t.np - kb * 64;
          // 16 along p: 32 bytes of a line, or two atoms of eight lines
          constexpr int STEP_A = MODE == GMM_FWD ? 2 : 128, STEP_B = MODE == GMM_DW ? 128 : 2;
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (q * 16 < left)
              tc::mma<CG>(d, da + q * STEP_A, db + q * STEP_B, idesc, c + q > 0);
          tc::commit<CG>(&empty[s]);
          if (c + 1 == nb) tc::commit<CG>(&acc_full[buf]);
        }
        __syncwarp();
      }
      it += nb;
    }
  } else if (MODE == GMM_DW && wid == 6) {  // ---- rows past a group's end
    // The second CTA of a pair tells the first one's warp, which acquires its
    // writes before it passes the stage on for both: the warp that issues the
    // matrix instructions waits at its own CTA's scope alone (a wait at the
    // cluster's costs it as much as two blocks).
    const uint32_t leader = CG == 2 ? tc::map_rank(tc::smem_addr(&cleared[0]), 0) : 0;
    uint32_t it = 0, parity = 0;  // parity: one bit to a stage, flipped at each use
    while (tiles.next(&t)) {
      const int nb = (t.np + 63) / 64, valid = t.np & 63;
      const uint32_t s = it % Cfg::STAGES;
      it += nb;
      if (valid == 0) continue;
      const uint32_t turn = parity >> s & 1;
      if (!wait(&tail[s], turn)) break;
      parity ^= 1u << s;
      const int panels = 2 + (instr_cols<CG>(t.jn) / CG + 63) / 64;
      const int zero = ((valid + 15) & ~15) - valid;  // the matrix instruction reads no more
      uint8_t *at = raw + (stage0 - tc::smem_addr(raw)) + s * Cfg::STAGE + valid * 128;
      for (int x = lane; x < panels * zero * 8; x += 32) {
        const int p = x / (zero * 8);
        *reinterpret_cast<uint4 *>(at + p * 8192 + (x - p * zero * 8) * 16) =
            make_uint4(0, 0, 0, 0);
      }
      ptx::fence_proxy_async_smem();
      __syncwarp();
      if (CG == 2 && rank != 0) {
        if (lane == 0) tc::mbar_arrive_release(leader + s * 8);
      } else {
        if (CG == 2) {
          if (!wait(&cleared[s], turn)) break;
          tc::acquire_cluster(&cleared[s], turn);
          __syncwarp();
        }
        if (lane == 0)
          for (int x = 0; x < CG; ++x) ptx::mbar_arrive(&full[s]);
      }
      __syncwarp();
    }
  } else if (wid >= 2) {  // ---- accumulator to C
    const int quad = wid & 3;  // the tensor memory lanes that this warp may read
    uint8_t *stage = raw + (stage0 - tc::smem_addr(raw)) + Cfg::STAGES * Cfg::STAGE +
                     quad * GMM_STAGING;
    uint32_t tile = 0;
    bool ok = true;
    while (ok && tiles.next(&t)) {
      const bool sum = t.np > 0;
      const uint32_t buf = tile & 1, aph = tile >> 1 & 1;
      if (sum) {
        ++tile;
        ok = wait(&acc_full[buf], aph);
        if (!ok) break;
        tc::fence_after_sync();
      }
      const int i0 = t.i0 + (int)rank * 128 + quad * 32;  // this warp's 32 of i
      OT *c = P.C + (MODE == GMM_DW ? t.g * P.stride_c : 0) + t.j0 * P.ldc + i0;
      const uint32_t src = tmem + ((uint32_t)quad << 21) + buf * BN;
      // the accumulator has been read: hand it back
      auto release = [&] {
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          if (CG == 2) tc::mbar_arrive_cluster(tc::map_rank(tc::smem_addr(&acc_empty[buf]), 0));
          else ptx::mbar_arrive(&acc_empty[buf]);
        }
      };
      const int ni = min(32, P.ni - i0);
      if constexpr (SPLIT) {
        // this warp's 32 of i: the part's sum goes to memory, and the warp that
        // brings the last part adds all of them, in their order
        const int64_t mine = (int64_t)quad * 32 * BN + lane, item = 128 * BN;
        float *to = P.partial + (t.tile * P.parts + t.part) * item + mine;
        for (int j = 0; j < t.jn; j += 32) {
          float v[32] = {};
          if (sum) tc::tmem_load32(src + j, v);
#pragma unroll
          for (int x = 0; x < 32; ++x)
            if (j + x < t.jn) __stcg(to + (j + x) * 32, v[x]);
        }
        if (sum) release();
        __threadfence();
        __syncwarp();
        unsigned before = 0;
        unsigned *arrived = P.arrived + t.tile * 4 + quad;
        if (lane == 0) before = atomicAdd(arrived, 1u);
        if (__shfl_sync(~0u, before, 0) + 1 < (unsigned)P.parts) continue;
        if (lane == 0) *arrived = 0;
        __threadfence();
        const float *from = P.partial + t.tile * P.parts * item + mine;
        for (int j = 0; j < t.jn; j += 32, c += 32 * P.ldc) {
          float v[32] = {};
          for (int p = 0; p < P.parts; p += 4) {  // four parts on their way at once
            float w[4][32];
#pragma unroll
            for (int y = 0; y < 4; ++y)
#pragma unroll
              for (int x = 0; x < 32; ++x)
                w[y][x] = p + y < P.parts && j + x < t.jn
                              ? __ldcg(from + (p + y) * item + (j + x) * 32)
                              : 0.0f;
#pragma unroll
            for (int y = 0; y < 4; ++y)
#pragma unroll
              for (int x = 0; x < 32; ++x) v[x] += w[y][x];
          }
#pragma unroll
          for (int x = 0; x < 32; ++x)
            *reinterpret_cast<float *>(stage + x * 144 + lane * 4) = v[x];
          __syncwarp();
          store_floats(stage, c, P.ldc, ni, min(32, t.jn - j), P.alpha, P.beta, P.aligned);
          __syncwarp();
        }
      } else if (sizeof(OT) == 2 && P.plain) {
        for (int j = 0; j < t.jn; j += 64, c += 64 * P.ldc) {
          if (sum) stage_pairs<OT>(stage, src + j, P.alpha);
          if (sum && j + 64 >= t.jn) release();
          else __syncwarp();
          store_pairs(sum ? stage : nullptr, c, P.ldc, ni, min(64, t.jn - j));
          __syncwarp();
        }
      } else {
        for (int j = 0; j < t.jn; j += 32, c += 32 * P.ldc) {
          stage_floats(stage, src + j, sum);
          if (sum && j + 32 >= t.jn) release();
          else __syncwarp();
          store_floats(stage, c, P.ldc, ni, min(32, t.jn - j), P.alpha, P.beta, P.aligned);
          __syncwarp();
        }
      }
    }
  }
  __syncwarp();
  tc::fence_before_sync();
  __syncthreads();
  if (dead && tid == 0) {
    // copies may still be on their way into this CTA pair's shared memory: the
    // leader's barriers count both CTAs' whole blocks, each CTA's own its partial ones
    for (int s = 0; s < Cfg::STAGES; ++s) {
      if (rank == 0) ptx::mbar_drain(&full[s], 50000000ull);
      if (MODE == GMM_DW) ptx::mbar_drain(&tail[s], 50000000ull);
    }
  }
  if (CG == 2) tc::cluster_sync();
  tc::fence_after_sync();
  if (wid == 1) tc::tmem_free<CG>(tmem, Cfg::COLS);
}

}  // namespace pf
