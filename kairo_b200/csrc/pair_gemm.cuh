// Dense product D = A * B^T on the tensor cores of sm_100a, tile by tile, with
// an epilogue that takes each accumulator tile straight from TMEM.
//
//   D[m, n] = sum_k A(m, k) * B(n, k),  16-bit operands, fp32 accumulation
//
// Each operand is a row-major matrix in global memory, read either with k
// along its rows (K-major: A is m x k) or with k down its rows (MN-major: A is
// k x m), as the tensor maps and the shared-memory descriptors say; nothing is
// transposed in memory.
//
// Tile.  A cluster of two CTAs computes 256 x 256: each CTA holds 128 rows of A
// and 128 rows of B in its shared memory, the leader's tcgen05.mma
// (cta_group::2) reads both, and each CTA's TMEM receives its own 128 rows x
// 256 columns.  A stage of 64 k costs a CTA 32 KB for 512 tensor cycles, 64
// bytes a cycle; one CTA alone would need 96 for the same rate (128 x 256 tiles).
//
// Segments.  The units add each step of 16 k with truncation towards zero, about
// 9e-8 of the sum so far: over 256 steps a logit would lose 1.2e-5 of itself, ten
// times what fp32 sums lose.  So a tile's sum is cut into segments of `seg` stages;
// the epilogue adds them up in registers (128 fp32 a thread), with rounding, while
// the next segment runs in the other half of TMEM.  A segment of 512 k takes 4096
// tensor cycles and its addition some 600 of the epilogue's.
//
// Roles (384 threads, one CTA per SM, persistent): warp 0 loads, warp 1
// allocates TMEM and (in the leader) issues the MMAs, warps 4..11 are the
// epilogue: two warps share each quarter of the lanes and take 128 columns
// each.  The 128 sums leave no room in the 168 registers that every thread
// starts with, so tiles of 256 columns move registers from the first four warps
// to the others.  Every wait on a barrier is bounded (ptx::wait_parity).
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "internal.h"
#include "ptx.cuh"
#include "tc_common.cuh"

namespace kairo {
namespace {

constexpr int kPairThreads = 384;
constexpr int kPairEpiWarps = 8;
constexpr int kPairEpiFirst = 4;  // the first of them
// Registers a thread after the launch: of warps 0..3 and of the epilogue's (tiles of 256 columns)
constexpr int kPairRegsLow = 72, kPairRegsHigh = 208;
constexpr int kPairRegsAll = 32 * (kPairEpiFirst * kPairRegsLow + kPairEpiWarps * kPairRegsHigh);
constexpr int kPairTileM = 256;      // rows of a cluster's tile (128 a CTA)
constexpr int kPairTileN = 256;
constexpr int kPairK = 64;           // k of one stage
constexpr int kPairHalf = 128 * kPairK * 2;  // bytes of one operand's part of a stage in one CTA
constexpr int kPairBoxRows = 64;  // of a copy, at most
// Bytes of a stage and stages, for tiles of `tn` columns; 192 KB in all.
constexpr int pair_stage_bytes(int tn) { return kPairHalf + tn / 2 * kPairK * 2; }
constexpr int pair_stages(int tn) { return 192 * 1024 / pair_stage_bytes(tn); }
constexpr int kPairEpiCols = kPairTileN / (kPairEpiWarps / 4);
constexpr int kPairOutBytes = 4096;  // of each epilogue warp, to turn rows a lane into rows a warp
constexpr size_t kPairSmem = 192 * 1024 + kPairEpiWarps * kPairOutBytes + 2048;
constexpr int kPairClusters = 74;    // pairs of a B200's 148 SMs, for plans that must not depend on the current device
static_assert(kPairSmem <= kMaxSmem, "shared memory");

// Tiles of one product.  They are visited `group_m` rows of tiles at a time,
// rows fastest: the group's A and the current columns' B stay in L2.
struct PairShape {
  int tiles_m, tiles_n, ksteps, group_m;
  int seg;     // stages of one segment
  int splits;  // parts of k, each a tile of its own
  int copies;  // of B's rows, copy_rows after one another: cluster c reads copy c % copies (one column of tiles only)
  int copy_rows;
};

struct PairTile {
  int mt, nt, split;
  int k0, k1;  // stages
};

__device__ __forceinline__ PairTile pair_tile(const PairShape& s, int t) {
  // divisions, the 64-bit ones above all, cost more than a short tile's products
  PairTile o;
  o.split = 0;
  o.k0 = 0;
  o.k1 = s.ksteps;
  if (s.splits > 1) {
    const int all = s.tiles_m * s.tiles_n;
    o.split = t / all;
    t -= o.split * all;
    o.k0 = static_cast<int>(static_cast<int64_t>(s.ksteps) * o.split / s.splits);
    o.k1 = static_cast<int>(static_cast<int64_t>(s.ksteps) * (o.split + 1) / s.splits);
  }
  const int per = s.group_m * s.tiles_n;
  const int g = t / per, r = t - g * per;
  const int m0 = g * s.group_m;
  const int gm = min(s.group_m, s.tiles_m - m0);
  o.nt = r / gm;
  o.mt = m0 + (r - o.nt * gm);
  return o;
}

// Epi supplies `struct Args` and
//   __device__ Epi(const Args&, int row_in_tile, int part, uint8_t* out)
//   __device__ void tile(const PairTile&, float (&v)[TN / 2])   its columns of one tile
//   __device__ void done()                                      after the CTA's last tile
// and is made once per thread and launch; `out` is the warp's kPairOutBytes.
//
// TN: columns of a tile.  64 or 128 where B has few rows (the tokens to be scored) and A is the large
// operand: a stage is then 16 KB of A and 4 or 8 of B, and a product costs 70 cycles instead of 128.
template <int IN_FMT, bool A_MN, bool B_MN, class Epi, int TN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    k_pair_gemm(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                const PairShape shape, unsigned* err, const __grid_constant__ typename Epi::Args eargs) {
  constexpr int ST = pair_stages(TN);
  constexpr int STAGE = pair_stage_bytes(TN);
  static_assert(TN == 256 || ((TN == 64 || TN == 128) && !B_MN), "columns of a tile");
  constexpr uint32_t IDESC = ptx::make_idesc_f16(IN_FMT, A_MN ? 1u : 0u, B_MN ? 1u : 0u, kPairTileM, TN);
  constexpr uint32_t TMEM_COLS = 2 * TN;
  constexpr int COLS = TN / (kPairEpiWarps / 4);  // of an epilogue warp
  // A CTA's half of an operand comes in boxes, one lane each: 64 k x up to 64 rows, or 64 columns x 64 k.
  constexpr int BOX_B = TN / 2 < kPairBoxRows ? TN / 2 : kPairBoxRows;
  constexpr int NA = 128 / kPairBoxRows, NB = TN / 2 / BOX_B;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* out = smem + ST * STAGE;
  uint64_t* full = reinterpret_cast<uint64_t*>(out + kPairEpiWarps * kPairOutBytes);  // used in the leader
  uint64_t* empty = full + ST;
  uint64_t* tfull = empty + ST;
  uint64_t* tempty = tfull + 2;  // used in the leader
  uint64_t* mma_done = tempty + 2;
  int* misc = reinterpret_cast<int*>(mma_done + 1);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(misc);
  volatile int* abort_flag = misc + 1;
  int* issued = misc + 4;  // [ST]: parity + 1 of the last load into each stage

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = ptx::cluster_rank();
  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      ptx::mbar_init(&full[s], 1);
      ptx::mbar_init(&empty[s], 1);
      issued[s] = 0;
    }
    for (int k = 0; k < 2; ++k) {
      ptx::mbar_init(&tfull[k], 1);
      ptx::mbar_init(&tempty[k], 2 * kPairEpiWarps);
    }
    ptx::mbar_init(mma_done, 1);
    misc[1] = 0;
    ptx::mbar_init_fence();
  }
  if (warp == 0 && lane == 0) {
    ptx::prefetch_tmap(&tmap_a);
    ptx::prefetch_tmap(&tmap_b);
  }
  __syncthreads();
  ptx::cluster_sync();  // both CTAs' barriers exist
  if (warp == 1) {
    ptx::tmem_alloc_pair(tmem_slot, TMEM_COLS);
    ptx::tmem_relinquish_pair();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int ntiles = shape.tiles_m * shape.tiles_n * shape.splits;
  const int first = blockIdx.x >> 1, step = gridDim.x >> 1;

  if (warp < kPairEpiFirst) {
    if constexpr (TN == 256) ptx::registers_down<kPairRegsLow>();
    if (warp == 0) {
      // ------------------------------------------------------------ loads
      const bool is_a = lane < NA;
      const uint64_t pol = ptx::policy_evict_last();
      const int box = is_a ? lane : lane - NA;
      const void* map = is_a ? static_cast<const void*>(&tmap_a) : static_cast<const void*>(&tmap_b);
      const uint32_t mine = lane < NA + NB ? 1u : 0u;
      const bool mn = is_a ? A_MN : B_MN;
      const uint32_t dst_off =
          (is_a ? 0u : kPairHalf) + static_cast<uint32_t>(mine ? box : 0) * (kPairBoxRows * kPairK * 2);
      const int shift = is_a ? 0 : first % shape.copies * shape.copy_rows;
      int sidx = 0;
      uint32_t sph = 0;
      bool alive = true;
      for (int t = first; t < ntiles && alive; t += step) {
        const PairTile pt = pair_tile(shape, t);
        const int tile0 = is_a ? pt.mt * 256 + static_cast<int>(rank) * 128 : pt.nt * TN + static_cast<int>(rank) * (TN / 2);
        const int r0 = tile0 + box * kPairBoxRows + shift;
        for (int k = pt.k0; k < pt.k1; ++k) {
          int ok = ptx::wait_parity(&empty[sidx], sph ^ 1u, abort_flag, err, kTagEmpty, kWaitCycles);
          ok = __shfl_sync(0xffffffffu, ok, 0);
          if (!ok) {
            alive = false;
            break;
          }
          const uint32_t bar = ptx::peer_smem_u32(&full[sidx], 0);
          if (rank == 0) {
            if (lane == 0) issued[sidx] = static_cast<int>(sph) + 1;
            ptx::mbar_expect_tx_if(lane == 0 ? 1u : 0u, &full[sidx], 2 * STAGE);
          }
          ptx::tma_load_2d_pair_if(mine, smem + sidx * STAGE + dst_off, map, mn ? r0 : k * kPairK,
                                   mn ? k * kPairK : r0, bar, pol);
          __syncwarp();
          if (rank == 0) ptx::mbar_arrive_if(lane == 0 ? 1u : 0u, &full[sidx]);
          if (++sidx == ST) {
            sidx = 0;
            sph ^= 1u;
          }
        }
      }
    } else if (warp == 1 && rank == 0) {
      // ------------------------------------------------------------ MMA issuer
      const uint32_t leader = lane == 0 ? 1u : 0u;
      const uint32_t sbase = ptx::smem_u32(smem);
      const uint64_t adesc = A_MN ? ptx::make_smem_desc(sbase, kPairBoxRows * kPairK * 2, 1024, 2u)
                                  : ptx::make_smem_desc(sbase, 16, 1024, 2u);
      const uint64_t bdesc = B_MN ? ptx::make_smem_desc(sbase + kPairHalf, kPairBoxRows * kPairK * 2, 1024, 2u)
                                  : ptx::make_smem_desc(sbase + kPairHalf, 16, 1024, 2u);
      const uint32_t a_lo = static_cast<uint32_t>(adesc), a_hi = static_cast<uint32_t>(adesc >> 32);
      const uint32_t b_lo = static_cast<uint32_t>(bdesc), b_hi = static_cast<uint32_t>(bdesc >> 32);
      // 16 k further: 32 bytes along a 128-byte row, or 16 rows of 128 bytes
      constexpr uint32_t AK = (A_MN ? 2048 : 32) >> 4, BK = (B_MN ? 2048 : 32) >> 4;
      int sidx = 0, slot = 0;
      uint32_t sph = 0, aphase = 0;
      bool alive = true;
      for (int t = first; t < ntiles && alive; t += step) {
        const PairTile pt = pair_tile(shape, t);
        for (int k0 = pt.k0; k0 < pt.k1; k0 += shape.seg) {
          int ok = ptx::wait_parity(&tempty[slot], aphase ^ 1u, abort_flag, err, kTagTmemEmpty, kWaitCycles);
          ok = __shfl_sync(0xffffffffu, ok, 0);
          if (!ok) {
            alive = false;
            break;
          }
          ptx::tc_fence_after();
          const uint32_t d = tmem_base + static_cast<uint32_t>(slot * TN);
          const int k1 = min(pt.k1, k0 + shape.seg);
          for (int k = k0; k < k1; ++k) {
            ok = ptx::wait_parity(&full[sidx], sph, abort_flag, err, kTagFull, kWaitCycles);
            ok = __shfl_sync(0xffffffffu, ok, 0);
            if (!ok) {
              alive = false;
              break;
            }
            const uint32_t s16 = static_cast<uint32_t>(sidx * STAGE) >> 4;
#pragma unroll
            for (int kk = 0; kk < kPairK / 16; ++kk)
              ptx::mma_f16_ss_pair_if(leader, d, a_lo + s16 + kk * AK, a_hi, b_lo + s16 + kk * BK, b_hi, IDESC,
                                      (k > k0 || kk > 0) ? 1u : 0u);
            ptx::mma_commit_pair_if(leader, &empty[sidx]);
            if (++sidx == ST) {
              sidx = 0;
              sph ^= 1u;
            }
          }
          if (!alive) break;
          ptx::mma_commit_pair_if(leader, &tfull[slot]);
          slot ^= 1;
          if (slot == 0) aphase ^= 1u;
        }
      }
      ptx::mma_commit_pair_if(leader, mma_done);
      int dummy = 0;
      ptx::wait_parity(mma_done, 0, reinterpret_cast<volatile int*>(&dummy), err, kTagDrain, kWaitCycles);
      __syncwarp();
    } else if (warp == 1) {
      // the leader's last commit arrives here after all its earlier ones
      int dummy = 0;
      ptx::wait_parity(mma_done, 0, reinterpret_cast<volatile int*>(&dummy), err, kTagDrain, 4 * kWaitCycles);
      __syncwarp();
    }
  } else {
    if constexpr (TN == 256) ptx::registers_up<kPairRegsHigh>();  // the launch checks that there are so many
    // ------------------------------------------------------------ epilogue
    const int q = warp & 3;
    const int part = (warp - kPairEpiFirst) >> 2;  // which kPairEpiCols columns of the tile
    Epi epi(eargs, static_cast<int>(rank) * 128 + q * 32 + lane, part, out + (warp - kPairEpiFirst) * kPairOutBytes);
    const uint32_t lane_addr = static_cast<uint32_t>(q * 32) << 16;
    int slot = 0;
    uint32_t aphase = 0;
    bool alive = true;
    for (int t = first; t < ntiles && alive; t += step) {
      const PairTile pt = pair_tile(shape, t);
      float v[COLS];
      for (int k0 = pt.k0; k0 < pt.k1; k0 += shape.seg) {
        int ok = ptx::wait_parity(&tfull[slot], aphase, abort_flag, err, kTagTmemFull, kWaitCycles);
        ok = __shfl_sync(0xffffffffu, ok, 0);
        if (!ok) {
          alive = false;
          break;
        }
        ptx::tc_fence_after();
        const uint32_t at = tmem_base + lane_addr + static_cast<uint32_t>(slot * TN + part * COLS);
        if (k0 == pt.k0) {
#pragma unroll
          for (int c = 0; c < COLS; c += 32) ptx::tmem_ld32(at + c, v + c);
          ptx::tmem_wait_ld();
        } else {
#pragma unroll
          for (int c = 0; c < COLS; c += 16) {
            float w[16];  // 32 more beside v would not stay in registers
            ptx::tmem_ld16(at + c, w);
            ptx::tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 16; ++j) v[c + j] += w[j];
          }
        }
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive_cluster(ptx::peer_smem_u32(&tempty[slot], 0));
        slot ^= 1;
        if (slot == 0) aphase ^= 1u;
      }
      if (!alive) break;
      epi.tile(pt, v);
    }
    if (alive) epi.done();
  }

  __syncthreads();
  if (rank == 0 && warp == 0 && lane == 0 && *abort_flag) {
    // copies that were issued land before shared memory is given up; a stage that the
    // other CTA never loaded runs into the wait's bound, long after its own copy
    int dummy = 0;
    for (int s = 0; s < ST; ++s)
      if (issued[s])
        ptx::wait_parity(&full[s], static_cast<uint32_t>(issued[s] - 1), reinterpret_cast<volatile int*>(&dummy), err,
                         kTagDrain, kWaitCycles);
  }
  __syncthreads();
  ptx::cluster_sync();  // no barrier or buffer of this CTA is used from the other one any more
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc_pair(tmem_base, TMEM_COLS);
  }
}

// Tensor map of one operand: K-major `rows` x `k`, or MN-major `k` x `rows` (rows of the tile along x).
inline kairo_status pair_operand_map(CUtensorMap* map, const void* base, kairo_dtype dt, bool mn, int64_t rows,
                                     int64_t k, int64_t ld, const char* what, int box_rows = kPairBoxRows) {
  if ((mn ? k : rows) <= 1) ld = static_cast<int64_t>(align_up(static_cast<size_t>(mn ? rows : k), 8));  // one row: any pitch
  const CUtensorMapDataType t = dt == KAIRO_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  return mn ? make_map_2d(map, base, t, 2, static_cast<uint64_t>(rows), static_cast<uint64_t>(k),
                          static_cast<uint64_t>(ld), 64, kPairK, what)
            : make_map_2d(map, base, t, 2, static_cast<uint64_t>(k), static_cast<uint64_t>(rows),
                          static_cast<uint64_t>(ld), kPairK, static_cast<uint32_t>(box_rows), what);
}

// Clusters of a launch of `tiles` tiles.
inline int pair_clusters(int64_t tiles) {
  return static_cast<int>(std::min<int64_t>(tiles, std::max(1, device_sm_count(current_device()) / 2)));
}

template <int IN_FMT, bool A_MN, bool B_MN, class Epi, int TN = kPairTileN>
kairo_status launch_pair_gemm(const CUtensorMap& a, const CUtensorMap& b, const PairShape& shape, unsigned* err,
                              const typename Epi::Args& args, cudaStream_t s) {
  auto* fn = &k_pair_gemm<IN_FMT, A_MN, B_MN, Epi, TN>;
  static std::atomic<uint64_t> ready{0};
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(fn), kPairSmem, &ready);
  if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(max dynamic smem)");
  if constexpr (TN == 256) {
    static std::atomic<int> regs{0};  // a thread's at the launch
    if (regs.load(std::memory_order_relaxed) == 0) {
      cudaFuncAttributes attr;
      e = cudaFuncGetAttributes(&attr, reinterpret_cast<const void*>(fn));
      if (e != cudaSuccess) return cuda_fail(e, "cudaFuncGetAttributes");
      regs.store(attr.numRegs, std::memory_order_relaxed);
    }
    if (regs.load(std::memory_order_relaxed) * kPairThreads < kPairRegsAll)
      return fail(KAIRO_STATUS_NOT_SUPPORTED, "the paired product was compiled for too few registers");
  }
  const int clusters = pair_clusters(static_cast<int64_t>(shape.tiles_m) * shape.tiles_n * shape.splits);
  fn<<<2 * clusters, kPairThreads, kPairSmem, s>>>(a, b, shape, err, args);
  e = cudaGetLastError();
  return e == cudaSuccess ? KAIRO_STATUS_SUCCESS : cuda_fail(e, "launch of the paired tensor-core product");
}

}  // namespace
}  // namespace kairo
