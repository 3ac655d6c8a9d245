// Gated projection of a feed-forward block with block-sparse weights:
//
//   G = X Wg^T,  U = X Wu^T,  H = act(G) * U         X: tokens x k, H: tokens x m
//   dG = dH * U * act'(G),  dU = dH * act(G)         (kairo_gated_linear_grad)
//
// both products, the activation and the product of the two in one kernel: G and
// U never leave the SM.  The backward call forms them again from X (as exact as
// in the forward pass, where copies kept in 16 bits would cost another rounding
// and 2 * tokens * m values) and writes dG and dU side by side as the stacked
// dP of kairo_bsr_sddmm and of the SpMM with the stacked transposed weight:
// block-rows 2i and 2i + 1 of the stacked matrix are block-row i of Wg and of Wu.
//
// Entries.  A block-row's entries are the block-columns where Wg or Wu keeps a
// block, in column order, each with its two stored blocks (-1: none).  Both
// products share the entry's panel of X, the larger operand; a missing block is
// a copy from behind the block storage, which the copy engine fills with zeros.
//
// k_gated (tensor cores).  A cluster of two CTAs takes T * 256 tokens and one
// block-row: an entry is one tcgen05.mma (cta_group::2) per 16 k and 256 tokens with
// M = 256 tokens and N = 2 * BM outputs; the even CTA's shared memory holds
// the gate block, the odd one's the up block, and each holds its own tokens'
// panels of X.  With blocks of 64 an entry costs a CTA 32 KB of X and 8 KB of weights (two
// separate products: 80 KB) and 8 products of 72 cycles.  8192 tokens, 8192 -> 32768 at 20 % of shared
// blocks, moves 17 GB into the SMs: 1.25 ms at the rate that gathers of panels reach by themselves (13.7 TB/s), 1.07
// the products.  It takes 1.6 to 1.7 ms from a cool start (1030 to 1100 TFLOP/s) and 1.80 to 1.86 in a row, where the
// power limit holds the SMs at 1.58 GHz; which role waits for the rest was not measured.  Not kept, all from a cool start
// against 1.6: tiles of 256 tokens (1.95 ms), blocks brought into L2 ahead (1.65), one 32 KB copy of a
// panel instead of four (1.61), other groups of token tiles (1.6 to 1.85).
//
// k_gated_short (33 to 256 tokens; blocks of 64: to 128, or 17 to 256 where they
// have many rows).  The same with one CTA a block-row and two CTAs an SM: a pair
// would multiply and fill panels of 256 tokens, and has half as many places to share
// the block-rows out to.  128 tokens, 4096 -> 14336 at 20 %: 27 us (k_gated 47); 64
// tokens, 8192 -> 32768: 61 us, where the blocks alone are 33 and the L2 hands each
// block-row the panels of its columns.
//
// k_gated_few (up to 32 tokens).  Bound by reading the blocks once.  A CTA takes 16
// rows of a block-row, its warps share out the entries; mma.sync fragments come
// straight from global memory, 16 bytes a lane (the order of k inside a block is
// free as long as both operands agree), and the warps' sums meet in shared memory.
// One token, 8192 -> 32768 at 20 %: 42 us, 5.1 TB/s.  A persistent form that asks
// for the next rows' operands before it joins the sums took 43.
#include <algorithm>

#include "convert.cuh"
#include "internal.h"
#include "ptx.cuh"
#include "tc_common.cuh"

namespace kairo {
namespace {

enum Activation : int {
  kSilu = KAIRO_ACTIVATION_SILU,
  kGelu = KAIRO_ACTIVATION_GELU,
  kGeluTanh = KAIRO_ACTIVATION_GELU_TANH,
  kRelu = KAIRO_ACTIVATION_RELU
};

__device__ __forceinline__ float sigmoid(float x) { return __fdividef(1.f, 1.f + __expf(-x)); }

// act(g), and act'(g) where GRAD.  Every act(0) is 0.
template <bool GRAD>
__device__ __forceinline__ float activate(int act, float g, float& slope) {
  if (act == kSilu) {
    const float s = sigmoid(g);
    if (GRAD) slope = s * (1.f + g * (1.f - s));
    return g * s;
  }
  if (act == kGelu) {
    const float cdf = 0.5f * erfcf(g * -0.70710678118654752f);
    if (GRAD) slope = cdf + g * 0.39894228040143268f * __expf(-0.5f * g * g);
    return g * cdf;
  }
  if (act == kGeluTanh) {
    // 0.5 * (1 + tanh(y)) = sigmoid(2 y), which keeps its digits for negative g
    const float c2 = 1.5957691216057308f;  // 2 * sqrt(2 / pi)
    const float s = sigmoid(c2 * (g + 0.044715f * g * g * g));
    const float t = s * (1.f - s);  // 0 from some |g| on, where g * g may be infinite
    if (GRAD) slope = s + (t == 0.f ? 0.f : g * t * c2 * (1.f + 0.134145f * g * g));
    return g * s;
  }
  if (GRAD) slope = g <= 0.f ? 0.f : 1.f;
  return g <= 0.f ? 0.f : g;  // a NaN stays one
}

struct GatedArgs {
  const int32_t* ent_ptr;  // nbr + 1
  const int4* entries;     // {block-column, gate block or -1, up block or -1, 0}
  const void* blocks;      // stored blocks
  const void* x;
  int64_t ldx;
  void* h;                 // forward
  int64_t ldh;
  const void* dh;          // backward
  int64_t lddh;
  void* dp;                // backward: tokens x (2 * nbr * BM)
  int64_t lddp;
  unsigned* err;
  int32_t n, m, k;
  int32_t nbr, nbc, nentries, nblocks;
  int32_t act;
  int32_t group;           // token tiles visited together
  int32_t vec_h, vec_dh;   // rows may be accessed 16 bytes at a time
};

// N outputs of one token from their sums: H, or dG and dU.
template <typename T, bool GRAD, int N>
__device__ __forceinline__ void gated_out(const GatedArgs& a, int token, int row, int bm, int c0, const float* g,
                                          const float* u) {
  const int first = row * bm + c0;  // output
  if constexpr (!GRAD) {
    float v[N], none = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = activate<false>(a.act, g[j], none) * u[j];
    T* p = static_cast<T*>(a.h) + static_cast<int64_t>(token) * a.ldh + first;
    if (a.vec_h && first + N <= a.m) {
      store_f32<T, N>(p, v);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (first + j < a.m) p[j] = from_f32<T>(v[j]);
    }
  } else {
    float d[N];
    const T* p = static_cast<const T*>(a.dh) + static_cast<int64_t>(token) * a.lddh + first;
    if (a.vec_dh && first + N <= a.m) {
      load_f32<T, N>(p, d);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) d[j] = first + j < a.m ? to_f32<T>(p[j]) : 0.f;
    }
    float dg[N], du[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      float slope = 0.f;
      const float v = activate<true>(a.act, g[j], slope);
      const bool out = first + j < a.m;  // behind the last output both are zero, whatever the blocks hold there
      dg[j] = out ? d[j] * u[j] * slope : 0.f;
      du[j] = out ? d[j] * v : 0.f;
    }
    T* q = static_cast<T*>(a.dp) + static_cast<int64_t>(token) * a.lddp + 2 * row * bm + c0;
    store_f32<T, N>(q, dg);
    store_f32<T, N>(q + bm, du);
  }
}

// ------------------------------------------------------------ tensor cores

constexpr int kGatedThreads = 320;
constexpr int kGatedEpiWarps = 8;
constexpr int kGatedStages = 5;

// Entries of one stage, so that a stage holds 64 k.
constexpr int gated_group(int bm) { return 64 / bm; }
constexpr int gated_block_bytes(int bm) { return (bm * bm * 2 + 1023) / 1024 * 1024; }
constexpr int gated_slot_bytes(int bm, int t) { return t * 128 * bm * 2 + gated_block_bytes(bm); }
constexpr int gated_stage_bytes(int bm, int t) { return gated_group(bm) * gated_slot_bytes(bm, t); }
constexpr size_t gated_smem(int bm, int t) { return static_cast<size_t>(kGatedStages) * gated_stage_bytes(bm, t) + 2048; }

struct GatedItem {
  int tile, row, e0, e1;  // token tile, block-row, entries
  int subs;               // subtiles of the tile
};

template <int BM, int T, int IN_FMT, typename TT, bool GRAD>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kGatedThreads, 1)
    k_gated(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w,
            const GatedArgs args) {
  constexpr int ST = kGatedStages;
  constexpr int E = gated_group(BM);
  constexpr int SLOT = gated_slot_bytes(BM, T);
  constexpr int STAGE = gated_stage_bytes(BM, T);
  constexpr int PANEL = T * 128 * BM * 2;
  constexpr uint32_t IDESC = ptx::make_idesc_f16(IN_FMT, 0u, 0u, 256u, 2 * BM);
  constexpr uint32_t SW = ptx::swizzle_code_for_row_bytes(BM * 2);
  constexpr uint32_t ACC = T * 2 * BM;  // columns of one accumulator
  constexpr uint32_t TMEM_COLS = 2 * ACC < 32 ? 32 : 2 * ACC;
  static_assert(TMEM_COLS <= 512 && (TMEM_COLS & (TMEM_COLS - 1)) == 0, "TMEM columns");

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + ST * STAGE);  // used in the leader
  uint64_t* empty = full + ST;
  uint64_t* tfull = empty + ST;
  uint64_t* tempty = tfull + 2;  // used in the leader
  uint64_t* mma_done = tempty + 2;
  int* misc = reinterpret_cast<int*>(mma_done + 1);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(misc);
  volatile int* abort_flag = misc + 1;
  int* issued = misc + 4;

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
      ptx::mbar_init(&tempty[k], 2 * kGatedEpiWarps);
    }
    ptx::mbar_init(mma_done, 1);
    misc[1] = 0;
    ptx::mbar_init_fence();
  }
  if (warp == 0 && lane == 0) {
    ptx::prefetch_tmap(&tmap_x);
    ptx::prefetch_tmap(&tmap_w);
  }
  __syncthreads();
  ptx::cluster_sync();
  if (warp == 1) {
    ptx::tmem_alloc_pair(tmem_slot, TMEM_COLS);
    ptx::tmem_relinquish_pair();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  // A tile is T subtiles of 256 tokens, 128 of them in each CTA.  What is left of the tokens after the
  // whole tiles is a tile of fewer subtiles, whose items come last.
  constexpr int TOKENS = T * 256;
  const int whole = args.n / TOKENS;
  const int tiles = (args.n + TOKENS - 1) / TOKENS;
  const int nitems = tiles * args.nbr;
  const int first = blockIdx.x >> 1, step = gridDim.x >> 1;
  // `group` token tiles at a time, their block-rows one after the other: the group's X stays in
  // L2 while the weights go by, and a block-row's blocks serve the group's tiles at about the same time.
  auto item = [&](int t) {
    GatedItem it;
    const int per = args.group * args.nbr;
    const int g = t / per, r = t - g * per;
    const int t0 = g * args.group;
    const int gn = min(args.group, whole - t0);
    if (t >= whole * args.nbr) {
      it.row = t - whole * args.nbr;
      it.tile = whole;
      it.subs = (args.n - whole * TOKENS + 255) / 256;
    } else {
      it.row = r / gn;
      it.tile = t0 + (r - it.row * gn);
      it.subs = T;
    }
    // offsets outside the entries are clamped by every role alike
    it.e0 = min(max(__ldg(args.ent_ptr + it.row), 0), args.nentries);
    it.e1 = min(max(__ldg(args.ent_ptr + it.row + 1), it.e0), args.nentries);
    return it;
  };

  if (warp == 0) {
    // ------------------------------------------------------------ loads
    const uint64_t pol_w = ptx::policy_evict_first();
    const uint64_t pol_x = ptx::policy_evict_last();
    constexpr int BOXES = T * 2 + 1;
    static_assert(E * BOXES <= 32, "one lane per copy");
    const void* map_x = &tmap_x;
    const void* map_w = &tmap_w;
    int sidx = 0;
    uint32_t sph = 0;
    bool alive = true;
    auto fetch = [&](const GatedItem& it, int at) {
      const int e = it.e0 + at + lane;
      return e < it.e1 ? __ldg(args.entries + e) : make_int4(0, -1, -1, 0);
    };
    // entries are read a window of 32 ahead of use, the next item's range and first window an item ahead
    GatedItem cur{}, nxt{};
    int4 w0 = make_int4(0, -1, -1, 0), n0 = w0;
    if (first < nitems) {
      cur = item(first);
      w0 = fetch(cur, 0);
    }
    for (int t = first; t < nitems && alive; t += step) {
      const bool more = t + step < nitems;
      n0 = make_int4(0, -1, -1, 0);
      if (more) {
        nxt = item(t + step);
        n0 = fetch(nxt, 0);
      }
      const int cnt = cur.e1 - cur.e0;
      const int y0 = cur.tile * TOKENS + static_cast<int>(rank) * 128;
      const uint32_t bytes = 2u * static_cast<uint32_t>(cur.subs * 128 * BM * 2 + BM * BM * 2);  // of an entry, both CTAs
      for (int at = 0; at < cnt && alive; at += 32) {
        const int4 w = w0;
        if (at + 32 < cnt) w0 = fetch(cur, at + 32);
        int col = w.x, blk = rank == 0 ? w.y : w.z;
        // one number out of range empties the entry in both CTAs
        if (at + lane < cnt && (static_cast<unsigned>(col) >= static_cast<unsigned>(args.nbc) || w.y < -1 ||
                                w.y >= args.nblocks || w.z < -1 || w.z >= args.nblocks)) {
          atomicCAS(args.err, 0u, KAIRO_DEVERR_BAD_INDEX);
          col = 0;
          blk = -1;
        }
        if (blk < 0) blk = args.nblocks;  // behind the storage: zeros
        for (int b0 = 0; b0 < 32 && at + b0 < cnt; b0 += E) {
          const int take = min(E, cnt - at - b0);
          int ok = ptx::wait_parity(&empty[sidx], sph ^ 1u, abort_flag, args.err, kTagEmpty, kWaitCycles);
          ok = __shfl_sync(0xffffffffu, ok, 0);
          if (!ok) {
            alive = false;
            break;
          }
          const uint32_t bar = ptx::peer_smem_u32(&full[sidx], 0);
          if (rank == 0) {
            if (lane == 0) issued[sidx] = static_cast<int>(sph) + 1;
            ptx::mbar_expect_tx_if(lane == 0 ? 1u : 0u, &full[sidx], bytes * static_cast<uint32_t>(take));
          }
          // one lane per box of 64 tokens and per block, so that all copies of a stage are issued at once
          const int e = lane / BOXES, part = lane - e * BOXES;  // entry of the stage; its panel's box, or its block
          const bool is_w = part == BOXES - 1;
          const uint32_t mine = e < take && (is_w || part < 2 * cur.subs) ? 1u : 0u;
          const int ecol = __shfl_sync(0xffffffffu, col, (b0 + e) & 31);
          const int eblk = __shfl_sync(0xffffffffu, blk, (b0 + e) & 31);
          uint8_t* st = smem + sidx * STAGE + (mine ? e : 0) * SLOT;
          ptx::tma_load_2d_pair_if(mine, is_w ? st + PANEL : st + part * (64 * BM * 2), is_w ? map_w : map_x,
                                   is_w ? 0 : ecol * BM, is_w ? eblk * BM : y0 + (part >> 1) * 256 + (part & 1) * 64, bar, is_w ? pol_w : pol_x);
          __syncwarp();
          if (rank == 0) ptx::mbar_arrive_if(lane == 0 ? 1u : 0u, &full[sidx]);
          if (++sidx == ST) {
            sidx = 0;
            sph ^= 1u;
          }
        }
      }
      cur = nxt;
      w0 = n0;
    }
  } else if (warp == 1 && rank == 0) {
    // ------------------------------------------------------------ MMA issuer
    const uint32_t leader = lane == 0 ? 1u : 0u;
    const uint32_t sbase = ptx::smem_u32(smem);
    const uint64_t adesc = ptx::make_smem_desc(sbase, 16, 8 * BM * 2, SW);
    const uint64_t bdesc = ptx::make_smem_desc(sbase + PANEL, 16, 8 * BM * 2, SW);
    const uint32_t a_lo = static_cast<uint32_t>(adesc), a_hi = static_cast<uint32_t>(adesc >> 32);
    const uint32_t b_lo = static_cast<uint32_t>(bdesc), b_hi = static_cast<uint32_t>(bdesc >> 32);
    int sidx = 0, slot = 0;
    uint32_t sph = 0, aphase = 0;
    bool alive = true;
    for (int t = first; t < nitems && alive; t += step) {
      const GatedItem it = item(t);
      const int cnt = it.e1 - it.e0;
      if (cnt == 0) continue;
      int ok = ptx::wait_parity(&tempty[slot], aphase ^ 1u, abort_flag, args.err, kTagTmemEmpty, kWaitCycles);
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (!ok) break;
      ptx::tc_fence_after();
      const uint32_t d = tmem_base + static_cast<uint32_t>(slot) * ACC;
      for (int at = 0; at < cnt; at += E) {
        ok = ptx::wait_parity(&full[sidx], sph, abort_flag, args.err, kTagFull, kWaitCycles);
        ok = __shfl_sync(0xffffffffu, ok, 0);
        if (!ok) {
          alive = false;
          break;
        }
#pragma unroll
        for (int e = 0; e < E; ++e) {
          if (at + e >= cnt) break;
          const uint32_t s16 = static_cast<uint32_t>(sidx * STAGE + e * SLOT) >> 4;
#pragma unroll
          for (int kk = 0; kk < BM / 16; ++kk) {
#pragma unroll
            for (int i = 0; i < T; ++i)
              ptx::mma_f16_ss_pair_if(i < it.subs ? leader : 0u, d + static_cast<uint32_t>(i * 2 * BM),
                                      a_lo + s16 + ((i * 128 * BM * 2 + kk * 32) >> 4), a_hi,
                                      b_lo + s16 + ((kk * 32) >> 4), b_hi, IDESC, (at > 0 || e > 0 || kk > 0) ? 1u : 0u);
          }
        }
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
    ptx::mma_commit_pair_if(leader, mma_done);
    int dummy = 0;
    ptx::wait_parity(mma_done, 0, reinterpret_cast<volatile int*>(&dummy), args.err, kTagDrain, kWaitCycles);
    __syncwarp();
  } else if (warp == 1) {
    // the leader's last commit arrives here after all its earlier ones
    int dummy = 0;
    ptx::wait_parity(mma_done, 0, reinterpret_cast<volatile int*>(&dummy), args.err, kTagDrain, 4 * kWaitCycles);
    __syncwarp();
  } else {
    // ------------------------------------------------------------ epilogue
    constexpr int UN = BM < 32 ? BM : 32;  // outputs of one step
    constexpr int STEPS = T * (BM / UN);
    const int q = warp & 3;
    const int part = (warp - 2) >> 2;
    const uint32_t lane_addr = static_cast<uint32_t>(q * 32) << 16;
    int slot = 0;
    uint32_t aphase = 0;
    for (int t = first; t < nitems; t += step) {
      const GatedItem it = item(t);
      const bool some = it.e1 > it.e0;
      if (some) {
        int ok = ptx::wait_parity(&tfull[slot], aphase, abort_flag, args.err, kTagTmemFull, kWaitCycles);
        ok = __shfl_sync(0xffffffffu, ok, 0);
        if (!ok) break;
        ptx::tc_fence_after();
      }
      const uint32_t at = tmem_base + lane_addr + static_cast<uint32_t>(slot) * ACC;
      for (int s = part; s < STEPS; s += 2) {
        const int i = s / (BM / UN), c0 = (s % (BM / UN)) * UN;
        if (i >= it.subs) break;
        const int token = it.tile * TOKENS + i * 256 + static_cast<int>(rank) * 128 + q * 32 + lane;
        float g[UN], u[UN];
        if (some) {
          if constexpr (UN == 32) {
            ptx::tmem_ld32(at + static_cast<uint32_t>(i * 2 * BM + c0), g);
            ptx::tmem_ld32(at + static_cast<uint32_t>(i * 2 * BM + BM + c0), u);
          } else {
            ptx::tmem_ld16(at + static_cast<uint32_t>(i * 2 * BM + c0), g);
            ptx::tmem_ld16(at + static_cast<uint32_t>(i * 2 * BM + BM + c0), u);
          }
          ptx::tmem_wait_ld();
        } else {
#pragma unroll
          for (int j = 0; j < UN; ++j) g[j] = u[j] = 0.f;
        }
        if (token < args.n) gated_out<TT, GRAD, UN>(args, token, it.row, BM, c0, g, u);
        __syncwarp();
      }
      if (some) {
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive_cluster(ptx::peer_smem_u32(&tempty[slot], 0));
        slot ^= 1;
        if (slot == 0) aphase ^= 1u;
      }
    }
  }

  __syncthreads();
  if (rank == 0 && warp == 0 && lane == 0 && *abort_flag) {
    int dummy = 0;
    for (int s = 0; s < ST; ++s)
      if (issued[s])
        ptx::wait_parity(&full[s], static_cast<uint32_t>(issued[s] - 1), reinterpret_cast<volatile int*>(&dummy),
                         args.err, kTagDrain, kWaitCycles);
  }
  __syncthreads();
  ptx::cluster_sync();
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc_pair(tmem_base, TMEM_COLS);
  }
}

// ------------------------------------------------------------ up to 256 tokens on the tensor cores

constexpr int kShortThreads = 192;
constexpr int kShortEpiWarps = 4;
constexpr int kShortTokens = 128;  // of a subtile; a CTA takes T of them
constexpr int short_slot_bytes(int bm, int t) { return t * kShortTokens * bm * 2 + 2 * bm * bm * 2; }  // X, gate, up
constexpr int short_stage_bytes(int bm, int t) { return gated_group(bm) * short_slot_bytes(bm, t); }
constexpr int short_stages(int bm, int t) { return 100 * 1024 / short_stage_bytes(bm, t); }
constexpr size_t short_smem(int bm, int t) {
  return static_cast<size_t>(short_stages(bm, t)) * short_stage_bytes(bm, t) + 2048;
}
constexpr bool short_fits(int t) {  // twice in an SM
  return 2 * (short_smem(64, t) + 1024) <= 228 * 1024 && 2 * (short_smem(32, t) + 1024) <= 228 * 1024 &&
         2 * (short_smem(16, t) + 1024) <= 228 * 1024;
}
static_assert(short_fits(1) && short_fits(2), "two CTAs of an SM");

// k_gated with one CTA for all tokens of a block-row: M = 128 tokens (64 of them copied where there are no more), N = 2 *
// BM outputs, the gate block's rows followed by the up block's.
template <int BM, int T, int IN_FMT, typename TT, bool GRAD>
__global__ void __launch_bounds__(kShortThreads, 2)
    k_gated_short(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w,
                  const GatedArgs args) {
  constexpr int ST = short_stages(BM, T);
  constexpr int E = gated_group(BM);
  constexpr int SLOT = short_slot_bytes(BM, T);
  constexpr int STAGE = short_stage_bytes(BM, T);
  constexpr int PANEL = T * kShortTokens * BM * 2;
  constexpr uint32_t IDESC = ptx::make_idesc_f16(IN_FMT, 0u, 0u, kShortTokens, 2 * BM);
  constexpr uint32_t SW = ptx::swizzle_code_for_row_bytes(BM * 2);
  constexpr uint32_t ACC = T * 2 * BM;
  constexpr int SLOTS = 2 * ACC <= 256 ? 2 : 1;  // accumulators: half the columns of an SM are this CTA's
  constexpr uint32_t TMEM_COLS = SLOTS * ACC;
  static_assert(SLOT % 1024 == 0 && PANEL % 1024 == 0 && TMEM_COLS >= 32 && TMEM_COLS <= 256, "layout");

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + ST * STAGE);
  uint64_t* empty = full + ST;
  uint64_t* tfull = empty + ST;
  uint64_t* tempty = tfull + 2;
  uint64_t* mma_done = tempty + 2;
  int* misc = reinterpret_cast<int*>(mma_done + 1);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(misc);
  volatile int* abort_flag = misc + 1;
  int* issued = misc + 4;  // [ST]: parity + 1 of the last load into each stage

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      ptx::mbar_init(&full[s], 1);
      ptx::mbar_init(&empty[s], 1);
      issued[s] = 0;
    }
    for (int k = 0; k < SLOTS; ++k) {
      ptx::mbar_init(&tfull[k], 1);
      ptx::mbar_init(&tempty[k], kShortEpiWarps);
    }
    ptx::mbar_init(mma_done, 1);
    misc[1] = 0;
    ptx::mbar_init_fence();
  }
  if (warp == 0 && lane == 0) {
    ptx::prefetch_tmap(&tmap_x);
    ptx::prefetch_tmap(&tmap_w);
  }
  if (warp == 1) {
    ptx::tmem_alloc(tmem_slot, TMEM_COLS);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  // entries of a block-row; offsets outside them are clamped by every role alike
  auto first_of = [&](int row) { return min(max(__ldg(args.ent_ptr + row), 0), args.nentries); };
  auto end_of = [&](int row, int e0) { return min(max(__ldg(args.ent_ptr + row + 1), e0), args.nentries); };

  if (warp == 0) {
    // ------------------------------------------------------------ loads
    const uint64_t pol_w = ptx::policy_evict_first();
    const uint64_t pol_x = ptx::policy_evict_last();
    constexpr int BOXES = 2 * T + 2;  // of 64 tokens, the gate block, the up block
    static_assert(E * BOXES <= 32, "one lane per copy");
    const int xboxes = (args.n + 63) / 64;
    const int e = lane / BOXES, part = lane - e * BOXES;
    const bool is_w = part >= 2 * T;
    const uint32_t bytes = static_cast<uint32_t>(xboxes * 64 * BM * 2 + 2 * BM * BM * 2);  // of an entry
    const uint32_t dst_off =
        static_cast<uint32_t>((e < E ? e : 0) * SLOT + (is_w ? PANEL + (part - 2 * T) * BM * BM * 2 : part * 64 * BM * 2));
    const void* map = is_w ? static_cast<const void*>(&tmap_w) : static_cast<const void*>(&tmap_x);
    const uint64_t pol = is_w ? pol_w : pol_x;
    int sidx = 0;
    uint32_t sph = 0;
    bool alive = true;
    for (int row = blockIdx.x; row < args.nbr && alive; row += gridDim.x) {
      const int e0 = first_of(row), cnt = end_of(row, e0) - e0;
      for (int at = 0; at < cnt && alive; at += 32) {
        const int4 w = at + lane < cnt ? __ldg(args.entries + e0 + at + lane) : make_int4(0, -1, -1, 0);
        int col = w.x, gate = w.y, up = w.z;
        if (at + lane < cnt && (static_cast<unsigned>(col) >= static_cast<unsigned>(args.nbc) || gate < -1 ||
                                gate >= args.nblocks || up < -1 || up >= args.nblocks)) {
          atomicCAS(args.err, 0u, KAIRO_DEVERR_BAD_INDEX);
          col = 0;
          gate = up = -1;
        }
        if (gate < 0) gate = args.nblocks;  // behind the storage: zeros
        if (up < 0) up = args.nblocks;
        for (int b0 = 0; b0 < 32 && at + b0 < cnt; b0 += E) {
          const int take = min(E, cnt - at - b0);
          int ok = ptx::wait_parity(&empty[sidx], sph ^ 1u, abort_flag, args.err, kTagEmpty, kWaitCycles);
          ok = __shfl_sync(0xffffffffu, ok, 0);
          if (!ok) {
            alive = false;
            break;
          }
          if (lane == 0) issued[sidx] = static_cast<int>(sph) + 1;
          ptx::mbar_expect_tx_if(lane == 0 ? 1u : 0u, &full[sidx], bytes * static_cast<uint32_t>(take));
          __syncwarp();
          const uint32_t mine = e < take && (is_w || part < xboxes) ? 1u : 0u;
          const int src = (b0 + e) & 31;
          const int ecol = __shfl_sync(0xffffffffu, col, src);
          const int egate = __shfl_sync(0xffffffffu, gate, src);
          const int eup = __shfl_sync(0xffffffffu, up, src);
          ptx::tma_load_2d_if(mine, smem + sidx * STAGE + dst_off, map, is_w ? 0 : ecol * BM,
                              is_w ? (part == 2 * T ? egate : eup) * BM : part * 64, &full[sidx], pol);
          __syncwarp();
          ptx::mbar_arrive_if(lane == 0 ? 1u : 0u, &full[sidx]);
          if (++sidx == ST) {
            sidx = 0;
            sph ^= 1u;
          }
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    const uint32_t leader = lane == 0 ? 1u : 0u;
    const int subs = (args.n + kShortTokens - 1) / kShortTokens;
    const uint32_t sbase = ptx::smem_u32(smem);
    const uint64_t adesc = ptx::make_smem_desc(sbase, 16, 8 * BM * 2, SW);
    const uint64_t bdesc = ptx::make_smem_desc(sbase + PANEL, 16, 8 * BM * 2, SW);
    const uint32_t a_lo = static_cast<uint32_t>(adesc), a_hi = static_cast<uint32_t>(adesc >> 32);
    const uint32_t b_lo = static_cast<uint32_t>(bdesc), b_hi = static_cast<uint32_t>(bdesc >> 32);
    int sidx = 0, slot = 0;
    uint32_t sph = 0, aphase = 0;
    bool alive = true;
    for (int row = blockIdx.x; row < args.nbr && alive; row += gridDim.x) {
      const int e0 = first_of(row), cnt = end_of(row, e0) - e0;
      if (cnt == 0) continue;
      int ok = ptx::wait_parity(&tempty[slot], aphase ^ 1u, abort_flag, args.err, kTagTmemEmpty, kWaitCycles);
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (!ok) break;
      ptx::tc_fence_after();
      const uint32_t d = tmem_base + static_cast<uint32_t>(slot) * ACC;
      for (int at = 0; at < cnt; at += E) {
        ok = ptx::wait_parity(&full[sidx], sph, abort_flag, args.err, kTagFull, kWaitCycles);
        ok = __shfl_sync(0xffffffffu, ok, 0);
        if (!ok) {
          alive = false;
          break;
        }
        ptx::tc_fence_after();
#pragma unroll
        for (int e = 0; e < E; ++e) {
          if (at + e >= cnt) break;
          const uint32_t s16 = static_cast<uint32_t>(sidx * STAGE + e * SLOT) >> 4;
#pragma unroll
          for (int kk = 0; kk < BM / 16; ++kk) {
#pragma unroll
            for (int i = 0; i < T; ++i)
              ptx::mma_f16_ss_if(i < subs ? leader : 0u, d + static_cast<uint32_t>(i * 2 * BM),
                                 a_lo + s16 + ((i * kShortTokens * BM * 2 + kk * 32) >> 4), a_hi,
                                 b_lo + s16 + ((kk * 32) >> 4), b_hi, IDESC, (at > 0 || e > 0 || kk > 0) ? 1u : 0u);
          }
        }
        ptx::mma_commit_if(leader, &empty[sidx]);
        if (++sidx == ST) {
          sidx = 0;
          sph ^= 1u;
        }
      }
      if (!alive) break;
      ptx::mma_commit_if(leader, &tfull[slot]);
      if (++slot == SLOTS) {
        slot = 0;
        aphase ^= 1u;
      }
    }
    ptx::mma_commit_if(leader, mma_done);
    int dummy = 0;
    ptx::wait_parity(mma_done, 0, reinterpret_cast<volatile int*>(&dummy), args.err, kTagDrain, kWaitCycles);
    __syncwarp();
  } else {
    // ------------------------------------------------------------ epilogue
    constexpr int UN = BM < 32 ? BM : 32;  // outputs of one step
    const int q = warp & 3;
    const uint32_t lane_addr = static_cast<uint32_t>(q * 32) << 16;
    int slot = 0;
    uint32_t aphase = 0;
    for (int row = blockIdx.x; row < args.nbr; row += gridDim.x) {
      const int e0 = first_of(row);
      const bool some = end_of(row, e0) > e0;
      if (some) {
        int ok = ptx::wait_parity(&tfull[slot], aphase, abort_flag, args.err, kTagTmemFull, kWaitCycles);
        ok = __shfl_sync(0xffffffffu, ok, 0);
        if (!ok) break;
        ptx::tc_fence_after();
      }
      const uint32_t at = tmem_base + lane_addr + static_cast<uint32_t>(slot) * ACC;
#pragma unroll 1
      for (int s = 0; s < T * (BM / UN); ++s) {
        const int i = s / (BM / UN), c0 = (s % (BM / UN)) * UN;
        const int token0 = i * kShortTokens + q * 32, token = token0 + lane;
        if (token0 >= args.n) break;
        const uint32_t here = at + static_cast<uint32_t>(i * 2 * BM + c0);
        float g[UN], u[UN];
        if (some) {
          if constexpr (UN == 32) {
            ptx::tmem_ld32(here, g);
            ptx::tmem_ld32(here + BM, u);
          } else {
            ptx::tmem_ld16(here, g);
            ptx::tmem_ld16(here + BM, u);
          }
          ptx::tmem_wait_ld();
        } else {
#pragma unroll
          for (int j = 0; j < UN; ++j) g[j] = u[j] = 0.f;
        }
        if (token < args.n) gated_out<TT, GRAD, UN>(args, token, row, BM, c0, g, u);
        __syncwarp();
      }
      if (some) {
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&tempty[slot]);
        if (++slot == SLOTS) {
          slot = 0;
          aphase ^= 1u;
        }
      }
    }
  }

  __syncthreads();
  if (threadIdx.x == 0 && *abort_flag) {
    // copies that were issued land before shared memory is given up
    int dummy = 0;
    for (int s = 0; s < ST; ++s)
      if (issued[s])
        ptx::wait_parity(&full[s], static_cast<uint32_t>(issued[s] - 1), reinterpret_cast<volatile int*>(&dummy),
                         args.err, kTagDrain, kWaitCycles);
  }
  __syncthreads();
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

// ------------------------------------------------------------ few tokens

template <typename T>
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_16816<__half>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                  uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma_16816<__nv_bfloat16>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 8 * C values of one row that lane t of a quad takes, in C pieces of 16 bytes (blocks of 64: C = 2; 32: 1),
// or the 4 of a 16-wide block's row.  `w` holds them as pairs.
template <int BM>
struct RowPart {
  static constexpr int WORDS = BM / 8;  // 32-bit words a lane takes of a row
  uint32_t w[WORDS];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) w[i] = 0u;
  }
  // `row` points at the row's first value, 16-byte aligned
  __device__ __forceinline__ void load(const uint16_t* row, int t) {
    if constexpr (BM == 16) {
      const uint2 v = __ldg(reinterpret_cast<const uint2*>(row) + t);
      w[0] = v.x;
      w[1] = v.y;
    } else {
#pragma unroll
      for (int c = 0; c < BM / 32; ++c) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(row) + c * 4 + t);
        w[4 * c] = v.x;
        w[4 * c + 1] = v.y;
        w[4 * c + 2] = v.z;
        w[4 * c + 3] = v.w;
      }
    }
  }
  // the same of a row that ends after `left` values, value by value
  __device__ __forceinline__ void load_edge(const uint16_t* row, int t, int left) {
    constexpr int V = BM == 16 ? 4 : 8;
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
      const int at = (2 * i / V) * 4 * V + t * V + 2 * i % V;
      const uint32_t lo = at < left ? row[at] : 0u, hi = at + 1 < left ? row[at + 1] : 0u;
      w[i] = lo | (hi << 16);
    }
  }
};

constexpr int kFewWarps = 8;

// NT * 8 tokens; grid: one CTA per 16 rows of a block-row.
template <int BM, int NT, typename T, bool GRAD>
__global__ void __launch_bounds__(32 * kFewWarps, NT == 1 ? 3 : 2) k_gated_few(const GatedArgs a, int vec_x) {
  constexpr int SLICES = BM / 16;
  __shared__ float sums[kFewWarps][2][NT * 8][17];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int gid = lane >> 2, t = lane & 3;
  const int row = blockIdx.x / SLICES, slice = blockIdx.x % SLICES;
  const int e0 = min(max(__ldg(a.ent_ptr + row), 0), a.nentries);
  const int e1 = min(max(__ldg(a.ent_ptr + row + 1), e0), a.nentries);
  float g[NT][4], u[NT][4];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) g[i][j] = u[i][j] = 0.f;
  const uint16_t* blocks = static_cast<const uint16_t*>(a.blocks) + (slice * 16 + gid) * BM;
  const uint16_t* x = static_cast<const uint16_t*>(a.x);
  struct Step {
    RowPart<BM> g0, g1, u0, u1, xs[NT];
  };
  // A warp's entries are read once, one a lane.  The operands of an entry are under way while the one
  // before it is multiplied, unless the registers of both would cost a resident CTA.
  constexpr bool AHEAD = BM < 64 || NT == 2;
  for (int base = e0; base < e1; base += 32 * kFewWarps) {
    const int mine = base + warp + lane * kFewWarps;
    int4 w = make_int4(0, -1, -1, 0);
    if (mine < e1) w = __ldg(a.entries + mine);
    if (static_cast<unsigned>(w.x) >= static_cast<unsigned>(a.nbc) || w.y < -1 || w.y >= a.nblocks || w.z < -1 ||
        w.z >= a.nblocks) {
      atomicCAS(a.err, 0u, KAIRO_DEVERR_BAD_INDEX);
      w = make_int4(0, -1, -1, 0);
    }
    const int cnt = max(0, min(32, (e1 - base - warp + kFewWarps - 1) / kFewWarps));
    auto load = [&](Step& s, int j) {
      const int col = __shfl_sync(0xffffffffu, w.x, j), gb = __shfl_sync(0xffffffffu, w.y, j),
                ub = __shfl_sync(0xffffffffu, w.z, j);
      if (gb >= 0) {
        const uint16_t* p = blocks + static_cast<int64_t>(gb) * BM * BM;
        s.g0.load(p, t);
        s.g1.load(p + 8 * BM, t);
      } else {
        s.g0.zero();
        s.g1.zero();
      }
      if (ub >= 0) {
        const uint16_t* p = blocks + static_cast<int64_t>(ub) * BM * BM;
        s.u0.load(p, t);
        s.u1.load(p + 8 * BM, t);
      } else {
        s.u0.zero();
        s.u1.zero();
      }
      const int left = a.k - col * BM;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const int token = i * 8 + gid;
        const uint16_t* p = x + static_cast<int64_t>(token) * a.ldx + col * BM;
        if (token >= a.n) s.xs[i].zero();
        else if (vec_x && left >= BM) s.xs[i].load(p, t);
        else s.xs[i].load_edge(p, t, left);
      }
    };
    auto multiply = [&](const Step& s) {
#pragma unroll
      for (int q = 0; q < BM / 16; ++q)
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          const uint32_t x0 = s.xs[i].w[2 * q], x1 = s.xs[i].w[2 * q + 1];
          mma_16816<T>(g[i], s.g0.w[2 * q], s.g1.w[2 * q], s.g0.w[2 * q + 1], s.g1.w[2 * q + 1], x0, x1);
          mma_16816<T>(u[i], s.u0.w[2 * q], s.u1.w[2 * q], s.u0.w[2 * q + 1], s.u1.w[2 * q + 1], x0, x1);
        }
    };
    if constexpr (AHEAD) {
      Step s0, s1;
      if (cnt > 0) load(s0, 0);
      for (int j = 0; j < cnt; j += 2) {
        if (j + 1 < cnt) load(s1, j + 1);
        multiply(s0);
        if (j + 1 < cnt) {
          if (j + 2 < cnt) load(s0, j + 2);
          multiply(s1);
        }
      }
    } else {
      for (int j = 0; j < cnt; ++j) {
        Step s0;
        load(s0, j);
        multiply(s0);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int token = i * 8 + 2 * t + (j & 1), r = gid + (j >> 1) * 8;
      sums[warp][0][token][r] = g[i][j];
      sums[warp][1][token][r] = u[i][j];
    }
  __syncthreads();
  for (int o = threadIdx.x; o < NT * 8 * 16; o += 32 * kFewWarps) {
    const int token = o >> 4, r = o & 15;
    if (token >= a.n) break;
    float gs = 0.f, us = 0.f;
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) {
      gs += sums[w][0][token][r];
      us += sums[w][1][token][r];
    }
    gated_out<T, GRAD, 1>(a, token, row, BM, slice * 16 + r, &gs, &us);
  }
}

// ------------------------------------------------------------ host side

constexpr int kAnyTokens = 8;   // up to here X may have any alignment
constexpr int kFewTokens = 32;
constexpr int kShortRows = 192;  // block-rows

template <int BM, int NT, typename T, bool GRAD>
void launch_few(const GatedArgs& a, cudaStream_t s) {
  const int vec_x = reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && (a.ldx % 8 == 0 || a.n <= 1);
  k_gated_few<BM, NT, T, GRAD><<<a.nbr * (BM / 16), 32 * kFewWarps, 0, s>>>(a, vec_x);
}

template <int BM, typename TT, int IN_FMT, bool GRAD>
kairo_status run_gated(GatedArgs a, cudaStream_t s) {
  // Fragments up to 32 tokens, or up to 16 where blocks of 64 have rows enough for the SMs: 32768 x 8192 at 20 %
  // twice (the blocks alone 33 us), 16 / 32 tokens 64 / 82 us by fragments, 59 / 59 by k_gated_short; 14336 x 4096
  // (224 block-rows) 23 / 29 and 25 / 25; 4096 x 4096 (64) 10 / 12 and 21 / 21.  Blocks of 32 and 16, 14336 x 4096,
  // 32 tokens: 31 and 39, by k_gated_short 33 and 70.  Between 33 and 256 tokens k_gated takes 47, 85 and 206 us
  // (blocks of 64, 32, 16); k_gated_short 27, 37 and 84 up to 128, and 45, 61 and 133 up to 256, where 4096 x 4096 in
  // blocks of 64 takes 37 us (k_gated 23).
  const bool rows = BM == 64 && a.nbr >= kShortRows;
  if (a.n <= (rows ? kFewTokens / 2 : kFewTokens)) {
    if (a.n <= 8) launch_few<BM, 1, TT, GRAD>(a, s);
    else if (a.n <= 16) launch_few<BM, 2, TT, GRAD>(a, s);
    else if (a.n <= 24) launch_few<BM, 3, TT, GRAD>(a, s);
    else launch_few<BM, 4, TT, GRAD>(a, s);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? KAIRO_STATUS_SUCCESS : cuda_fail(e, "launch of k_gated_few");
  }
  const CUtensorMapDataType dt = IN_FMT == 0 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  auto few = [&](auto tc) -> kairo_status {
    constexpr int T = decltype(tc)::value;
    CUtensorMap mx, mw;
    kairo_status st = make_map_2d(&mx, a.x, dt, 2, static_cast<uint64_t>(a.k), static_cast<uint64_t>(a.n),
                                  static_cast<uint64_t>(a.ldx), BM, 64, "X");
    if (st == KAIRO_STATUS_SUCCESS)
      st = make_map_2d(&mw, a.blocks, dt, 2, BM, static_cast<uint64_t>(a.nblocks) * BM, BM, BM, BM,
                       "block storage");
    if (st) return st;
    auto* fn = &k_gated_short<BM, T, IN_FMT, TT, GRAD>;
    static std::atomic<uint64_t> ready{0};
    cudaError_t e = allow_smem(reinterpret_cast<const void*>(fn), short_smem(BM, T), &ready);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(max dynamic smem)");
    const int grid = std::min(a.nbr, 2 * device_sm_count(current_device()));
    fn<<<grid, kShortThreads, short_smem(BM, T), s>>>(mx, mw, a);
    e = cudaGetLastError();
    return e == cudaSuccess ? KAIRO_STATUS_SUCCESS : cuda_fail(e, "launch of k_gated_short");
  };
  if (a.n <= kShortTokens) return few(std::integral_constant<int, 1>{});
  if (a.n <= 2 * kShortTokens && (BM < 64 || rows)) return few(std::integral_constant<int, 2>{});
  auto go = [&](auto tc) -> kairo_status {
    constexpr int T = decltype(tc)::value;
    CUtensorMap mx, mw;
    kairo_status st = make_map_2d(&mx, a.x, dt, 2, static_cast<uint64_t>(a.k), static_cast<uint64_t>(a.n),
                                  static_cast<uint64_t>(a.ldx), BM, 64, "X");
    if (st == KAIRO_STATUS_SUCCESS)
      st = make_map_2d(&mw, a.blocks, dt, 2, BM, static_cast<uint64_t>(a.nblocks) * BM, BM, BM, BM,
                       "block storage");
    if (st) return st;
    auto* fn = &k_gated<BM, T, IN_FMT, TT, GRAD>;
    static std::atomic<uint64_t> ready{0};
    cudaError_t e = allow_smem(reinterpret_cast<const void*>(fn), gated_smem(BM, T), &ready);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(max dynamic smem)");
    const int tiles = static_cast<int>(ceil_div64(a.n, T * 256));
    // a group's X takes about a quarter of the L2
    a.group = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(std::max(1, a.n / (T * 256)), (32LL << 20) / (static_cast<int64_t>(T) * 512 * a.k))));
    const int64_t items = static_cast<int64_t>(tiles) * a.nbr;
    const int clusters = static_cast<int>(std::min<int64_t>(items, std::max(1, device_sm_count(current_device()) / 2)));
    fn<<<2 * clusters, kGatedThreads, gated_smem(BM, T), s>>>(mx, mw, a);
    e = cudaGetLastError();
    return e == cudaSuccess ? KAIRO_STATUS_SUCCESS : cuda_fail(e, "launch of k_gated");
  };
  if constexpr (BM == 64) {
    if (a.n <= 256) return go(std::integral_constant<int, 1>{});
  }
  return go(std::integral_constant<int, 2>{});
}

template <bool GRAD>
kairo_status dispatch_gated(const GatedArgs& a, int bm, kairo_dtype dt, cudaStream_t s) {
  if (dt == KAIRO_DTYPE_F16) {
    if (bm == 16) return run_gated<16, __half, 0, GRAD>(a, s);
    if (bm == 32) return run_gated<32, __half, 0, GRAD>(a, s);
    return run_gated<64, __half, 0, GRAD>(a, s);
  }
  if (bm == 16) return run_gated<16, __nv_bfloat16, 1, GRAD>(a, s);
  if (bm == 32) return run_gated<32, __nv_bfloat16, 1, GRAD>(a, s);
  return run_gated<64, __nv_bfloat16, 1, GRAD>(a, s);
}

bool row_vec(const void* p, int64_t ld, int64_t rows) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (ld % 8 == 0 || rows <= 1);
}

kairo_status gated_check(const kairo_gated* w, const void* x, int64_t ldx, int64_t n, int32_t act, const void* err) {
  if (!w) return fail(KAIRO_STATUS_INVALID_VALUE, "null weight descriptor");
  if (w->rows < 0 || w->cols < 0 || w->nentries < 0 || w->nblocks < 0 || n < 0)
    return fail(KAIRO_STATUS_INVALID_VALUE, "invalid size");
  if (w->block != 16 && w->block != 32 && w->block != 64)
    return fail(KAIRO_STATUS_NOT_SUPPORTED, "the gated projection takes square blocks of 16, 32 or 64");
  if (w->dtype != KAIRO_DTYPE_F16 && w->dtype != KAIRO_DTYPE_BF16)
    return fail(KAIRO_STATUS_NOT_SUPPORTED, "the gated projection takes f16 or bf16");
  if (w->rows > 0x3fffff00LL || w->cols > 0x7fffff00LL || n > 0x7fffff00LL || w->nentries > 0x7fffffffLL ||
      (w->nblocks + 1) * w->block > 0x7fffffffLL ||
      ceil_div64(n, 256) * ceil_div64(w->rows, w->block) > 0x7fffffffLL)
    return fail(KAIRO_STATUS_NOT_SUPPORTED, "sizes beyond 32-bit coordinates");
  if (act < kSilu || act > kRelu) return fail(KAIRO_STATUS_INVALID_VALUE, "unknown activation");
  if (ldx < w->cols) return fail(KAIRO_STATUS_INVALID_VALUE, "leading dimension too small");
  if (n == 0 || w->rows == 0) return KAIRO_STATUS_SUCCESS;
  if (!w->ent_ptr || !err || (w->nentries > 0 && (!w->entries || !w->blocks || !x)))
    return fail(KAIRO_STATUS_INVALID_VALUE, "null pointer argument");
  // a missing block is a copy from behind the storage, which needs a block in front
  if (w->nentries > 0 && w->nblocks == 0) return fail(KAIRO_STATUS_INVALID_VALUE, "entries without a stored block");
  if (reinterpret_cast<uintptr_t>(w->entries) % 16 || reinterpret_cast<uintptr_t>(w->blocks) % 16)
    return fail(KAIRO_STATUS_INVALID_VALUE, "entries and blocks must be 16-byte aligned");
  if (n > kAnyTokens && w->nentries > 0 && !row_vec(x, ldx, n))
    return fail(KAIRO_STATUS_INVALID_VALUE, "X must have 16-byte aligned rows");
  return KAIRO_STATUS_SUCCESS;
}

GatedArgs gated_args(const kairo_gated* w, const void* x, int64_t ldx, int64_t n, int32_t act, unsigned* err) {
  GatedArgs a{};
  a.ent_ptr = w->ent_ptr;
  a.entries = reinterpret_cast<const int4*>(w->entries);
  a.blocks = w->blocks;
  a.x = x;
  a.ldx = ldx;
  a.err = err;
  a.n = static_cast<int32_t>(n);
  a.m = static_cast<int32_t>(w->rows);
  a.k = static_cast<int32_t>(w->cols);
  a.nbr = static_cast<int32_t>(ceil_div64(w->rows, w->block));
  a.nbc = static_cast<int32_t>(ceil_div64(w->cols, w->block));
  a.nentries = static_cast<int32_t>(w->nentries);
  a.nblocks = static_cast<int32_t>(w->nblocks);
  a.act = act;
  return a;
}

}  // namespace
}  // namespace kairo

using namespace kairo;

extern "C" kairo_status kairo_gated_linear(const kairo_gated* w, const void* x, int64_t ldx, int64_t n,
                                           int32_t activation, void* h, int64_t ldh, unsigned* error_word,
                                           void* stream) {
  kairo_status st = gated_check(w, x, ldx, n, activation, error_word);
  if (st) return st;
  if (ldh < w->rows) return fail(KAIRO_STATUS_INVALID_VALUE, "leading dimension too small");
  if (n == 0 || w->rows == 0) return KAIRO_STATUS_SUCCESS;
  if (!h) return fail(KAIRO_STATUS_INVALID_VALUE, "null pointer argument");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (w->nentries == 0) {
    const cudaError_t e = cudaMemset2DAsync(h, static_cast<size_t>(ldh) * 2, 0, static_cast<size_t>(w->rows) * 2,
                                            static_cast<size_t>(n), s);
    return e == cudaSuccess ? KAIRO_STATUS_SUCCESS : cuda_fail(e, "cudaMemset2DAsync(H)");
  }
  GatedArgs a = gated_args(w, x, ldx, n, activation, error_word);
  a.h = h;
  a.ldh = ldh;
  a.vec_h = row_vec(h, ldh, n);
  return dispatch_gated<false>(a, w->block, w->dtype, s);
}

extern "C" kairo_status kairo_gated_linear_grad(const kairo_gated* w, const void* x, int64_t ldx, int64_t n,
                                                int32_t activation, const void* dh, int64_t lddh, void* dp,
                                                int64_t lddp, unsigned* error_word, void* stream) {
  kairo_status st = gated_check(w, x, ldx, n, activation, error_word);
  if (st) return st;
  const int64_t stacked = 2 * ceil_div64(w->rows, w->block) * w->block;
  if (lddh < w->rows || lddp < stacked || lddp % 8)
    return fail(KAIRO_STATUS_INVALID_VALUE, "leading dimension too small, or that of dP no multiple of 8");
  if (n == 0 || w->rows == 0) return KAIRO_STATUS_SUCCESS;
  if (!dh || !dp) return fail(KAIRO_STATUS_INVALID_VALUE, "null pointer argument");
  if (reinterpret_cast<uintptr_t>(dp) % 16) return fail(KAIRO_STATUS_INVALID_VALUE, "dP must be 16-byte aligned");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (w->nentries == 0) {
    const cudaError_t e = cudaMemset2DAsync(dp, static_cast<size_t>(lddp) * 2, 0, static_cast<size_t>(stacked) * 2,
                                            static_cast<size_t>(n), s);
    return e == cudaSuccess ? KAIRO_STATUS_SUCCESS : cuda_fail(e, "cudaMemset2DAsync(dP)");
  }
  GatedArgs a = gated_args(w, x, ldx, n, activation, error_word);
  a.dh = dh;
  a.lddh = lddh;
  a.vec_dh = row_vec(dh, lddh, n);
  a.dp = dp;
  a.lddp = lddp;
  return dispatch_gated<true>(a, w->block, w->dtype, s);
}
