// Kernels of the low-rank adapters (adapters.cu has the mathematics and the
// entry points).
//
// Both are bound by memory: per token and feature they do 2 * rank operations
// on 2 bytes read (rank 16: 16 operations a byte, where the machine does 250),
// so they use warp-level matrix instructions fed straight from global memory
// and spend their design on wide loads, few launches and many bytes in flight.
//
// Fragments without shared memory.  A 16 x 8 x 16 product does not care which
// feature stands at which place of its contraction or of its columns, as long
// as both operands agree:
//  - contraction over features (low = X down^T): lane (g, t) = (lane / 4,
//    lane % 4) takes 16 contiguous bytes, features 8 t .. 8 t + 7 of its row, as
//    the contraction places 2t, 2t+1, 2t+8, 2t+9 of two products, for tokens
//    and rank rows alike;
//  - features as columns (low up, and the weight gradients): lane (g, t)
//    takes 8 contiguous features of the rank rows (tokens) 2t, 2t+1, 2t+8,
//    2t+9 as column g of eight products, and so holds of the result the 8
//    features of column 2t and those of column 2t+1, for its rows.
// Every access is a 16-byte vector, and the features of the columns are dealt
// out so that the four lanes t of one access stand side by side: 64 bytes of a
// row, whole sectors.  (With columns 2t and 2t+1 side by side instead, each
// access touched half sectors, and the rank-16 expansion of 8192 x 8192 took 91
// us where it now takes 56.)
//
// low is an fp32 value.  For a product with 16-bit weights it is split into
// terms of the weights' type, each the rounding of what the ones before leave:
// two for 16-bit results (rest at most 2^-17 of it), three for fp32 results
// (2^-23).  In fp16, whose range is narrow, it is first scaled by a power of
// two (exact) that brings the largest of the row to [1, 2), and the rest is
// one of that largest (2^-25 of it at least, a term's smallest step).  An infinity
// in low, or in what it is multiplied by, spoils what it enters: of its terms some
// are zero or of the other sign, so that the sum is NaN where it would be infinite.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "convert.cuh"
#include "internal.h"
#include "q8.cuh"

namespace kairo {

// One work item of the plan: up to 16, 32 or 64 tokens of one adapter.
struct LowRankTile {
  int32_t adapter;  // -1: tokens without one
  int32_t begin;    // first position in the order
  int32_t count;
  int32_t pad;
};

struct LowRankApplyArgs {
  const void* x;
  const void* down;
  const void* up;
  const void* base;   // null: zero
  void* y;            // null: low alone
  float* low;         // null: not stored
  const float* scale; // null: 1
  const int32_t* order;
  const LowRankTile* tiles;
  const int32_t* ntiles;
  int64_t ldx, ldb, ldy;
  int32_t k, n, rank;
  int32_t base_f32;
};

// One or two weight gradients of one launch.
struct LowRankWgradArgs {
  struct One {
    const float* s;      // (tokens, rank)
    const void* z;       // (tokens, k), or null when given in 8 bits:
    const int8_t* codes;
    const float* steps;
    void* grad;          // (adapters, rank, k)
    int64_t ldz, ldq, lds;
    int32_t k;
  } one[2];
  const int32_t* order;
  const int32_t* starts;
  int64_t tokens;
  int32_t rank;
  int32_t count;
  int32_t widest;        // largest k
};

// Launches (adapters_bf16.cu, adapters_f16.cu).  `tile` is 16, 32 or 64 tokens,
// `clusters` the bound on the number of tiles, `cluster` CTAs per tile.
template <typename T>
cudaError_t launch_low_rank_apply(const LowRankApplyArgs& a, bool y_f32, bool vec, int tile, int64_t clusters,
                                  int cluster, cudaStream_t s);
template <typename T>
cudaError_t launch_low_rank_wgrad(const LowRankWgradArgs& a, bool grad_f32, bool vec, int64_t adapters, int cluster,
                                  cudaStream_t s);

namespace lowrank {

constexpr int kWarps = 8;
constexpr int kThreadsPerCta = kWarps * 32;
constexpr int kChunk = 64;  // tokens per staged chunk of the weight gradient
// Features up to which the matrix units add up a contraction by themselves, in
// up to kContractSteps steps of 32 features a warp.  They truncate, always
// towards zero: up to 1e-7 of the sum in each of the two products of a step, and
// 1.1e-5 after 131072 features of one sign.  Longer contractions (LONG) are cut
// into parts of that many steps, added with rounding; 2^22 features came to
// 3.9e-4 in one sum.  (In one kernel for both, the registers that this takes
// made the short ones spill.)
constexpr int kContractSteps = 64;
constexpr int kLongFeatures = kContractSteps * 32 * kWarps * 8;  // clusters of 8 from 131072 features on
static_assert(kContractSteps % 2 == 0, "two steps to a turn of 64 features");

__device__ __forceinline__ uint32_t smem_addr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t peer_addr(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
constexpr int kMaxCluster = 8;

// The sum over the cluster, in rank order, of the value (or four) at the same
// shared address of every CTA.  The loads are issued together, so that the
// latency of a peer's memory is paid once and not for each of eight.
__device__ __forceinline__ float peer_sum(uint32_t addr, uint32_t csize) {
  float v[kMaxCluster];
#pragma unroll
  for (uint32_t c = 0; c < kMaxCluster; ++c) {
    v[c] = 0.f;
    if (c < csize) asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v[c]) : "r"(peer_addr(addr, c)));
  }
  float s = v[0];
#pragma unroll
  for (uint32_t c = 1; c < kMaxCluster; ++c) s += v[c];
  return s;
}
__device__ __forceinline__ float4 peer_sum4(uint32_t addr, uint32_t csize) {
  float4 v[kMaxCluster];
#pragma unroll
  for (uint32_t c = 0; c < kMaxCluster; ++c) {
    v[c] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (c < csize)
      asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                   : "=f"(v[c].x), "=f"(v[c].y), "=f"(v[c].z), "=f"(v[c].w)
                   : "r"(peer_addr(addr, c)));
  }
  float4 s = v[0];
#pragma unroll
  for (uint32_t c = 1; c < kMaxCluster; ++c) {
    s.x += v[c].x;
    s.y += v[c].y;
    s.z += v[c].z;
    s.w += v[c].w;
  }
  return s;
}
__device__ __forceinline__ void peer_store(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}

template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same_v<T, __nv_bfloat16>) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

__device__ __forceinline__ uint32_t word(const uint4& v, int i) {
  return i == 0 ? v.x : (i == 1 ? v.y : (i == 2 ? v.z : v.w));
}

// Element j (0..7) of two 16-byte vectors as one pair.
__device__ __forceinline__ uint32_t pair_of(const uint4& lo, const uint4& hi, int j) {
  return __byte_perm(word(lo, j >> 1), word(hi, j >> 1), (j & 1) ? 0x7632 : 0x5410);
}

template <typename T>
__device__ __forceinline__ uint16_t bits16(float v) {
  const T h = from_f32<T>(v);
  return *reinterpret_cast<const uint16_t*>(&h);
}
template <typename T>
__device__ __forceinline__ uint32_t bits16x2(float v0, float v1) {
  if constexpr (std::is_same_v<T, __half>) {
    const __half2 h = __floats2half2_rn(v0, v1);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(v0, v1);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
template <typename T>
__device__ __forceinline__ float value16(uint16_t b) {
  return to_f32<T>(*reinterpret_cast<const T*>(&b));
}

// 2^-e and 2^e with 2^e <= m < 2^(e+1), within what fp32 can hold; 1 for zero
// and for infinities and NaN.
__device__ __forceinline__ void power_scale(float m, float* down, float* up) {
  int e = static_cast<int>(__float_as_uint(m) >> 23) - 127;
  if (!(m > 0.f) || e == 128) e = 0;
  e = max(-126, min(126, e));
  *down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
  *up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
}

// ---------------------------------------------------------------- apply

// A lane's own shared memory as an extension of its registers: asynchronous
// copies land where the same lane reads them, so that many loads are in flight
// without registers to hold them and without any barrier.  Vector i of a slot
// stands at [i][lane].
template <typename T>
__device__ __forceinline__ void fetch(uint32_t dst, const T* p, int left) {
  // no byte is read where left <= 0; 16 zero bytes are written
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(p), "r"(left > 0 ? 16 : 0) : "memory");
}
// Place in a 512-byte vector slot of the 16 bytes that are chunk `c` of the 128
// bytes of row `t`: a row is written as one (in lane order, a copy of four rows
// took 16 passes over the banks instead of 4, and the weight gradient 46 us
// where it now takes 29), and whole sectors of the rows change places so that
// lanes that read together meet different banks.
__device__ __forceinline__ uint32_t by_rows(int c, int t) {
  return static_cast<uint32_t>(t * 8 + (c ^ (2 * t))) * 16u;
}
// The same for the 8 codes that are chunk `c` of the 64 codes of row `t`.
__device__ __forceinline__ uint32_t codes_by_rows(int c, int t) {
  return static_cast<uint32_t>(t * 8 + (c ^ (4 * (t >> 1)))) * 8u;
}
// Operands at any address of their type (VEC false): the same slots, filled by
// the whole warp value by value, a row at a time, so that an access meets one
// line of one row (with every lane loading its own 8 values one by one it met
// eight; 4431 tokens, 1776 -> 8734, rank 16: 249 -> 160 us.  Asynchronous copies of
// aligned words, shifted when they are read, took 121 there, but 70 instead of 54
// for 2349 tokens at rank 32 and 10.4 instead of 8.7 for one token).  What a lane
// reads was then written by others: a warp barrier stands between filling and
// reading, and between reading and the next filling.
// CONST: nothing writes the operand during the launch (base may be y).
template <typename T, bool CONST = true>
__device__ __forceinline__ uint32_t value_at(const T* row, int c, int n) {
  using Bits = std::conditional_t<sizeof(T) == 2, uint16_t, uint32_t>;
  if (c >= n) return 0u;
  const Bits* p = reinterpret_cast<const Bits*>(row) + c;
  return CONST ? __ldg(p) : *p;
}
__device__ __forceinline__ void put16(uint32_t dst, uint32_t v) {
  asm volatile("st.shared.u16 [%0], %1;" ::"r"(dst), "h"(static_cast<uint16_t>(v)) : "memory");
}
__device__ __forceinline__ void put32(uint32_t dst, uint32_t v) {
  asm volatile("st.shared.u32 [%0], %1;" ::"r"(dst), "r"(v) : "memory");
}
__device__ __forceinline__ uint4 landed(uint32_t src) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(src)
               : "memory");
  return v;
}
__device__ __forceinline__ uint2 landed_codes(uint32_t src) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(src) : "memory");
  return v;
}

__device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void wait_all_but() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Tile shape and memory of one instance.  MT x 16 tokens, NT x 8 rank rows;
// STAGES steps of 32 features in flight in the contraction.  ALIAS: the warps'
// partial tiles take the ring's place while they are summed, which makes room
// for twice the tokens at ranks above 32; the expansion's loads then start behind
// that sum.
template <int MT_, int NT_, int STAGES_, bool ALIAS_ = false>
struct ApplyShape {
  static constexpr int MT = MT_, NT = NT_, STAGES = STAGES_;
  static constexpr bool ALIAS = ALIAS_;
  static constexpr int ROWS = 16 * MT;
  static constexpr int RP = 8 * NT;          // rank, padded
  static constexpr int PITCH = RP + 8;       // 16-bit terms: rows 16 bytes apart in banks
  static constexpr int LOW = ROWS * RP;      // floats of one low tile
  static constexpr int KT = NT / 2;          // rank steps of 16
  static constexpr int STEP = 2 * MT + NT;   // vectors of one contraction step
  // Vectors per lane: the contraction's steps, or one turn of the expansion
  // (4 for each rank step of up; 4 for the base rows of 16 tokens, 8 in fp32).
  static constexpr int ring(bool base_f32) {
    const int e = 4 * KT + (base_f32 ? 8 : 4) * MT;
    return STAGES * STEP > e ? STAGES * STEP : e;
  }
  static constexpr size_t ring_bytes(bool base_f32) { return static_cast<size_t>(kWarps) * ring(base_f32) * 512; }
  // Floats of the warps' partial tiles; afterwards, with operands at any
  // address, 8 rows of 64 results of every warp on their way out.
  static constexpr int out_pitch(int y_bytes) { return 64 * y_bytes + 16; }
  static constexpr int red(int y_bytes, bool vec) {
    const int tiles = (ALIAS ? 1 : kWarps / 2) * LOW, out = kWarps * 8 * out_pitch(y_bytes) / 4;
    return vec || tiles > out ? tiles : out;
  }
  static constexpr size_t bytes(int terms, bool base_f32, int y_bytes, bool vec) {
    const size_t tiles = static_cast<size_t>(red(y_bytes, vec)) + LOW;
    return ring_bytes(base_f32) + (tiles + ROWS) * 4 + static_cast<size_t>(terms) * ROWS * PITCH * 2;
  }
};

// One cluster per tile.  Its CTAs and warps share out the features of the
// contraction, 64 at a time; partial low tiles meet in shared memory, then over
// the cluster's distributed shared memory; each CTA gets the whole low tile
// and its warps share out the output features, 64 at a time.  One launch, low
// never travels through global memory.  The loads of the expansion (up and
// base) are started before the tile is summed, so that the barriers cost no
// memory time; afterwards each load of the next turn starts as soon as its slot
// has been read.
template <typename T, typename TY, typename S, int TERMS, bool BASE_F32, bool VEC, bool LONG, int MINB>
__global__ void __launch_bounds__(kThreadsPerCta, MINB) k_apply(const LowRankApplyArgs a) {
  constexpr int MT = S::MT, NT = S::NT, KT = S::KT;
  constexpr int RING = S::ring(BASE_F32);
  extern __shared__ __align__(16) uint8_t smem[];
  static_assert(!S::ALIAS || S::ring_bytes(BASE_F32) >= kWarps / 2 * S::LOW * 4, "partial tiles fit in the ring");
  float* part = reinterpret_cast<float*>(smem + S::ring_bytes(BASE_F32));  // [LOW]: this CTA's partial tile
  float* red = S::ALIAS ? reinterpret_cast<float*>(smem) : part;  // [kWarps / 2][LOW]
  float* low = part + S::red(sizeof(TY), VEC);                   // [LOW]: the whole tile
  float* row_up = low + S::LOW;                                  // [ROWS]: power of two of every row (fp16)
  uint16_t* terms = reinterpret_cast<uint16_t*>(row_up + S::ROWS);  // [TERMS][ROWS][PITCH]

  const uint32_t crank = cluster_rank(), csize = cluster_size();
  const int64_t ti = blockIdx.x / csize;
  if (ti >= *a.ntiles) return;  // the whole cluster
  const LowRankTile tile = a.tiles[ti];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int slot = static_cast<int>(crank) * kWarps + warp;      // this warp among the cluster's
  const int stride = static_cast<int>(csize) * kWarps * 64;      // features between a warp's turns
  const int count = min(tile.count, S::ROWS);
  const uint32_t ring0 = smem_addr(smem) + static_cast<uint32_t>(warp * RING * 512);
  const uint32_t ring = ring0 + static_cast<uint32_t>(lane * 16);  // rows by g: the lanes t side by side
  const int up_chunk = 4 * (g & 1) + (g >> 1);  // the 8 features of a turn of 64 that are this lane's columns
  const uint32_t up_ring = ring0 + by_rows(up_chunk, t);
  const bool live = tile.adapter >= 0;
  int tok[MT][2];  // tokens of this lane's rows, -1: none
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = m * 16 + h * 8 + g;
      tok[m][h] = row < count ? a.order[tile.begin + row] : -1;
    }

  float acc[MT][NT][4];
  // Sum over the CTA's warps, into the first, as a tree: the upper half hands over to the lower.
  auto sum_warps = [&]() {
#pragma unroll
    for (int half = kWarps / 2; half >= 1; half /= 2) {
      if (warp >= half && warp < 2 * half) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              red[(warp - half) * S::LOW + ((m * NT + j) * 4 + i) * 32 + lane] = acc[m][j][i];
      }
      __syncthreads();
      if (warp < half) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[m][j][i] += red[warp * S::LOW + ((m * NT + j) * 4 + i) * 32 + lane];
      }
      __syncthreads();
    }
  };
  int parts = 1;  // of the contraction (LONG)
  auto steps_from = [&](int first) { return first < a.k ? 2 * ((a.k - first + stride - 1) / stride) : 0; };
  if (live) {
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[m][j][i] = 0.f;
    // Steps of 32 features, two to a turn of 64; `rest`: with those of later parts.
    int rest = steps_from(slot * 64);
    int steps = LONG ? min(rest, kContractSteps) : rest;
    const int most = steps_from(static_cast<int>(crank) * kWarps * 64);  // of the CTA's first warp: the same for all
    int kk = slot * 64 + 8 * t;  // this lane's features of the next step to start
    const T* wrow = static_cast<const T*>(a.down) + (static_cast<int64_t>(tile.adapter) * a.rank + g) * a.k;
    const int64_t wstep = static_cast<int64_t>(8) * a.k;
    const T* xrow[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        xrow[m][h] = static_cast<const T*>(a.x) + static_cast<int64_t>(max(tok[m][h], 0)) * a.ldx;
    auto issue = [&](int i, int at) {
      if (i < steps) {
        if constexpr (VEC) {
          const int left = a.k - kk;
          const int off = left > 0 ? kk : 0;
          const uint32_t dst = ring + static_cast<uint32_t>(at * S::STEP * 512);
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            const bool there = j * 8 + g < a.rank;
            fetch<T>(dst + j * 512, wrow + (there ? j * wstep + off : off - g * static_cast<int64_t>(a.k)),
                     there ? left : 0);
          }
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              fetch<T>(dst + (NT + 2 * m + h) * 512, xrow[m][h] + off, tok[m][h] >= 0 ? left : 0);
        } else {
          static_assert(MT == 1, "two vectors of tokens");
          constexpr int UW = 4;  // vectors under way: two took 9.1 us for one token, 661 -> 114, four 8.7
          const int c = kk - 8 * t + lane;
          const T* w0 = static_cast<const T*>(a.down) + static_cast<int64_t>(tile.adapter) * a.rank * a.k;
          const uint32_t dst = ring0 + static_cast<uint32_t>(at * S::STEP * 512 + lane * 2);
#pragma unroll
          for (int v0 = 0; v0 < S::STEP; v0 += UW) {
            uint32_t v[UW][8];
#pragma unroll
            for (int u = 0; u < UW; ++u)
#pragma unroll
              for (int r = 0; r < 8; ++r) {
                if (v0 + u >= S::STEP) {
                  v[u][r] = 0u;
                } else if (v0 + u < NT) {
                  const int rr = (v0 + u) * 8 + r;
                  v[u][r] = rr < a.rank ? value_at<T>(w0 + static_cast<int64_t>(rr) * a.k, c, a.k) : 0u;
                } else {
                  const int tk = __shfl_sync(0xffffffffu, tok[0][v0 + u - NT], 4 * r);
                  v[u][r] = tk >= 0 ? value_at<T>(static_cast<const T*>(a.x) + static_cast<int64_t>(tk) * a.ldx, c, a.k)
                                    : 0u;
                }
              }
#pragma unroll
            for (int u = 0; u < UW; ++u)
#pragma unroll
              for (int r = 0; r < 8; ++r)
                if (v0 + u < S::STEP) put16(dst + (v0 + u) * 512 + r * 64, v[u][r]);
          }
        }
        kk += (i & 1) ? stride - 32 : 32;
      }
      commit();
    };
    for (;;) {
#pragma unroll
      for (int i = 0; i < S::STAGES; ++i) issue(i, i);
      int at = 0;
      for (int i = 0; i < steps; ++i) {
        wait_all_but<S::STAGES - 1>();
        if constexpr (!VEC) __syncwarp();
        const uint32_t src = ring + static_cast<uint32_t>(at * S::STEP * 512);
        uint4 wb[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) wb[j] = landed(src + j * 512);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const uint4 x0 = landed(src + (NT + 2 * m) * 512), x1 = landed(src + (NT + 2 * m + 1) * 512);
          const uint32_t a0[4] = {x0.x, x1.x, x0.y, x1.y};
          const uint32_t a1[4] = {x0.z, x1.z, x0.w, x1.w};
#pragma unroll
          for (int j = 0; j < NT; ++j) mma<T>(acc[m][j], a0, wb[j].x, wb[j].y);
#pragma unroll
          for (int j = 0; j < NT; ++j) mma<T>(acc[m][j], a1, wb[j].z, wb[j].w);
        }
        if constexpr (!VEC) __syncwarp();
        issue(i + S::STAGES, at);  // every vector of the slot is in use above
        at = at + 1 == S::STAGES ? 0 : at + 1;
      }
      if (!LONG || parts * kContractSteps >= most) break;
      // The whole CTA's sum so far is kept where the finished tile will stand:
      // no peer writes there before the cluster's barrier.
      wait_all_but<0>();
      __syncthreads();
      sum_warps();
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float* kept = low + ((m * NT + j) * 4 + i) * 32 + lane;
            if (warp == 0) *kept = parts > 1 ? *kept + acc[m][j][i] : acc[m][j][i];
            acc[m][j][i] = 0.f;
          }
      ++parts;
      rest -= kContractSteps;
      steps = min(rest, kContractSteps);
    }
  }

  // Loads of a turn of the expansion, in the order of their use: one unit of up
  // for each rank step, one of base for each 16 tokens (two in fp32).  Unit u
  // has the slot of its own; a turn that does not exist, a tile without an
  // adapter and a missing base fill theirs with zeros and read nothing.
  constexpr int BU = BASE_F32 ? 2 : 1;
  constexpr int UNITS = KT + BU * MT;
  const T* up = static_cast<const T*>(a.up) + static_cast<int64_t>(max(tile.adapter, 0)) * a.rank * a.n;
  auto issue_up = [&](int n0, int kt) {
    if constexpr (VEC) {
      const int c = n0 + 8 * up_chunk, left = live && c < a.n ? a.n - c : 0;
      const uint32_t dst = up_ring + static_cast<uint32_t>(kt * 4 * 512);
      const T* col = live ? up + (left > 0 ? c : 0) : static_cast<const T*>(a.x);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = kt * 16 + 2 * t + (i & 1) + (i >> 1) * 8;
        const bool there = live && r < a.rank;
        fetch<T>(dst + i * 512, col + (there ? r * static_cast<int64_t>(a.n) : 0), there ? left : 0);
      }
    } else if (live) {
      // value `lane` and `lane` + 32 of row 2 q + .. of each vector
      const uint32_t dst = ring0 + static_cast<uint32_t>(kt * 4 * 512 + 2 * (lane & 7));
      uint32_t v[4][4][2];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            const int r = kt * 16 + 2 * q + (i & 1) + (i >> 1) * 8;
            v[i][q][s] = r < a.rank ? value_at<T>(up + static_cast<int64_t>(r) * a.n, n0 + lane + 32 * s, a.n) : 0u;
          }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int s = 0; s < 2; ++s) put16(dst + i * 512 + by_rows((lane >> 3) + 4 * s, q), v[i][q][s]);
    }
    commit();
  };
  auto issue_base = [&](int n0, int m, int b) {  // m and b are known when compiled
    const uint32_t dst = (VEC ? ring : ring0) + static_cast<uint32_t>((KT + BU * m + b) * 4 * 512);
    if constexpr (!VEC) {
      constexpr int ROWS_OF = BASE_F32 ? 1 : 2;  // halves of the tokens in this unit
#pragma unroll
      for (int h0 = 0; h0 < ROWS_OF; ++h0) {
        const int mine = a.base ? tok[m][BASE_F32 ? b : h0] : -1;
        uint32_t v[8][2];
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const int tk = __shfl_sync(0xffffffffu, mine, 4 * r);
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            const int c = n0 + 32 * s + lane;
            if constexpr (BASE_F32)
              v[r][s] = tk >= 0 ? value_at<float, false>(
                                      static_cast<const float*>(a.base) + static_cast<int64_t>(tk) * a.ldb, c, a.n)
                                : 0u;
            else
              v[r][s] = tk >= 0 ? value_at<T, false>(static_cast<const T*>(a.base) + static_cast<int64_t>(tk) * a.ldb, c,
                                                     a.n)
                                : 0u;
          }
        }
#pragma unroll
        for (int r = 0; r < 8; ++r)
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            if constexpr (BASE_F32)
              put32(dst + (2 * s + ((lane >> 2) & 1)) * 512 + (4 * r + (lane >> 3)) * 16 + (lane & 3) * 4, v[r][s]);
            else
              put16(dst + (2 * h0 + s) * 512 + r * 64 + lane * 2, v[r][s]);
          }
      }
    } else if constexpr (BASE_F32) {
      const int tk = a.base ? tok[m][b] : -1;
      const float* row = tk >= 0 ? static_cast<const float*>(a.base) + static_cast<int64_t>(tk) * a.ldb
                                 : reinterpret_cast<const float*>(a.x);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = n0 + 32 * (i >> 1) + 8 * t + 4 * (i & 1);
        const int left = tk >= 0 ? a.n - c : 0;
        fetch<float>(dst + i * 512, row + (left > 0 ? c : 0), left);
      }
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int tk = a.base ? tok[m][h] : -1;
        const T* row = tk >= 0 ? static_cast<const T*>(a.base) + static_cast<int64_t>(tk) * a.ldb
                               : static_cast<const T*>(a.x);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int c = n0 + 32 * q + 8 * t;
          const int left = tk >= 0 ? a.n - c : 0;
          fetch<T>(dst + (2 * h + q) * 512, row + (left > 0 ? c : 0), left);
        }
      }
    }
    commit();
  };
  auto start_turn = [&]() {
    if (!a.y) return;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) issue_up(slot * 64, kt);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int b = 0; b < BU; ++b) issue_base(slot * 64, m, b);
  };
  if (!S::ALIAS || !live) start_turn();

  if (live) {
    if constexpr (S::ALIAS) {
      wait_all_but<0>();  // of the empty groups: every copy has been used
      __syncthreads();
    }
    sum_warps();
    if (S::ALIAS) start_turn();  // the ring is free again
    if (warp == 0) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          if (LONG && parts > 1) {
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[m][j][i] += low[((m * NT + j) * 4 + i) * 32 + lane];
          }
          float* to = part + (m * 16 + g) * S::RP + j * 8 + 2 * t;
          *reinterpret_cast<float2*>(to) = make_float2(acc[m][j][0], acc[m][j][1]);
          *reinterpret_cast<float2*>(to + 8 * S::RP) = make_float2(acc[m][j][2], acc[m][j][3]);
        }
    }
    cluster_sync();
    // Each CTA sums its share of the tile over the cluster, in rank order, and
    // gives the result to all.
    const float scale = a.scale ? a.scale[tile.adapter] : 1.f;
    const uint32_t part_addr = smem_addr(part), low_addr = smem_addr(low);
    const int share = (S::LOW + static_cast<int>(csize) - 1) / static_cast<int>(csize);
    const int i0 = static_cast<int>(crank) * share, i1 = min(S::LOW, i0 + share);
    for (int i = i0 + threadIdx.x; i < i1; i += kThreadsPerCta) {
      const float v = peer_sum(part_addr + 4u * i, csize) * scale;
      for (uint32_t c = 0; c < csize; ++c) peer_store(peer_addr(low_addr + 4u * i, c), v);
      const int row = i / S::RP, r = i - row * S::RP;
      if (a.low && row < count && r < a.rank)
        a.low[static_cast<int64_t>(a.order[tile.begin + row]) * a.rank + r] = v;
    }
    cluster_sync();
  } else if (a.low && crank == 0) {
    for (int i = threadIdx.x; i < count * a.rank; i += kThreadsPerCta) {
      const int row = i / a.rank;
      a.low[static_cast<int64_t>(a.order[tile.begin + row]) * a.rank + (i - row * a.rank)] = 0.f;
    }
  }
  if (!a.y) return;

  if (live) {
    if constexpr (std::is_same_v<T, __half>) {
      for (int row = warp; row < S::ROWS; row += kWarps) {
        uint32_t m = 0;
        for (int r = lane; r < S::RP; r += 32) m = max(m, __float_as_uint(low[row * S::RP + r]) & 0x7fffffffu);
        m = __reduce_max_sync(0xffffffffu, m);
        float dn, sc;
        power_scale(__uint_as_float(m), &dn, &sc);
        for (int r = lane; r < S::RP; r += 32) low[row * S::RP + r] *= dn;
        if (lane == 0) row_up[row] = sc;
      }
      __syncthreads();
    }
    for (int i = threadIdx.x; i < S::LOW; i += kThreadsPerCta) {
      const int row = i / S::RP, r = i - row * S::RP;
      float v = low[i];
#pragma unroll
      for (int q = 0; q < TERMS; ++q) {
        const uint16_t b = bits16<T>(v);
        terms[(q * S::ROWS + row) * S::PITCH + r] = b;
        v -= value16<T>(b);
      }
    }
    __syncthreads();
  }

  TY* y = static_cast<TY*>(a.y);
  // ldmatrix: lane l names row l % 16 and rank half l / 16 of a 16 x 16 tile.
  const uint32_t terms_addr = smem_addr(terms) + static_cast<uint32_t>((lane & 15) * S::PITCH + (lane >> 4) * 8) * 2u;
  for (int n0 = slot * 64; n0 < a.n; n0 += stride) {
    const int later = n0 + stride;
    uint32_t b0[KT][8], b1[KT][8];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      wait_all_but<UNITS - 1>();
      if constexpr (!VEC) __syncwarp();
      const uint32_t src = up_ring + static_cast<uint32_t>(kt * 4 * 512);
      const uint4 v0 = landed(src), v1 = landed(src + 512), v2 = landed(src + 1024), v3 = landed(src + 1536);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        b0[kt][j] = pair_of(v0, v1, j);
        b1[kt][j] = pair_of(v2, v3, j);
      }
      if constexpr (!VEC) __syncwarp();
      issue_up(later, kt);
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      float out[2][16];  // rows g and g + 8: features n0 + 8 t .., n0 + 32 + 8 t ..
#pragma unroll
      for (int b = 0; b < BU; ++b) {
        wait_all_but<UNITS - 1>();
        if constexpr (!VEC) __syncwarp();
        const uint32_t src = ring + static_cast<uint32_t>((KT + BU * m + b) * 4 * 512);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint4 v = landed(src + i * 512);
          if constexpr (BASE_F32) {
            out[b][4 * i] = __uint_as_float(v.x);
            out[b][4 * i + 1] = __uint_as_float(v.y);
            out[b][4 * i + 2] = __uint_as_float(v.z);
            out[b][4 * i + 3] = __uint_as_float(v.w);
          } else {
#pragma unroll
            for (int q = 0; q < 8; ++q)
              out[i >> 1][(i & 1) * 8 + q] = value16<T>(static_cast<uint16_t>(word(v, q >> 1) >> (16 * (q & 1))));
          }
        }
        if constexpr (!VEC) __syncwarp();
        issue_base(later, m, b);
      }
      if (m * 16 >= count) continue;  // the same for the whole cluster
      if (live) {
        float d[8][4];
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) d[j][i] = 0.f;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
          for (int q = TERMS - 1; q >= 0; --q) {
            uint32_t f[4];
            ldmatrix4(f, terms_addr + static_cast<uint32_t>((q * S::ROWS + m * 16) * S::PITCH + kt * 16) * 2u);
#pragma unroll
            for (int j = 0; j < 8; ++j) mma<T>(d[j], f, b0[kt][j], b1[kt][j]);
          }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float p = 1.f;
          if constexpr (std::is_same_v<T, __half>) p = row_up[m * 16 + h * 8 + g];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            out[h][j] += d[j][2 * h] * p;
            out[h][8 + j] += d[j][2 * h + 1] * p;
          }
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if constexpr (VEC) {
          if (tok[m][h] < 0) continue;
          TY* to = y + static_cast<int64_t>(tok[m][h]) * a.ldy;
          constexpr int W = 16 / static_cast<int>(sizeof(TY));  // features per 16 bytes
#pragma unroll
          for (int q = 0; q < 16 / W; ++q) {
            const int c = n0 + 32 * (W * q / 8) + 8 * t + W * q % 8;
            if (c < a.n) {
              float f[W];
#pragma unroll
              for (int i = 0; i < W; ++i) f[i] = out[h][W * q + i];
              store_f32<TY, W>(to + c, f);
            }
          }
        } else {
          // 8 rows through the shared memory of the partial tiles, then row by row
          constexpr int P = S::out_pitch(sizeof(TY));
          uint8_t* rows = reinterpret_cast<uint8_t*>(part) + warp * 8 * P;
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            float f[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = out[h][8 * q + i];
            store_f32<TY, 8>(reinterpret_cast<TY*>(rows + g * P) + 32 * q + 8 * t, f);
          }
          __syncwarp();
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            const int tk = __shfl_sync(0xffffffffu, tok[m][h], 4 * r);
            if (tk < 0) break;  // the rows behind the tile's last
            const TY* from = reinterpret_cast<const TY*>(rows + r * P);
#pragma unroll
            for (int s = 0; s < 2; ++s) {
              const int c = n0 + 32 * s + lane;
              if (c < a.n) y[static_cast<int64_t>(tk) * a.ldy + c] = from[32 * s + lane];
            }
          }
          __syncwarp();
        }
      }
    }
  }
}

// cudaFuncSetAttribute once per device and instance.
template <typename F>
cudaError_t allow_smem(F* fn, size_t bytes, std::atomic<uint64_t>* done) {
  if (bytes <= 48 * 1024) return cudaSuccess;
  const int dev = current_device();
  const uint64_t bit = uint64_t(1) << (dev & 63);
  if (dev >= 0 && dev < 64 && (done->load(std::memory_order_relaxed) & bit)) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
  if (e == cudaSuccess && dev >= 0 && dev < 64) done->fetch_or(bit, std::memory_order_relaxed);
  return e;
}

template <typename T, typename TY, typename S, bool BASE_F32, bool VEC, bool LONG = false>
cudaError_t launch_apply_as(const LowRankApplyArgs& a, int64_t clusters, int cluster, cudaStream_t s) {
  constexpr int TERMS = std::is_same_v<TY, float> ? 3 : 2;
  constexpr size_t bytes = S::bytes(TERMS, BASE_F32, sizeof(TY), VEC);
  static_assert(bytes <= 227 * 1024, "shared memory of one CTA");
  constexpr int MINB = bytes <= 113 * 1024 ? 2 : 1;
  auto* fn = &k_apply<T, TY, S, TERMS, BASE_F32, VEC, LONG, MINB>;
  static std::atomic<uint64_t> done{0};
  cudaError_t e = allow_smem(fn, bytes, &done);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(clusters * cluster));
  cfg.blockDim = dim3(kThreadsPerCta);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = s;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = static_cast<unsigned>(cluster);
  at.val.clusterDim.y = 1;
  at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, fn, a);
}

template <typename T, typename TY, typename S, bool VEC>
cudaError_t launch_apply(const LowRankApplyArgs& a, int64_t clusters, int cluster, cudaStream_t s) {
  static_assert(S::MT == 1, "the shapes of 16 tokens");
  if (a.k > kLongFeatures)
    return a.base_f32 ? launch_apply_as<T, TY, S, true, VEC, true>(a, clusters, cluster, s)
                      : launch_apply_as<T, TY, S, false, VEC, true>(a, clusters, cluster, s);
  return a.base_f32 ? launch_apply_as<T, TY, S, true, VEC>(a, clusters, cluster, s)
                    : launch_apply_as<T, TY, S, false, VEC>(a, clusters, cluster, s);
}

template <typename T, typename TY>
cudaError_t pick_apply(const LowRankApplyArgs& a, bool vec, int tile, int64_t clusters, int cluster, cudaStream_t s) {
  using R16 = ApplyShape<1, 2, 4>;
  using R32 = ApplyShape<1, 4, 2>;
  using R64 = ApplyShape<1, 8, 2>;
  using R128 = ApplyShape<1, 16, 2>;
  if (!vec) {
    if (a.rank <= 16) return launch_apply<T, TY, R16, false>(a, clusters, cluster, s);
    if (a.rank <= 32) return launch_apply<T, TY, R32, false>(a, clusters, cluster, s);
    if (a.rank <= 64) return launch_apply<T, TY, R64, false>(a, clusters, cluster, s);
    return launch_apply<T, TY, R128, false>(a, clusters, cluster, s);
  }
  // the tall tiles: 16-bit bases, but for 32 tokens at rank 64
  if (a.rank <= 16)
    return tile == 64 ? launch_apply_as<T, TY, ApplyShape<4, 2, 2>, false, true>(a, clusters, cluster, s)
                      : launch_apply<T, TY, R16, true>(a, clusters, cluster, s);
  if (a.rank <= 32)
    return tile == 32 ? launch_apply_as<T, TY, ApplyShape<2, 4, 2>, false, true>(a, clusters, cluster, s)
                      : launch_apply<T, TY, R32, true>(a, clusters, cluster, s);
  if (a.rank <= 64)
    return tile == 64   ? launch_apply_as<T, TY, ApplyShape<4, 8, 2, true>, false, true>(a, clusters, cluster, s)
           : tile == 32 ? launch_apply_as<T, TY, ApplyShape<2, 8, 3>, true, true>(a, clusters, cluster, s)
                        : launch_apply<T, TY, R64, true>(a, clusters, cluster, s);
  return tile == 32 ? launch_apply_as<T, TY, ApplyShape<2, 16, 2, true>, false, true>(a, clusters, cluster, s)
                    : launch_apply<T, TY, R128, true>(a, clusters, cluster, s);
}

// ---------------------------------------------------------------- weight gradient

// Tile shape and memory of one instance.  A warp owns MR x 16 rank rows and 64
// features; RG warps side by side cover the rank, kWarps / RG column groups
// the CTA's features; UNITS steps of 16 tokens in flight.  From rank 17 on a
// warp takes 32 rank rows and the registers of two CTAs: each z value read by
// half as many warps is worth more than twice the warps (8192 tokens, 8192
// features, 4 adapters: rank 32 54 -> 44 us, 64 130 -> 86, 128 293 -> 202).
template <int RG_, int MR_, int UNITS_>
struct WgradShape {
  static constexpr int RG = RG_, MR = MR_, UNITS = UNITS_;
  static constexpr int RP = 16 * RG * MR;
  static constexpr int PITCH = RP + 8;
  static constexpr int COLS = 64 * (kWarps / RG);
  static constexpr int PER_THREAD = kChunk * RP / kThreadsPerCta;  // s values of a chunk
  static constexpr size_t RING_BYTES = static_cast<size_t>(kWarps) * UNITS * 4 * 512;
  static constexpr size_t PART_BYTES = static_cast<size_t>(RP) * COLS * 4;
  static constexpr size_t SHARED_BYTES = RING_BYTES > PART_BYTES ? RING_BYTES : PART_BYTES;
  static constexpr size_t bytes(int terms, bool half, bool q8) {
    return SHARED_BYTES + (q8 ? static_cast<size_t>(2 * kChunk * (COLS / 64)) * 4 : 0) +
           static_cast<size_t>(2 * RP + 4 * kChunk) * 4 + 2 * static_cast<size_t>(terms) * kChunk * PITCH * 2 +
           (half ? kThreadsPerCta * 8 : 0);
  }
};

// grad[a, r, c] = sum over the tokens of adapter a of s[t, r] z[t, c].
//
// The adapter's tokens are shared out over the cluster in chunks of 64, whose
// s values are split into terms once in shared memory for all warps; z goes
// straight to the lanes that use it, UNITS steps ahead.  A chunk's sum is
// formed by the matrix units (4 steps per term) and added to the running sum in
// fp32 with rounding, so that a long batch loses nothing to the units'
// truncation.  The cluster's partial sums are added in rank order.
//
// DIRECT: bf16 results of batches up to kDirectTokens are added up by the units
// themselves.  They truncate twice per step and term at most, 2^-10 of the sum over
// such a batch, a quarter of half a step of the result, were all of it one CTA's;
// 32768 tokens of one sign and one adapter came out 3.05e-4 too small on
// average, and 3.0e-4 when added with rounding (the results' own rounding).
// 8192 tokens, 8192 features, rank 32 80 -> 73 us; 4096 tokens, rank 64 92 -> 83, 128
// 220 -> 188.
constexpr int64_t kDirectTokens = 32768;
template <typename T, typename TG, typename S, int TERMS, bool Q8, bool VEC, bool DIRECT, int MINB>
__global__ void __launch_bounds__(kThreadsPerCta, MINB) k_wgrad(const LowRankWgradArgs args) {
  const LowRankWgradArgs::One& a = args.one[blockIdx.z];
  const int rank = args.rank;
  constexpr int MR = S::MR, RP = S::RP;
  constexpr bool HALF = std::is_same_v<T, __half>;
  static_assert(!DIRECT || (!HALF && sizeof(TG) == 2), "bf16 results only");
  extern __shared__ __align__(16) uint8_t smem[];
  float* part = reinterpret_cast<float*>(smem);                    // [RP][COLS]: this CTA's sum, after the ring's use
  float* scales = reinterpret_cast<float*>(smem + S::SHARED_BYTES);  // [2][RP]: power of two of every rank row (fp16)
  int* toks = reinterpret_cast<int*>(scales + 2 * RP);             // [4][kChunk]: -1 behind the last
  float* steps = reinterpret_cast<float*>(toks + 4 * kChunk);      // [2][COLS / 64][kChunk] (8 bits)
  uint16_t* terms =  // [2][TERMS][kChunk][PITCH]
      reinterpret_cast<uint16_t*>(steps + (Q8 ? 2 * (S::COLS / 64) * kChunk : 0));
  uint2* largest = reinterpret_cast<uint2*>(terms + 2 * TERMS * kChunk * S::PITCH);  // by thread (fp16)

  const uint32_t crank = cluster_rank(), csize = cluster_size();
  const int adapter = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int rg = warp % S::RG;
  const int lc = (warp / S::RG) * 64;                              // first feature of the warp in the CTA
  const int c0 = static_cast<int>(blockIdx.x / csize) * S::COLS;
  if (c0 >= a.k) return;  // the whole cluster: the other gradient is wider
  const int p0 = args.starts[adapter], p1 = args.starts[adapter + 1];
  // This CTA's chunks: crank, crank + csize, ...; only the last of all is short.
  const int first = p0 + static_cast<int>(crank) * kChunk;
  const int hop = static_cast<int>(csize) * kChunk;
  const int chunks = first < p1 ? (p1 - first + hop - 1) / hop : 0;
  const int last_have = chunks > 0 ? min(kChunk, p1 - (first + (chunks - 1) * hop)) : 0;
  const int units = chunks > 0 ? 4 * (chunks - 1) + (last_have + 15) / 16 : 0;
  const int cz = c0 + lc + 8 * g;  // features this lane loads
  const int left = a.k - cz;
  const uint32_t ring0 = smem_addr(smem) + static_cast<uint32_t>(warp * S::UNITS * 4 * 512);
  const uint32_t ring = ring0 + (Q8 ? codes_by_rows(g, t) : by_rows(g, t));

  // The tokens of a chunk are in shared memory three chunks ahead of its use.
  static_assert(S::UNITS <= 8, "a unit's tokens are known when it starts");
  auto chunk_token = [&](int n) {
    const int p = first + n * hop + threadIdx.x;
    return n < chunks && p < p1 ? __ldg(args.order + p) : -1;
  };
  if (threadIdx.x < kChunk) {
#pragma unroll
    for (int n = 0; n < 3; ++n) toks[n * kChunk + threadIdx.x] = chunk_token(n);
  }
  __syncthreads();
  // Unit u: 16 tokens of chunk u / 4, of which this lane takes 2t, 2t+1, 2t+8, 2t+9.
  const T* zcol = Q8 ? nullptr : static_cast<const T*>(a.z) + (left > 0 ? cz : 0);
  const int8_t* qcol = Q8 ? a.codes + (left > 0 ? cz : 0) : nullptr;
  auto issue = [&](int u, int at) {
    if (u < units) {
      if constexpr (!VEC) {
        const uint32_t dst = ring0 + static_cast<uint32_t>(at * 4 * 512 + 2 * (lane & 7));
        const int* unit = toks + ((u >> 2) & 3) * kChunk + (u & 3) * 16;
        const int c = c0 + lc + lane;
#pragma unroll
        for (int i0 = 0; i0 < 4; i0 += 2) {
          uint32_t v[2][4][2];
#pragma unroll
          for (int w = 0; w < 2; ++w)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const int tok = unit[2 * q + w + (i0 >> 1) * 8];
#pragma unroll
              for (int s = 0; s < 2; ++s)
                v[w][q][s] =
                    tok >= 0 ? value_at<T>(static_cast<const T*>(a.z) + static_cast<int64_t>(tok) * a.ldz, c + 32 * s, a.k)
                             : 0u;
            }
#pragma unroll
          for (int w = 0; w < 2; ++w)
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
              for (int s = 0; s < 2; ++s)
                put16(dst + (i0 + w) * 512 + by_rows((lane >> 3) + 4 * s, q), v[w][q][s]);
        }
        commit();
        return;
      }
      const uint32_t dst = ring + static_cast<uint32_t>(at * 4 * 512);
      const int* mine = toks + ((u >> 2) & 3) * kChunk + (u & 3) * 16 + 2 * t;
      const int2 ta = *reinterpret_cast<const int2*>(mine), tb = *reinterpret_cast<const int2*>(mine + 8);
      const int tk[4] = {ta.x, ta.y, tb.x, tb.y};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int n = tk[i] >= 0 ? left : 0;
        const int tok = max(tk[i], 0);
        if constexpr (!Q8) {
          fetch<T>(dst + i * 512, zcol + static_cast<int64_t>(tok) * a.ldz, n);
        } else {
          // code rows are 16-byte aligned and padded to 8
          asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst + i * 512),
                       "l"(qcol + static_cast<int64_t>(tok) * a.ldq), "r"(max(0, min(n, 8)))
                       : "memory");
        }
      }
    }
    commit();
  };
#pragma unroll
  for (int u = 0; u < S::UNITS; ++u) issue(u, u);

  // s of a chunk: the thread's share in registers, then split into terms.
  // (A group of 64 features is one warp's: one step per token and warp.)
  constexpr int STEPS = Q8 ? kChunk * (S::COLS / 64) / kThreadsPerCta + (kChunk * (S::COLS / 64) < kThreadsPerCta) : 1;
  float mine[S::PER_THREAD], my_step[STEPS];
  auto load_s = [&](int n) {
    if constexpr (Q8) {
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const int e = i * kThreadsPerCta + threadIdx.x;
        const int tok = toks[(n & 3) * kChunk + e % kChunk], c = c0 + 64 * (e / kChunk);
        my_step[i] = (tok >= 0 && e / kChunk < S::COLS / 64 && c < a.k)
                         ? __ldg(a.steps + static_cast<int64_t>(c >> 6) * a.lds + tok)
                         : 0.f;
      }
    }
    // pairs of neighbours in a rank row's order, for words of two terms
    const int r = 2 * static_cast<int>(threadIdx.x % (RP / 2));
#pragma unroll
    for (int i = 0; i < S::PER_THREAD; i += 2) {
      const int tok = toks[(n & 3) * kChunk + (i / 2 * kThreadsPerCta + threadIdx.x) / (RP / 2)];
      const float* s = a.s + static_cast<int64_t>(max(tok, 0)) * rank + r;
      mine[i] = (tok >= 0 && r < rank) ? __ldg(s) : 0.f;
      mine[i + 1] = (tok >= 0 && r + 1 < rank) ? __ldg(s + 1) : 0.f;
    }
  };
  auto store_s = [&](int n) {
    if constexpr (Q8) {
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const int e = i * kThreadsPerCta + threadIdx.x;
        if (e / kChunk < S::COLS / 64) steps[(n & 1) * (S::COLS / 64) * kChunk + e] = my_step[i];
      }
    }
    float dn0 = 1.f, dn1 = 1.f;
    if constexpr (HALF) {
      // All pairs of a thread are of the same two rank rows, which it shares with
      // kThreadsPerCta / (RP / 2) - 1 others.
      static_assert(kThreadsPerCta % (RP / 2) == 0, "a thread's pairs are of two rank rows");
      uint2 m = make_uint2(0u, 0u);
#pragma unroll
      for (int i = 0; i < S::PER_THREAD; i += 2) {
        m.x = max(m.x, __float_as_uint(mine[i]) & 0x7fffffffu);
        m.y = max(m.y, __float_as_uint(mine[i + 1]) & 0x7fffffffu);
      }
      largest[threadIdx.x] = m;
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kThreadsPerCta / (RP / 2); ++j) {
        const uint2 o = largest[j * (RP / 2) + threadIdx.x % (RP / 2)];
        m.x = max(m.x, o.x);
        m.y = max(m.y, o.y);
      }
      float up0, up1;
      power_scale(__uint_as_float(m.x), &dn0, &up0);
      power_scale(__uint_as_float(m.y), &dn1, &up1);
      if (threadIdx.x < RP / 2)
        *reinterpret_cast<float2*>(scales + (n & 1) * RP + 2 * threadIdx.x) = make_float2(up0, up1);
    }
#pragma unroll
    for (int i = 0; i < S::PER_THREAD; i += 2) {
      float v0 = mine[i] * dn0, v1 = mine[i + 1] * dn1;
      uint16_t* to = terms + ((n & 1) * TERMS * kChunk + (i / 2 * kThreadsPerCta + threadIdx.x) / (RP / 2)) * S::PITCH +
                     2 * (threadIdx.x % (RP / 2));
#pragma unroll
      for (int q = 0; q < TERMS; ++q) {
        const uint32_t b = bits16x2<T>(v0, v1);
        *reinterpret_cast<uint32_t*>(to + q * kChunk * S::PITCH) = b;
        v0 -= value16<T>(static_cast<uint16_t>(b));
        v1 -= value16<T>(static_cast<uint16_t>(b >> 16));
      }
    }
  };
  if (chunks > 0) {
    load_s(0);
    store_s(0);
  }
  __syncthreads();

  float sum[MR][8][4];
#pragma unroll
  for (int m = 0; m < MR; ++m)
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[m][j][i] = 0.f;
  const uint32_t terms_addr =
      smem_addr(terms) + static_cast<uint32_t>(((lane & 7) + ((lane >> 4) & 1) * 8) * S::PITCH + rg * MR * 16 +
                                               ((lane >> 3) & 1) * 8) * 2u;
  int at = 0;
  for (int n = 0; n < chunks; ++n) {
    const int later = threadIdx.x < kChunk ? chunk_token(n + 3) : -1;
    if (n + 1 < chunks) load_s(n + 1);
    auto multiply = [&](float (&acc)[MR][8][4]) {
      const int here = min(4, units - 4 * n);
#pragma unroll 1
      for (int ks = 0; ks < here; ++ks) {
        wait_all_but<S::UNITS - 1>();
        if constexpr (!VEC) __syncwarp();
        const uint32_t src = ring + static_cast<uint32_t>(at * 4 * 512);
        uint4 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (!Q8) {
            v[i] = landed(src + i * 512);
          } else {
            const int row = ks * 16 + 2 * t + (i & 1) + (i >> 1) * 8;
            v[i] = read_back<T>(landed_codes(src + i * 512),
                                steps[((n & 1) * (S::COLS / 64) + (lc >> 6)) * kChunk + row]);
          }
        }
        uint32_t b0[8], b1[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          b0[j] = pair_of(v[0], v[1], j);
          b1[j] = pair_of(v[2], v[3], j);
        }
        if constexpr (!VEC) __syncwarp();
        issue(4 * n + ks + S::UNITS, at);
        at = at + 1 == S::UNITS ? 0 : at + 1;
#pragma unroll
        for (int m = 0; m < MR; ++m)
#pragma unroll
          for (int q = TERMS - 1; q >= 0; --q) {
            uint32_t f[4];
            ldmatrix4_trans(f, terms_addr + static_cast<uint32_t>((((n & 1) * TERMS + q) * kChunk + ks * 16) * S::PITCH +
                                                                  m * 16) * 2u);
#pragma unroll
            for (int j = 0; j < 8; ++j) mma<T>(acc[m][j], f, b0[j], b1[j]);
          }
      }
    };
    if constexpr (DIRECT) {
      multiply(sum);
    } else {
      float acc[MR][8][4];
#pragma unroll
      for (int m = 0; m < MR; ++m)
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[m][j][i] = 0.f;
      multiply(acc);
#pragma unroll
      for (int m = 0; m < MR; ++m) {
        float pa = 1.f, pb = 1.f;
        if constexpr (HALF) {
          pa = scales[(n & 1) * RP + (rg * MR + m) * 16 + g];
          pb = scales[(n & 1) * RP + (rg * MR + m) * 16 + g + 8];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          sum[m][j][0] += acc[m][j][0] * pa;
          sum[m][j][1] += acc[m][j][1] * pa;
          sum[m][j][2] += acc[m][j][2] * pb;
          sum[m][j][3] += acc[m][j][3] * pb;
        }
      }
    }
    if (n + 1 < chunks) store_s(n + 1);  // the other half of terms: read by no warp since the last barrier
    if (threadIdx.x < kChunk) toks[((n + 3) & 3) * kChunk + threadIdx.x] = later;
    __syncthreads();
  }
  wait_all_but<0>();
  __syncthreads();  // the ring becomes the partial sums
#pragma unroll
  for (int m = 0; m < MR; ++m)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float* row = part + ((rg * MR + m) * 16 + h * 8 + g) * S::COLS + lc + 16 * t;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const float (*v)[4] = &sum[m][4 * q];
        *reinterpret_cast<float4*>(row + 4 * q) = make_float4(v[0][2 * h], v[1][2 * h], v[2][2 * h], v[3][2 * h]);
        *reinterpret_cast<float4*>(row + 8 + 4 * q) =
            make_float4(v[0][2 * h + 1], v[1][2 * h + 1], v[2][2 * h + 1], v[3][2 * h + 1]);
      }
    }
  cluster_sync();
  const uint32_t part_addr = smem_addr(part);
  TG* grad = static_cast<TG*>(a.grad) + static_cast<int64_t>(adapter) * rank * a.k;
  const int total = rank * S::COLS / 4;
  for (int i = static_cast<int>(crank) * kThreadsPerCta + threadIdx.x; i < total;
       i += static_cast<int>(csize) * kThreadsPerCta) {
    const int r = i / (S::COLS / 4), c = c0 + 4 * (i - r * (S::COLS / 4));
    const float4 v = peer_sum4(part_addr + 16u * i, csize);
    const float f[4] = {v.x, v.y, v.z, v.w};
    TG* to = grad + static_cast<int64_t>(r) * a.k + c;
    if (VEC && !Q8 && c < a.k) {  // k is a multiple of 8
      store_f32<TG, 4>(to, f);
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (c + q < a.k) to[q] = from_f32<TG>(f[q]);
    }
  }
  cluster_sync();  // the others may still read this CTA's sums
}

template <typename T, typename TG, typename S, bool Q8, bool VEC, bool DIRECT>
cudaError_t launch_wgrad(const LowRankWgradArgs& a, int64_t adapters, int cluster, cudaStream_t s) {
  constexpr int TERMS = std::is_same_v<TG, float> ? 3 : 2;
  constexpr size_t bytes = S::bytes(TERMS, std::is_same_v<T, __half>, Q8);
  static_assert(bytes <= 227 * 1024, "shared memory of one CTA");
  constexpr int MINB = S::MR == 1 && bytes <= 113 * 1024 ? 2 : 1;  // MR 2 needs the registers of both
  auto* fn = &k_wgrad<T, TG, S, TERMS, Q8, VEC, DIRECT, MINB>;
  static std::atomic<uint64_t> done{0};
  cudaError_t e = allow_smem(fn, bytes, &done);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(ceil_div64(a.widest, S::COLS) * cluster), static_cast<unsigned>(adapters),
                     static_cast<unsigned>(a.count));
  cfg.blockDim = dim3(kThreadsPerCta);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = s;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = static_cast<unsigned>(cluster);
  at.val.clusterDim.y = 1;
  at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, fn, a);
}

template <typename T, typename TG, bool Q8, bool VEC, bool DIRECT>
cudaError_t pick_shape(const LowRankWgradArgs& a, int64_t adapters, int cluster, cudaStream_t s) {
  if (a.rank <= 16) return launch_wgrad<T, TG, WgradShape<1, 1, 5>, Q8, VEC, DIRECT>(a, adapters, cluster, s);
  if (a.rank <= 32) return launch_wgrad<T, TG, WgradShape<1, 2, 8>, Q8, VEC, DIRECT>(a, adapters, cluster, s);
  if (a.rank <= 64) return launch_wgrad<T, TG, WgradShape<2, 2, 8>, Q8, VEC, DIRECT>(a, adapters, cluster, s);
  return launch_wgrad<T, TG, WgradShape<4, 2, 4>, Q8, VEC, DIRECT>(a, adapters, cluster, s);
}

template <typename T, typename TG, bool Q8, bool VEC>
cudaError_t pick_wgrad(const LowRankWgradArgs& a, int64_t adapters, int cluster, cudaStream_t s) {
  if constexpr (std::is_same_v<T, __nv_bfloat16> && sizeof(TG) == 2) {
    if (a.tokens <= kDirectTokens) return pick_shape<T, TG, Q8, VEC, true>(a, adapters, cluster, s);
  }
  return pick_shape<T, TG, Q8, VEC, false>(a, adapters, cluster, s);
}

}  // namespace lowrank

// Definitions of the launches for one element type.
#define KAIRO_LOW_RANK_LAUNCHES(T)                                                                                   \
  template <>                                                                                                        \
  cudaError_t launch_low_rank_apply<T>(const LowRankApplyArgs& a, bool y_f32, bool vec, int tile, int64_t clusters,  \
                                       int cluster, cudaStream_t s) {                                               \
    return y_f32 ? lowrank::pick_apply<T, float>(a, vec, tile, clusters, cluster, s)                                 \
                 : lowrank::pick_apply<T, T>(a, vec, tile, clusters, cluster, s);                                    \
  }                                                                                                                  \
  template <>                                                                                                        \
  cudaError_t launch_low_rank_wgrad<T>(const LowRankWgradArgs& a, bool grad_f32, bool vec, int64_t adapters,         \
                                       int cluster, cudaStream_t s) {                                               \
    if (a.one[0].codes)                                                                                              \
      return grad_f32 ? lowrank::pick_wgrad<T, float, true, true>(a, adapters, cluster, s)                           \
                      : lowrank::pick_wgrad<T, T, true, true>(a, adapters, cluster, s);                              \
    if (vec)                                                                                                         \
      return grad_f32 ? lowrank::pick_wgrad<T, float, false, true>(a, adapters, cluster, s)                          \
                      : lowrank::pick_wgrad<T, T, false, true>(a, adapters, cluster, s);                             \
    return grad_f32 ? lowrank::pick_wgrad<T, float, false, false>(a, adapters, cluster, s)                           \
                    : lowrank::pick_wgrad<T, T, false, false>(a, adapters, cluster, s);                              \
  }

}  // namespace kairo
