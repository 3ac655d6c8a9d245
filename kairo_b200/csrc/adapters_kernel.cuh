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
//    takes features 8 g .. 8 g + 7 of the rank rows (tokens) 2t, 2t+1, 2t+8,
//    2t+9 as column g of eight products, and so holds of the result 16
//    contiguous features 16 t .. 16 t + 15 of its rows.
// Every access is a whole 16-byte vector of a fully used sector.
//
// low is an fp32 value.  For a product with 16-bit weights it is split into
// terms of the weights' type, each the rounding of what the ones before leave:
// two for 16-bit results (rest at most 2^-17 of it), three for fp32 results
// (2^-23).  In fp16, whose range is narrow, it is first scaled by a power of
// two (exact) that brings the largest of the row to [1, 2).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "convert.cuh"
#include "internal.h"

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

struct LowRankWgradArgs {
  const float* s;      // (tokens, rank)
  const void* z;       // (tokens, k), or null when given in 8 bits
  const int8_t* codes;
  const float* steps;
  void* grad;          // (adapters, rank, k)
  const int32_t* order;
  const int32_t* starts;
  int64_t ldz, ldq, lds;
  int32_t k, rank;
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
__device__ __forceinline__ float peer_load(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
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

// 8 elements at p, of which the first `left` exist (left may be <= 0).  VEC:
// p is 16-byte aligned and left is a multiple of 8 or not positive.
template <typename T, bool VEC>
__device__ __forceinline__ uint4 load8(const T* p, int left) {
  uint4 v = make_uint4(0u, 0u, 0u, 0u);
  if constexpr (VEC) {
    if (left > 0) v = __ldg(reinterpret_cast<const uint4*>(p));
  } else {
    uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) w[i >> 1] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(p)[i]) << (16 * (i & 1));
    v = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return v;
}

template <typename T>
__device__ __forceinline__ uint16_t bits16(float v) {
  const T h = from_f32<T>(v);
  return *reinterpret_cast<const uint16_t*>(&h);
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

template <int MT, int NT>
struct ApplySmem {
  static constexpr int ROWS = 16 * MT;
  static constexpr int RP = 8 * NT;          // rank, padded
  static constexpr int PITCH = RP + 8;       // 16-bit terms: rows 16 bytes apart in banks
  static constexpr int LOW = ROWS * RP;      // floats of one low tile
};

// One cluster per tile.  Its CTAs and warps share out the features of the
// contraction, 64 at a time; partial low tiles meet in shared memory, then over
// the cluster's distributed shared memory; each CTA gets the whole low tile
// and its warps share out the output features, 64 at a time.  One launch, low
// never travels through global memory.
template <typename T, typename TY, int MT, int NT, int TERMS, bool VEC>
__global__ void __launch_bounds__(kThreadsPerCta, NT > 8 ? 1 : 2) k_apply(const LowRankApplyArgs a) {
  using S = ApplySmem<MT, NT>;
  extern __shared__ __align__(16) uint8_t smem[];
  float* red = reinterpret_cast<float*>(smem);                   // [kWarps][LOW], reused below
  float* part = red + kWarps * S::LOW;                           // [LOW]: this CTA's partial tile
  float* low = part + S::LOW;                                    // [LOW]: the whole tile
  float* row_up = low + S::LOW;                                  // [ROWS]: power of two of every row (fp16)
  uint16_t* terms = reinterpret_cast<uint16_t*>(row_up + S::ROWS);  // [TERMS][ROWS][PITCH]

  const uint32_t crank = cluster_rank(), csize = cluster_size();
  const int64_t ti = blockIdx.x / csize;
  if (ti >= *a.ntiles) return;  // the whole cluster
  const LowRankTile tile = a.tiles[ti];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int slot = static_cast<int>(crank) * kWarps + warp;      // this warp among the cluster's
  const int slots = static_cast<int>(csize) * kWarps;
  const int count = min(tile.count, S::ROWS);
  int tok[MT][2];  // tokens of this lane's rows, -1: none
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = m * 16 + h * 8 + g;
      tok[m][h] = row < count ? a.order[tile.begin + row] : -1;
    }

  if (tile.adapter >= 0) {
    const T* down = static_cast<const T*>(a.down) + static_cast<int64_t>(tile.adapter) * a.rank * a.k;
    float acc[MT][NT][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[m][j][i] = 0.f;
    const T* xrow[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        xrow[m][h] = static_cast<const T*>(a.x) + static_cast<int64_t>(max(tok[m][h], 0)) * a.ldx;
    for (int k0 = slot * 64; k0 < a.k; k0 += slots * 64) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int kk = k0 + half * 32 + 8 * t;
        const int left = a.k - kk;
        uint4 xa[MT][2], wb[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const int r = j * 8 + g;
          wb[j] = load8<T, VEC>(down + static_cast<int64_t>(r) * a.k + kk, r < a.rank ? left : 0);
        }
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int h = 0; h < 2; ++h) xa[m][h] = load8<T, VEC>(xrow[m][h] + kk, tok[m][h] >= 0 ? left : 0);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const uint32_t a0[4] = {xa[m][0].x, xa[m][1].x, xa[m][0].y, xa[m][1].y};
          const uint32_t a1[4] = {xa[m][0].z, xa[m][1].z, xa[m][0].w, xa[m][1].w};
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            mma<T>(acc[m][j], a0, wb[j].x, wb[j].y);
            mma<T>(acc[m][j], a1, wb[j].z, wb[j].w);
          }
        }
      }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        float* at = red + warp * S::LOW + (m * 16 + g) * S::RP + j * 8 + 2 * t;
        *reinterpret_cast<float2*>(at) = make_float2(acc[m][j][0], acc[m][j][1]);
        *reinterpret_cast<float2*>(at + 8 * S::RP) = make_float2(acc[m][j][2], acc[m][j][3]);
      }
    __syncthreads();
    for (int i = threadIdx.x; i < S::LOW; i += kThreadsPerCta) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) v += red[w * S::LOW + i];
      part[i] = v;
    }
    cluster_sync();
    // Each CTA sums its share of the tile over the cluster, in rank order, and
    // gives the result to all.
    const float scale = a.scale ? a.scale[tile.adapter] : 1.f;
    const uint32_t part_addr = smem_addr(part), low_addr = smem_addr(low);
    const int share = (S::LOW + static_cast<int>(csize) - 1) / static_cast<int>(csize);
    const int i0 = static_cast<int>(crank) * share, i1 = min(S::LOW, i0 + share);
    for (int i = i0 + threadIdx.x; i < i1; i += kThreadsPerCta) {
      float v = 0.f;
      for (uint32_t c = 0; c < csize; ++c) v += peer_load(peer_addr(part_addr + 4u * i, c));
      v *= scale;
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

  const bool live = tile.adapter >= 0;
  if (live) {
    if constexpr (std::is_same_v<T, __half>) {
      for (int row = warp; row < S::ROWS; row += kWarps) {
        uint32_t m = 0;
        for (int r = lane; r < S::RP; r += 32) m = max(m, __float_as_uint(low[row * S::RP + r]) & 0x7fffffffu);
        m = __reduce_max_sync(0xffffffffu, m);
        float dn, up;
        power_scale(__uint_as_float(m), &dn, &up);
        for (int r = lane; r < S::RP; r += 32) low[row * S::RP + r] *= dn;
        if (lane == 0) row_up[row] = up;
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

  constexpr int KT = NT / 2;  // rank steps of 16
  const T* up = static_cast<const T*>(a.up) + static_cast<int64_t>(max(tile.adapter, 0)) * a.rank * a.n;
  TY* y = static_cast<TY*>(a.y);
  // ldmatrix: lane l names row l % 16 and rank half l / 16 of a 16 x 16 tile.
  const uint32_t terms_addr = smem_addr(terms) + static_cast<uint32_t>((lane & 15) * S::PITCH + (lane >> 4) * 8) * 2u;
  for (int n0 = slot * 64; n0 < a.n; n0 += slots * 64) {
    uint32_t b0[KT][8], b1[KT][8];
    if (live) {
      const int c = n0 + 8 * g;
      const int left = a.n - c;
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        uint4 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = kt * 16 + 2 * t + (i & 1) + (i >> 1) * 8;
          v[i] = load8<T, VEC>(up + static_cast<int64_t>(r) * a.n + c, r < a.rank ? left : 0);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          b0[kt][j] = pair_of(v[0], v[1], j);
          b1[kt][j] = pair_of(v[2], v[3], j);
        }
      }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      if (m * 16 >= count) break;
      float out[2][16];  // rows g and g + 8: features n0 + 16 t ..
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int i = 0; i < 16; ++i) out[h][i] = 0.f;
        if (tok[m][h] < 0 || !a.base) continue;
        const int c = n0 + 16 * t;
        const int64_t at = static_cast<int64_t>(tok[m][h]) * a.ldb + c;
        if (a.base_f32) {
          const float* b = static_cast<const float*>(a.base) + at;
          if constexpr (VEC) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
              if (c + 4 * q < a.n) {
                const float4 v = *reinterpret_cast<const float4*>(b + 4 * q);
                out[h][4 * q] = v.x;
                out[h][4 * q + 1] = v.y;
                out[h][4 * q + 2] = v.z;
                out[h][4 * q + 3] = v.w;
              }
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (c + i < a.n) out[h][i] = b[i];
          }
        } else {
          const T* b = static_cast<const T*>(a.base) + at;
          if constexpr (VEC) {
#pragma unroll
            for (int q = 0; q < 2; ++q)
              if (c + 8 * q < a.n) {
                float f[8];
                load_f32<T, 8>(b + 8 * q, f);
#pragma unroll
                for (int i = 0; i < 8; ++i) out[h][8 * q + i] = f[i];
              }
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (c + i < a.n) out[h][i] = to_f32<T>(b[i]);
          }
        }
      }
      if (live) {
        float acc[8][4];
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[j][i] = 0.f;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
          for (int q = TERMS - 1; q >= 0; --q) {
            uint32_t f[4];
            ldmatrix4(f, terms_addr + static_cast<uint32_t>((q * S::ROWS + m * 16) * S::PITCH + kt * 16) * 2u);
#pragma unroll
            for (int j = 0; j < 8; ++j) mma<T>(acc[j], f, b0[kt][j], b1[kt][j]);
          }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float p = 1.f;
          if constexpr (std::is_same_v<T, __half>) p = row_up[m * 16 + h * 8 + g];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            out[h][j] += acc[j][2 * h] * p;
            out[h][8 + j] += acc[j][2 * h + 1] * p;
          }
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (tok[m][h] < 0) continue;
        const int c = n0 + 16 * t;
        TY* d = y + static_cast<int64_t>(tok[m][h]) * a.ldy + c;
        if constexpr (VEC) {
          constexpr int W = 16 / static_cast<int>(sizeof(TY));  // features per 16 bytes
#pragma unroll
          for (int q = 0; q < 16 / W; ++q)
            if (c + W * q < a.n) {
              float f[W];
#pragma unroll
              for (int i = 0; i < W; ++i) f[i] = out[h][W * q + i];
              store_f32<TY, W>(d + W * q, f);
            }
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (c + i < a.n) d[i] = from_f32<TY>(out[h][i]);
        }
      }
    }
  }
}

template <typename T, typename TY, int MT, int NT, bool VEC>
cudaError_t launch_apply(const LowRankApplyArgs& a, int64_t clusters, int cluster, cudaStream_t s) {
  using S = ApplySmem<MT, NT>;
  constexpr int TERMS = std::is_same_v<TY, float> ? 3 : 2;
  constexpr size_t bytes = static_cast<size_t>((kWarps + 2) * S::LOW + S::ROWS) * 4 +
                           static_cast<size_t>(TERMS) * S::ROWS * S::PITCH * 2;
  auto* fn = &k_apply<T, TY, MT, NT, TERMS, VEC>;
  cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
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

template <typename T, typename TY>
cudaError_t pick_apply(const LowRankApplyArgs& a, bool vec, int tile, int64_t clusters, int cluster, cudaStream_t s) {
  if (!vec) {
    if (a.rank <= 16) return launch_apply<T, TY, 1, 2, false>(a, clusters, cluster, s);
    if (a.rank <= 32) return launch_apply<T, TY, 1, 4, false>(a, clusters, cluster, s);
    if (a.rank <= 64) return launch_apply<T, TY, 1, 8, false>(a, clusters, cluster, s);
    return launch_apply<T, TY, 1, 16, false>(a, clusters, cluster, s);
  }
  if (a.rank <= 16)
    return tile == 64 ? launch_apply<T, TY, 4, 2, true>(a, clusters, cluster, s)
                      : launch_apply<T, TY, 1, 2, true>(a, clusters, cluster, s);
  if (a.rank <= 32)
    return tile == 64 ? launch_apply<T, TY, 4, 4, true>(a, clusters, cluster, s)
                      : launch_apply<T, TY, 1, 4, true>(a, clusters, cluster, s);
  if (a.rank <= 64)
    return tile == 32 ? launch_apply<T, TY, 2, 8, true>(a, clusters, cluster, s)
                      : launch_apply<T, TY, 1, 8, true>(a, clusters, cluster, s);
  return launch_apply<T, TY, 1, 16, true>(a, clusters, cluster, s);
}

// ---------------------------------------------------------------- weight gradient

// grad[a, r, c] = sum over the tokens of adapter a of s[t, r] z[t, c].
//
// A warp owns 16 rank rows and 64 features; RG warps side by side cover the
// rank, kWarps / RG column groups the CTA's features.  The tokens of the
// adapter are shared out over the cluster in chunks of 64, whose s values are
// split into terms once in shared memory for all warps.  A chunk's sum is
// formed by the matrix units (4 steps per term) and added to the running
// sum in fp32 with rounding, so that a long batch loses nothing to the units'
// truncation.  The cluster's partial sums are added in rank order.
template <typename T, bool Q8, bool VEC>
__device__ __forceinline__ uint4 load_z(const LowRankWgradArgs& a, int tok, int c, int left) {
  if (tok < 0) return make_uint4(0u, 0u, 0u, 0u);
  if constexpr (!Q8) {
    return load8<T, VEC>(static_cast<const T*>(a.z) + static_cast<int64_t>(tok) * a.ldz + c, left);
  } else {
    // code rows are 16-byte aligned: 8 codes may be read together when 8 exist
    uint32_t w[4] = {0u, 0u, 0u, 0u};
    if (left > 0) {
      const int8_t* q = a.codes + static_cast<int64_t>(tok) * a.ldq + c;
      const float step = a.steps[static_cast<int64_t>(c >> 6) * a.lds + tok];
      uint32_t b[2] = {0u, 0u};
      if (left >= 8) {
        const uint2 v = *reinterpret_cast<const uint2*>(q);
        b[0] = v.x;
        b[1] = v.y;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i < left) b[i >> 2] |= static_cast<uint32_t>(static_cast<uint8_t>(q[i])) << (8 * (i & 3));
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float f = static_cast<float>(static_cast<int8_t>(b[i >> 2] >> (8 * (i & 3)))) * step;
        w[i >> 1] |= static_cast<uint32_t>(i < left ? bits16<T>(f) : 0) << (16 * (i & 1));
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <int RG>
struct WgradSmem {
  static constexpr int RP = 16 * RG;
  static constexpr int PITCH = RP + 8;
  static constexpr int COLS = 64 * (kWarps / RG);
};

template <typename T, typename TG, int RG, int TERMS, bool Q8, bool VEC>
__global__ void __launch_bounds__(kThreadsPerCta, 2) k_wgrad(const LowRankWgradArgs a) {
  using S = WgradSmem<RG>;
  extern __shared__ __align__(16) uint8_t smem[];
  float* part = reinterpret_cast<float*>(smem);                    // [RP][COLS]: this CTA's sum
  float* raw = part;                                               // [kChunk][RP]: s of a chunk (before the sum)
  float* up = part + S::RP * S::COLS;                              // [RP]: power of two of every rank row (fp16)
  int* toks = reinterpret_cast<int*>(up + S::RP);                  // [kChunk]
  uint16_t* terms = reinterpret_cast<uint16_t*>(toks + kChunk);    // [TERMS][kChunk][PITCH]

  const uint32_t crank = cluster_rank(), csize = cluster_size();
  const int adapter = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int rg = warp % RG;
  const int lc = (warp / RG) * 64;                                 // first feature of the warp in the CTA
  const int c0 = (blockIdx.x / csize) * S::COLS;
  const int p0 = a.starts[adapter], p1 = a.starts[adapter + 1];
  float sum[8][4];
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[j][i] = 0.f;
  const int cz = c0 + lc + 8 * g;  // features this lane loads
  const int left = a.k - cz;
  const uint32_t terms_addr =
      smem_addr(terms) +
      static_cast<uint32_t>(((lane & 7) + ((lane >> 4) & 1) * 8) * S::PITCH + rg * 16 + ((lane >> 3) & 1) * 8) * 2u;
  for (int q0 = p0 + static_cast<int>(crank) * kChunk; q0 < p1; q0 += static_cast<int>(csize) * kChunk) {
    const int have = min(kChunk, p1 - q0);
    __syncthreads();  // the last chunk's terms are no longer read
    if (threadIdx.x < kChunk) toks[threadIdx.x] = threadIdx.x < have ? a.order[q0 + threadIdx.x] : -1;
    __syncthreads();
    for (int i = threadIdx.x; i < kChunk * S::RP; i += kThreadsPerCta) {
      const int row = i / S::RP, r = i - row * S::RP;
      const int tok = toks[row];
      float v = (tok >= 0 && r < a.rank) ? a.s[static_cast<int64_t>(tok) * a.rank + r] : 0.f;
      if constexpr (std::is_same_v<T, __half>) {
        raw[i] = v;
      } else {
#pragma unroll
        for (int q = 0; q < TERMS; ++q) {
          const uint16_t b = bits16<T>(v);
          terms[(q * kChunk + row) * S::PITCH + r] = b;
          v -= value16<T>(b);
        }
      }
    }
    __syncthreads();
    if constexpr (std::is_same_v<T, __half>) {
      for (int r = warp; r < S::RP; r += kWarps) {
        const uint32_t v0 = __float_as_uint(raw[lane * S::RP + r]) & 0x7fffffffu;
        const uint32_t v1 = __float_as_uint(raw[(lane + 32) * S::RP + r]) & 0x7fffffffu;
        const uint32_t m = __reduce_max_sync(0xffffffffu, max(v0, v1));
        float dn, u;
        power_scale(__uint_as_float(m), &dn, &u);
        if (lane == 0) up[r] = u;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int row = lane + 32 * h;
          float v = raw[row * S::RP + r] * dn;
#pragma unroll
          for (int q = 0; q < TERMS; ++q) {
            const uint16_t b = bits16<T>(v);
            terms[(q * kChunk + row) * S::PITCH + r] = b;
            v -= value16<T>(b);
          }
        }
      }
      __syncthreads();
    }
    float acc[8][4];
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[j][i] = 0.f;
#pragma unroll
    for (int ks = 0; ks < kChunk / 16; ++ks) {
      if (ks * 16 >= have) break;
      uint4 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v[i] = load_z<T, Q8, VEC>(a, toks[ks * 16 + 2 * t + (i & 1) + (i >> 1) * 8], cz, left);
#pragma unroll
      for (int q = TERMS - 1; q >= 0; --q) {
        uint32_t f[4];
        ldmatrix4_trans(f, terms_addr + static_cast<uint32_t>((q * kChunk + ks * 16) * S::PITCH) * 2u);
#pragma unroll
        for (int j = 0; j < 8; ++j) mma<T>(acc[j], f, pair_of(v[0], v[1], j), pair_of(v[2], v[3], j));
      }
    }
    float pa = 1.f, pb = 1.f;
    if constexpr (std::is_same_v<T, __half>) {
      pa = up[rg * 16 + g];
      pb = up[rg * 16 + g + 8];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      sum[j][0] += acc[j][0] * pa;
      sum[j][1] += acc[j][1] * pa;
      sum[j][2] += acc[j][2] * pb;
      sum[j][3] += acc[j][3] * pb;
    }
  }
  __syncthreads();  // raw and part share memory
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float* row = part + (rg * 16 + h * 8 + g) * S::COLS + lc + 16 * t;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      row[j] = sum[j][2 * h];
      row[8 + j] = sum[j][2 * h + 1];
    }
  }
  cluster_sync();
  const uint32_t part_addr = smem_addr(part);
  TG* grad = static_cast<TG*>(a.grad) + static_cast<int64_t>(adapter) * a.rank * a.k;
  const int total = a.rank * S::COLS;
  for (int i = static_cast<int>(crank) * kThreadsPerCta + threadIdx.x; i < total;
       i += static_cast<int>(csize) * kThreadsPerCta) {
    const int r = i / S::COLS, c = i - r * S::COLS;
    float v = 0.f;
    for (uint32_t q = 0; q < csize; ++q) v += peer_load(peer_addr(part_addr + 4u * i, q));
    if (c0 + c < a.k) grad[static_cast<int64_t>(r) * a.k + c0 + c] = from_f32<TG>(v);
  }
  cluster_sync();  // the others may still read this CTA's sums
}

template <typename T, typename TG, int RG, bool Q8, bool VEC>
cudaError_t launch_wgrad(const LowRankWgradArgs& a, int64_t adapters, int cluster, cudaStream_t s) {
  using S = WgradSmem<RG>;
  constexpr int TERMS = std::is_same_v<TG, float> ? 3 : 2;
  constexpr size_t bytes = static_cast<size_t>(S::RP * S::COLS + S::RP + kChunk) * 4 +
                           static_cast<size_t>(TERMS) * kChunk * S::PITCH * 2;
  static_assert(S::COLS >= kChunk, "raw fits in part");
  auto* fn = &k_wgrad<T, TG, RG, TERMS, Q8, VEC>;
  cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(ceil_div64(a.k, S::COLS) * cluster), static_cast<unsigned>(adapters));
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

template <typename T, typename TG, bool Q8, bool VEC>
cudaError_t pick_wgrad(const LowRankWgradArgs& a, int64_t adapters, int cluster, cudaStream_t s) {
  if (a.rank <= 16) return launch_wgrad<T, TG, 1, Q8, VEC>(a, adapters, cluster, s);
  if (a.rank <= 32) return launch_wgrad<T, TG, 2, Q8, VEC>(a, adapters, cluster, s);
  if (a.rank <= 64) return launch_wgrad<T, TG, 4, Q8, VEC>(a, adapters, cluster, s);
  return launch_wgrad<T, TG, 8, Q8, VEC>(a, adapters, cluster, s);
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
    if (a.codes)                                                                                                     \
      return grad_f32 ? lowrank::pick_wgrad<T, float, true, true>(a, adapters, cluster, s)                           \
                      : lowrank::pick_wgrad<T, T, true, true>(a, adapters, cluster, s);                              \
    if (vec)                                                                                                         \
      return grad_f32 ? lowrank::pick_wgrad<T, float, false, true>(a, adapters, cluster, s)                          \
                      : lowrank::pick_wgrad<T, T, false, true>(a, adapters, cluster, s);                             \
    return grad_f32 ? lowrank::pick_wgrad<T, float, false, false>(a, adapters, cluster, s)                           \
                    : lowrank::pick_wgrad<T, T, false, false>(a, adapters, cluster, s);                              \
  }

}  // namespace kairo
