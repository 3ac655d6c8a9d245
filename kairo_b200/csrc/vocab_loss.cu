// Softmax cross entropy of hidden states against a vocabulary table, without
// keeping the logits, and its gradients.
//
//   z[t, v] = scale * X[t] . W[v]            X: tokens x dim, W: vocab x dim
//   lse[t]  = log sum_v exp z[t, v]
//   loss[t] = lse[t] - z[t, y_t]             0 where y_t is outside [0, vocab)
//   G[t, v] = f[t] * (exp(z[t, v] - lse[t]) - [v = y_t])
//   dX = scale * G W,   dW = scale * G^T X
// with f[t] the gradient by token t's loss (0 where the token does not count).
//
// Forward: one pass of k_pair_gemm over W.  A thread of its epilogue owns one
// token of the tile; it keeps the running maximum and sum of its columns (base
// 2) and picks the target's logit as it goes by, so 8 bytes leave the SM per
// token and 128 columns.  k_lse joins them.  Up to 128 tokens the two operands change
// places: the table, all there is to read, fills whole tiles, and the products
// cost half and draw less power, which the clock shows (64 tokens of 131072 x
// 4096 took 270 us with tiles of 256 tokens when calls followed one another, and 200 from a cool start).
//
// Backward: pieces of the vocabulary, as many columns as keep a 16-bit G of
// all tokens within kPieceBytes.  Per piece the logits are formed again and
// leave as G; dX += G W_piece and dW_piece = G^T X read it as it lies.  That is
// 8 tokens * vocab * dim operations for the 6 that logits kept in memory would
// need; it keeps 2 * tokens bytes a column of the piece instead of 4 * tokens * vocab.
//
// Measured.  8192 tokens, 131072 x 2048, bf16: the forward pass 3.1 ms (1400 TFLOP/s), G 3.4, dX 3.0, dW 3.0
// (1465) one after the other from a cool start; in a row 13.7 to 14.5 ms, 1215 to 1285 TFLOP/s of what is done, where
// the power limit leaves cuBLAS 1355 (SM clock 1.27 GHz).  131072 x 4096 in a row: one token 190 to 207 us (5.2 to 5.7
// TB/s), 64 tokens 197 to 225 (the power limit again, 1.74 GHz).
//
// Rounding.  z, the maxima, sums and lse are fp32.  G is rounded once to the
// operands' 16 bits, as an operand of both products must be: relative to each
// entry up to 2^-8 (bf16) or 2^-11, as the results' own rounding; over many entries the two together are off by 1.4 times
// what one is.  Up to 128 tokens G is held as the sum of two such numbers (`halves`).  The factor that all tokens
// share (the gradient by a mean or a sum) stays out of G and is applied to the
// fp32 sums: -1 + p of a target is then near -1, which rounds exactly, where f *
// (-1 + p) would round every target's entry alike.  In fp16 G also carries 2^15,
// so that probabilities down to 2^-39 are not lost.
#include <algorithm>
#include <cmath>

#include "convert.cuh"
#include "pair_gemm.cuh"

namespace kairo {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int64_t kPieceBytes = 512LL << 20;
constexpr float kHalfLift = 32768.f;  // 2^15, see above
// Probabilities up to here need no second row in G.  They add up to 1 at most, so that their squares' root is an eighth
// (the root of this number), and each is rounded by itself: an eighth of what one rounding does to an entry of 1.
constexpr float kLargeProbability = 1.f / 64.f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Token targets, int32 or int64.
struct Targets {
  const void* p;
  int bytes;
  __device__ __forceinline__ int64_t operator[](int64_t i) const {
    return bytes == 8 ? static_cast<const int64_t*>(p)[i] : static_cast<int64_t>(static_cast<const int32_t*>(p)[i]);
  }
};

// ------------------------------------------------------------ epilogues

// Logits in base 2 are v * stats_scale(scale), of -v where scale < 0.  Not 0: masked columns are -inf.
__host__ __device__ __forceinline__ float stats_scale(float scale) { return fmaxf(fabsf(scale) * kLog2e, 1e-38f); }

// Running maximum and sum of exp2 of one token's columns.  The maximum is a rounded product, but what is subtracted
// from the exact ones (fma), so that the terms that count are as exact as v.
struct StatsEpi {
  struct Args {
    float2* part;   // [slots][tokens]
    float* target;  // [tokens], the target's v
    Targets ids;
    int tokens, vocab;
    float scale;
    int by_cluster;  // one row of tiles: a CTA's tiles share a slot
    unsigned* ticket;  // of k_lse, zeroed here
  };
  const Args& a;
  int row, part, mt = -1;
  int64_t id = -1;
  float m = -INFINITY, s = 0.f;

  __device__ StatsEpi(const Args& args, int row_in_tile, int p, uint8_t*) : a(args), row(row_in_tile), part(p) {
    if (blockIdx.x == 0 && row_in_tile == 0 && p == 0) *a.ticket = 0u;
  }

  __device__ __forceinline__ void flush(int token, int64_t slot) {
    if (token < a.tokens) a.part[slot * a.tokens + token] = make_float2(m, s);
    m = -INFINITY;
    s = 0.f;
  }

  __device__ void tile(const PairTile& pt, float (&v)[kPairEpiCols]) {
    const int token = pt.mt * kPairTileM + row;
    if (__all_sync(0xffffffffu, token >= a.tokens)) return;
    if (pt.mt != mt) {
      mt = pt.mt;
      id = token < a.tokens ? a.ids[token] : -1;
    }
    const int col0 = pt.nt * kPairTileN + part * kPairEpiCols;
    const int64_t at = id - col0;
    const bool here = id >= 0 && id < a.vocab && at >= 0 && at < kPairEpiCols;
    if (__any_sync(0xffffffffu, here)) {
      float z = 0.f;
#pragma unroll
      for (int j = 0; j < kPairEpiCols; ++j)
        if (at == j) z = v[j];
      if (here && token < a.tokens) a.target[token] = z;
    }
    const float k = stats_scale(a.scale);
    if (a.scale < 0.f) {
#pragma unroll
      for (int j = 0; j < kPairEpiCols; ++j) v[j] = -v[j];
    }
    if (col0 + kPairEpiCols > a.vocab) {
#pragma unroll
      for (int j = 0; j < kPairEpiCols; ++j)
        if (col0 + j >= a.vocab) v[j] = -INFINITY;
    }
    float top = v[0];
#pragma unroll
    for (int j = 1; j < kPairEpiCols; ++j) top = fmaxf(top, v[j]);
    top = fmaxf(m, top * k);
    const float ref = top == -INFINITY ? 0.f : top;
    float sum[4] = {s * ex2(m - ref), 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < kPairEpiCols; ++j) sum[j & 3] += ex2(fmaf(v[j], k, -ref));
    m = top;
    s = (sum[0] + sum[1]) + (sum[2] + sum[3]);
    if (!a.by_cluster) flush(token, static_cast<int64_t>(pt.nt) * (kPairTileN / kPairEpiCols) + part);
  }

  __device__ void done() {
    if (a.by_cluster) flush(row, static_cast<int64_t>(blockIdx.x >> 1) * (kPairTileN / kPairEpiCols) + part);
  }
};

// The 8 16-bit values from value `e` (0..7) on of the 16 in a, b.
__device__ __forceinline__ uint4 shift8(uint4 a, uint4 b, int e) {
  uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  if (e & 4) {
#pragma unroll
    for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
  }
  if (e & 2) {
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
  }
  if (e & 1) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 16);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// The same for few tokens, with the vocabulary down the rows: a warp has 32 rows of the table and GROUPS times 32
// tokens, of which lane j keeps the j-th.
template <int GROUPS>
struct FewStatsEpi {
  static constexpr int TOKENS = 64 * GROUPS;  // columns of a tile
  struct Args {
    float2* part;  // [clusters * 8][tokens]
    float* target;
    Targets ids;
    int tokens, vocab;
    float scale;
    unsigned* ticket;
  };
  const Args& a;
  int row, token;  // of the first group
  int64_t id[GROUPS];
  float m[GROUPS], s[GROUPS];

  __device__ FewStatsEpi(const Args& args, int row_in_tile, int part, uint8_t*)
      : a(args), row(row_in_tile), token(part * 32 * GROUPS + static_cast<int>(threadIdx.x & 31)) {
    if (blockIdx.x == 0 && row_in_tile == 0 && part == 0) *a.ticket = 0u;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      id[g] = token + 32 * g < a.tokens ? a.ids[token + 32 * g] : -1;
      if (id[g] >= a.vocab) id[g] = -1;
      m[g] = -INFINITY;
      s[g] = 0.f;
    }
  }

  // 32 values of each lane -> lane j has `op` over all lanes' value j
  template <class F>
  static __device__ __forceinline__ float across(float (&v)[32], F op) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const bool up = lane & o;
#pragma unroll
      for (int i = 0; i < o; ++i) {
        const float give = up ? v[i] : v[i + o], keep = up ? v[i + o] : v[i];
        v[i] = op(keep, __shfl_xor_sync(0xffffffffu, give, o));
      }
    }
    return v[0];
  }

  __device__ void tile(const PairTile& pt, float (&all)[32 * GROUPS]) {
    const int lane = threadIdx.x & 31;
    const int r = pt.mt * kPairTileM + row;
    const float k = stats_scale(a.scale);
    const bool in = r < a.vocab, minus = a.scale < 0.f;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      if (token - lane + 32 * g >= a.tokens) break;
      const int64_t at = id[g] - (r - lane);
      const unsigned hits = __ballot_sync(0xffffffffu, id[g] >= 0 && at >= 0 && at < 32);
      if (hits) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (hits >> j & 1u) {
            const int from = static_cast<int>(__shfl_sync(0xffffffffu, at, j));
            const float z = __shfl_sync(0xffffffffu, all[32 * g + j], from);
            if (lane == j) a.target[token + 32 * g] = z;
          }
      }
      float v[32], w[32];
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        v[j] = in ? (minus ? -all[32 * g + j] : all[32 * g + j]) : -INFINITY;
        w[j] = v[j];
      }
      const float top = fmaxf(m[g], across(w, [](float x, float y) { return fmaxf(x, y); }) * k);
      const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int j = 0; j < 32; ++j) w[j] = ex2(fmaf(v[j], k, -__shfl_sync(0xffffffffu, ref, j)));
      const float sum = across(w, [](float x, float y) { return x + y; });
      s[g] = s[g] * ex2(m[g] - ref) + sum;
      m[g] = top;
    }
  }

  __device__ void done() {
    const int64_t slot = static_cast<int64_t>(blockIdx.x) * 4 + ((row >> 5) & 3);
#pragma unroll
    for (int g = 0; g < GROUPS; ++g)
      if (token + 32 * g < a.tokens) a.part[slot * a.tokens + token + 32 * g] = make_float2(m[g], s[g]);
  }
};

// A warp's 32 rows x kPairEpiCols results, a row a lane, rounded to T at p (16-byte aligned rows of
// pitch ld; `rows` and `cols` of them exist).  They pass through shared memory, 64 columns at a
// time, so that a store instruction writes 128 bytes of each of four rows (a row a lane: 16 bytes of
// each of 32 rows).  REST: not the results but what rounding them leaves.
template <typename T, bool REST = false>
__device__ __forceinline__ void put_rows(uint8_t* out, const float (&v)[kPairEpiCols], T* p, int64_t ld, int rows,
                                         int cols) {
  const int lane = threadIdx.x & 31, c = lane & 7, r0 = lane >> 3;
  uint8_t* const mine = out + lane * 128;            // the row this lane puts down,
  const uint8_t* const even = out + r0 * 128 + ((c ^ r0) * 16);  // and its piece of rows r0 + 8 i
  const uint8_t* const odd = out + r0 * 128 + ((c ^ (r0 + 4)) * 16) + 512;  // and r0 + 8 i + 4
  T* at = p + r0 * ld + 8 * c;
#pragma unroll
  for (int h = 0; h < kPairEpiCols; h += 64) {
    if (h >= cols) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        w[j] = v[h + 8 * e + j];
        if (REST) w[j] -= to_f32<T>(from_f32<T>(w[j]));
      }
      store_f32<T, 8>(reinterpret_cast<T*>(mine + ((e ^ c) * 16)), w);
    }
    __syncwarp();
    const int n = cols - (h + 8 * c);
    T* dst = at + h;
    if (rows >= 32 && n >= 8) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint4 a = *reinterpret_cast<const uint4*>(even + i * 1024);
        const uint4 b = *reinterpret_cast<const uint4*>(odd + i * 1024);
        *reinterpret_cast<uint4*>(dst) = a;
        dst += 4 * ld;
        *reinterpret_cast<uint4*>(dst) = b;
        dst += 4 * ld;
      }
    } else {
#pragma unroll 1
      for (int r = r0; r < rows; r += 4, dst += 4 * ld) {
        if (r >= 32) break;
        const uint4 w = *reinterpret_cast<const uint4*>(out + r * 128 + ((c ^ (r & 7)) * 16));
        if (n >= 8) {
          *reinterpret_cast<uint4*>(dst) = w;
        } else {
          const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (j < n) dst[j] = e[j];
        }
      }
    }
    __syncwarp();
  }
}

// The same in fp32 (rows of p 16-byte aligned, room for whole groups of 4 columns), added to what is there unless `first`.
__device__ __forceinline__ void sum_rows(uint8_t* out, const float (&v)[kPairEpiCols], float* p, int64_t ld, int rows,
                                         int cols, bool first) {
  const int lane = threadIdx.x & 31, c = lane & 7, r0 = lane >> 3;
  uint8_t* const mine = out + lane * 128;
  const uint8_t* const even = out + r0 * 128 + ((c ^ r0) * 16);
  const int other = 512 + ((c ^ (r0 + 4)) - (c ^ r0)) * 16;  // to the same piece four rows on
  float* at = p + r0 * ld + 4 * c;
  const int last = min(rows, 32);
#pragma unroll
  for (int h = 0; h < kPairEpiCols; h += 32) {
    if (h >= cols) return;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      *reinterpret_cast<float4*>(mine + ((e ^ c) * 16)) =
          make_float4(v[h + 4 * e], v[h + 4 * e + 1], v[h + 4 * e + 2], v[h + 4 * e + 3]);
    __syncwarp();
    if (h + 4 * c < cols) {
      float* dst = at + h;
      const uint8_t* src = even;
#pragma unroll 1  // unrolled, its addresses do not stay in registers beside v
      for (int r = r0; r < last; r += 8, src += 1024) {
        float4 w = *reinterpret_cast<const float4*>(src);
        float4 u = *reinterpret_cast<const float4*>(src + other);
        float4* const to = reinterpret_cast<float4*>(dst);
        float4* const next = reinterpret_cast<float4*>(dst + 4 * ld);
        const bool two = r + 4 < last;
        if (!first) {
          const float4 o = *to;
          w = make_float4(w.x + o.x, w.y + o.y, w.z + o.z, w.w + o.w);
          if (two) {
            const float4 n = *next;
            u = make_float4(u.x + n.x, u.y + n.y, u.z + n.z, u.w + n.w);
          }
        }
        *to = w;
        if (two) *next = u;
        dst += 8 * ld;
      }
    }
    __syncwarp();
  }
}

// G of one piece of the vocabulary.  TWO: what its rounding leaves goes to the rows from `tokens` on.
template <typename T, bool TWO>
struct GradEpi {
  struct Args {
    T* g;              // [tokens][ldg]
    int64_t ldg;       // columns of the piece, a multiple of the tile
    const float* lse;
    const float* f;    // the token's factor, 0 where it does not count
    Targets ids;
    int tokens, vocab, v0;
    float scale;
  };
  const Args& a;
  int row, part, mt = -1;
  int64_t id = -1;
  float lse2 = 0.f, f = 0.f;

  uint8_t* out;

  __device__ GradEpi(const Args& args, int row_in_tile, int p, uint8_t* o) : a(args), row(row_in_tile), part(p), out(o) {}

  __device__ void tile(const PairTile& pt, float (&v)[kPairEpiCols]) {
    const int token = pt.mt * kPairTileM + row;
    const int token0 = token - static_cast<int>(threadIdx.x & 31);  // of the warp
    if (token0 >= a.tokens) return;
    if (pt.mt != mt) {
      mt = pt.mt;
      if (token < a.tokens) {
        id = a.ids[token];
        lse2 = a.lse[token] * kLog2e;
        f = a.f[token];
      }
    }
    const int col0 = pt.nt * kPairTileN + part * kPairEpiCols;  // in the piece
    const float k = a.scale * kLog2e;
    const int64_t at = id - (a.v0 + col0);
#pragma unroll
    for (int j = 0; j < kPairEpiCols; ++j) v[j] = ex2(fmaf(v[j], k, -lse2)) * f;
    bool large = __any_sync(0xffffffffu, at >= 0 && at < kPairEpiCols);
    if (large) {
#pragma unroll
      for (int j = 0; j < kPairEpiCols; ++j)
        if (at == j) v[j] -= f;
    }
    if constexpr (TWO) {
      float top = 0.f;
#pragma unroll
      for (int j = 0; j < kPairEpiCols; ++j) top = fmaxf(top, fabsf(v[j]));
      large |= __any_sync(0xffffffffu, top > kLargeProbability * fabsf(f));
    }
    // a token that does not count has no gradient, whatever its logits are
    const int n = f == 0.f ? 0 : a.vocab - (a.v0 + col0);
    if (n < kPairEpiCols) {
#pragma unroll
      for (int j = 0; j < kPairEpiCols; ++j)
        if (j >= n) v[j] = 0.f;
    }
    T* const p = a.g + static_cast<int64_t>(token0) * a.ldg + col0;
    put_rows<T>(out, v, p, a.ldg, a.tokens - token0, kPairEpiCols);
    if constexpr (TWO) {
      T* const rest = p + a.tokens * a.ldg;
      if (large) {
        put_rows<T, true>(out, v, rest, a.ldg, a.tokens - token0, kPairEpiCols);
      } else {
        constexpr int kPieces = kPairEpiCols * sizeof(T) / 16;  // of a row
        const int lane = threadIdx.x & 31, rows = min(32, a.tokens - token0);
        for (int r = lane / kPieces; r < rows; r += 32 / kPieces)
          reinterpret_cast<uint4*>(rest + r * a.ldg)[lane % kPieces] = make_uint4(0u, 0u, 0u, 0u);
      }
    }
  }

  __device__ void done() {}
};

// Sums times *factor as T, or, where k is split or comes in pieces, fp32 sums of each split
// (added to those of earlier pieces unless `first`), which k_join finishes.
template <typename T>
struct SumEpi {
  struct Args {
    T* out;            // rows 16-byte aligned
    int64_t ldo;
    float* acc;        // [splits][rows][ldacc], rows 16-byte aligned; NULL: to `out`
    int64_t ldacc;
    const float* factor;
    int rows, cols;
    int first;
  };
  const Args& a;
  int row, part;
  uint8_t* out;
  float factor;

  __device__ SumEpi(const Args& args, int row_in_tile, int p, uint8_t* o)
      : a(args), row(row_in_tile), part(p), out(o), factor(*args.factor) {}

  __device__ void tile(const PairTile& pt, float (&v)[kPairEpiCols]) {
    const int r0 = pt.mt * kPairTileM + row - static_cast<int>(threadIdx.x & 31);  // the warp's first
    const int col0 = pt.nt * kPairTileN + part * kPairEpiCols;
    const int rows = a.rows - r0, cols = a.cols - col0;
    if (rows <= 0 || cols <= 0) return;
    if (a.acc) {
      float* p = a.acc + (static_cast<int64_t>(pt.split) * a.rows + r0) * a.ldacc + col0;
      sum_rows(out, v, p, a.ldacc, rows, cols, a.first != 0);
    } else {
#pragma unroll
      for (int j = 0; j < kPairEpiCols; ++j) v[j] *= factor;
      put_rows<T>(out, v, a.out + static_cast<int64_t>(r0) * a.ldo + col0, a.ldo, rows, cols);
    }
  }

  __device__ void done() {}
};

// ------------------------------------------------------------ small kernels

enum Reduction : int { kNone = KAIRO_REDUCTION_NONE, kSum = KAIRO_REDUCTION_SUM, kMean = KAIRO_REDUCTION_MEAN };

// Sum of `v` over the CTA (any number of whole warps), in a fixed order; every thread gets it.
__device__ float cta_sum(float v) {
  __shared__ float w[32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) w[threadIdx.x >> 5] = v;
  __syncthreads();
  const int nw = blockDim.x >> 5;
  float t = (threadIdx.x & 31) < nw ? w[threadIdx.x & 31] : 0.f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  return t;
}

// lse and loss of 32 tokens a CTA from their partial maxima and sums; the CTA that finishes last
// reduces the losses, always in the same order.
__global__ void __launch_bounds__(1024) k_lse(const float2* __restrict__ part, int slots,
                                              const float* __restrict__ target, Targets ids, int tokens, int vocab,
                                              float scale, int reduction, float* __restrict__ each,
                                              float* __restrict__ lse, float* __restrict__ loss, unsigned* ticket) {
  __shared__ float2 sm[32][33];
  __shared__ bool last;
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
  const int t = blockIdx.x * 32 + x;
  float m = -INFINITY, s = 0.f;
  if (t < tokens) {
    auto join = [&](float2 p) {
      const float top = fmaxf(m, p.x);
      const float ref = top == -INFINITY ? 0.f : top;
      s = s * ex2(m - ref) + p.y * ex2(p.x - ref);
      m = top;
    };
    int i = y;
    for (; i + 96 < slots; i += 128) {
      float2 p[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) p[u] = part[static_cast<int64_t>(i + 32 * u) * tokens + t];
#pragma unroll
      for (int u = 0; u < 4; ++u) join(p[u]);
    }
    for (; i < slots; i += 32) join(part[static_cast<int64_t>(i) * tokens + t]);
  }
  sm[y][x] = make_float2(m, s);
  __syncthreads();
  if (y == 0 && t < tokens) {
    float top = m;
    for (int u = 1; u < 32; ++u) top = fmaxf(top, sm[u][x].x);
    const float ref = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    for (int u = 0; u < 32; ++u) sum += sm[u][x].y * ex2(sm[u][x].x - ref);
    // back from base 2 by what the logits were scaled with; in 64 bits, so that a small loss, the difference of
    // two large numbers, has no more of their rounding than v has
    const double high = scale == 0.f ? 0.0 : static_cast<double>(ref) * (fabs(static_cast<double>(scale)) / stats_scale(scale));
    const double rest = static_cast<double>(logf(sum));
    const int64_t id = ids[t];
    lse[t] = static_cast<float>(high + rest);
    each[t] = id >= 0 && id < vocab
                  ? static_cast<float>((high - static_cast<double>(target[t]) * static_cast<double>(scale)) + rest)
                  : 0.f;
  }
  if (reduction == kNone) return;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(ticket, 1u) == gridDim.x - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  float sum = 0.f, count = 0.f;
  for (int i = threadIdx.x; i < tokens; i += blockDim.x) {
    sum += __ldcg(each + i);
    const int64_t id = ids[i];
    count += id >= 0 && id < vocab ? 1.f : 0.f;
  }
  sum = cta_sum(sum);
  count = cta_sum(count);
  if (threadIdx.x == 0) *loss = reduction == kMean ? sum / fmaxf(count, 1.f) : sum;
}

// out = *factor * the splits' sums.  WAYS threads share the splits of 4 columns (their sums are added in
// a fixed order): one thread would wait for 64 of them in turn.
template <typename T, int WAYS>
__global__ void __launch_bounds__(256) k_join(const float* __restrict__ acc, int64_t ldacc, int splits, int64_t rows,
                                              int64_t cols, const float* __restrict__ factor, T* __restrict__ out,
                                              int64_t ldo) {
  const int64_t groups = (cols + 3) / 4, total = rows * groups;
  const float f = *factor;
  const int way = threadIdx.x % WAYS;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (256 / WAYS);
  for (int64_t i0 = static_cast<int64_t>(blockIdx.x) * (256 / WAYS); i0 < total; i0 += step) {
    const int64_t i = i0 + threadIdx.x / WAYS;
    const int64_t r = i / groups, c = (i - r * groups) * 4;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (i < total) {
#pragma unroll 8
      for (int k = way; k < splits; k += WAYS) {
        const float4 w = __ldcs(reinterpret_cast<const float4*>(acc + (k * rows + r) * ldacc + c));
        s = make_float4(s.x + w.x, s.y + w.y, s.z + w.z, s.w + w.w);
      }
    }
#pragma unroll
    for (int o = 1; o < WAYS; o <<= 1) {
      s.x += __shfl_xor_sync(0xffffffffu, s.x, o);
      s.y += __shfl_xor_sync(0xffffffffu, s.y, o);
      s.z += __shfl_xor_sync(0xffffffffu, s.z, o);
      s.w += __shfl_xor_sync(0xffffffffu, s.w, o);
    }
    if (i >= total || way != 0) continue;
    const float v[4] = {s.x * f, s.y * f, s.z * f, s.w * f};
    T* dst = out + r * ldo + c;
    if (c + 4 <= cols && reinterpret_cast<uintptr_t>(dst) % 8 == 0) {
      store_f32<T, 4>(dst, v);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c + j < cols) dst[j] = from_f32<T>(v[j]);
    }
  }
}

// Rows of 16-bit values with 16-byte alignment: dst (rows x ldd, ldd a multiple of 8) = src (its rows over
// and over where it has fewer), zeros behind column `cols` and, where `ids` is given, in the rows of tokens that do not count.
// CTA 0 writes the tokens' factors and the one they share (`factor`) first.
struct PrepArgs {
  const float* grad;  // by the loss: one number, or every token's (kNone)
  Targets ids;
  int tokens, vocab, reduction;
  float scale, lift;
  float* f;
  float* factor;
};

__device__ void prep_factors(const PrepArgs& p) {
  float count = 0.f, top = 0.f;
  for (int i = threadIdx.x; i < p.tokens; i += blockDim.x) {
    const int64_t id = p.ids[i];
    if (id >= 0 && id < p.vocab) {
      count += 1.f;
      // one that is not finite spoils its own token's G; the others keep their power of two
      if (p.reduction == kNone && isfinite(p.grad[i])) top = fmaxf(top, fabsf(p.grad[i]));
    }
  }
  float shared_factor;
  if (p.reduction == kNone) {
    // the largest factor's power of two, so that factors of any size keep their digits in 16 bits
    __shared__ float tops[32];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();
    for (int i = 0; i < static_cast<int>(blockDim.x >> 5); ++i) top = fmaxf(top, tops[i]);
    int e = 0;
    if (top > 0.f) frexpf(top, &e);
    shared_factor = ldexpf(1.f, max(-100, min(100, e)));
  } else {
    count = cta_sum(count);
    shared_factor = *p.grad / (p.reduction == kMean ? fmaxf(count, 1.f) : 1.f);
  }
  for (int i = threadIdx.x; i < p.tokens; i += blockDim.x) {
    const int64_t id = p.ids[i];
    const float own = p.reduction == kNone ? p.grad[i] / shared_factor : 1.f;
    p.f[i] = id >= 0 && id < p.vocab ? own * p.lift : 0.f;
  }
  if (threadIdx.x == 0) *p.factor = shared_factor * p.scale / p.lift;
}

// A power of two of lanes, 32 at most, takes a row of `pieces` vectors: no division per vector.
__device__ __forceinline__ int lanes_for(int64_t pieces) {
  int l = 1;
  while (l < 32 && l < pieces) l <<= 1;
  return l;
}

__global__ void __launch_bounds__(256) k_rows(const uint16_t* __restrict__ src, int64_t lds, int64_t src_rows,
                                              int64_t cols, int64_t rows, uint16_t* __restrict__ dst, int64_t ldd, Targets ids, int vocab,
                                              PrepArgs prep) {
  int cta = blockIdx.x, ctas = gridDim.x;
  if (prep.f) {
    if (cta == 0) return prep_factors(prep);
    --cta;
    --ctas;
  }
  const int64_t pieces = ldd / 8;
  const int lanes = lanes_for(pieces), per = 256 / lanes;
  const uint16_t* end = src + (src_rows - 1) * lds + cols;  // nothing is read outside [src, end)
  for (int64_t r = static_cast<int64_t>(cta) * per + threadIdx.x / lanes; r < rows; r += static_cast<int64_t>(ctas) * per) {
    bool live = true;
    if (ids.p) {
      const int64_t id = ids[r < src_rows ? r : r % src_rows];
      live = id >= 0 && id < vocab;
    }
    // four vectors at a time, so that their loads are under way together
    for (int64_t q0 = threadIdx.x % lanes; q0 < pieces; q0 += 4 * lanes) {
      uint4 lo[4], hi[4];
      bool whole[4];
      const uint16_t* row = src + (r < src_rows ? r : r % src_rows) * lds;
      // past a 16-byte boundary (the same for all vectors of a row)
      const int e = static_cast<int>((reinterpret_cast<uintptr_t>(row) >> 1) & 7u);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int64_t c = (q0 + u * lanes) * 8;
        const uint16_t* p = row + c - e;
        whole[u] = live && c + 8 <= cols && p >= src && p + (e ? 16 : 8) <= end;
        lo[u] = whole[u] ? __ldg(reinterpret_cast<const uint4*>(p)) : make_uint4(0u, 0u, 0u, 0u);
        hi[u] = whole[u] && e ? __ldg(reinterpret_cast<const uint4*>(p) + 1) : make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int64_t q = q0 + u * lanes, c = q * 8;
        if (q >= pieces) break;
        uint4 w = shift8(lo[u], hi[u], e);
        if (live && !whole[u]) {
          uint32_t h[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) h[j] = c + j < cols ? row[c + j] : 0u;
          w = make_uint4(h[0] | (h[1] << 16), h[2] | (h[3] << 16), h[4] | (h[5] << 16), h[6] | (h[7] << 16));
        }
        *reinterpret_cast<uint4*>(dst + r * ldd + c) = w;
      }
    }
  }
}

// The way back: rows of a 16-byte aligned src (pitch lds) to rows at any address.
__global__ void __launch_bounds__(256) k_rows_back(const uint16_t* __restrict__ src, int64_t lds, int64_t rows,
                                                   int64_t cols, uint16_t* __restrict__ dst, int64_t ldd) {
  const int64_t pieces = cols / 8 + 2;  // the values before the first 16-byte boundary, vectors, the rest
  const int lanes = lanes_for(pieces), per = 256 / lanes;
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * per + threadIdx.x / lanes; r < rows;
       r += static_cast<int64_t>(gridDim.x) * per) {
    const uint16_t* p = src + r * lds;
    uint16_t* d = dst + r * ldd;
    const int lead = static_cast<int>((8u - static_cast<unsigned>(reinterpret_cast<uintptr_t>(d) >> 1)) & 7u);
    for (int64_t q0 = threadIdx.x % lanes; q0 < pieces; q0 += 4 * lanes) {
      uint4 lo[4], hi[4];
      const int e = lead & 7;  // of every vector's first value past a 16-byte boundary of src
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int64_t q = q0 + u * lanes, e0 = lead + 8 * (q - 1);
        const bool whole = q > 0 && e0 + 8 <= cols;
        const uint4* at = reinterpret_cast<const uint4*>(p + (whole ? e0 - e : 0));
        lo[u] = whole ? __ldg(at) : make_uint4(0u, 0u, 0u, 0u);
        hi[u] = whole && e ? __ldg(at + 1) : make_uint4(0u, 0u, 0u, 0u);  // e0 + 8 <= cols <= lds: within the row
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int64_t q = q0 + u * lanes, e0 = lead + 8 * (q - 1);
        if (q >= pieces) break;
        if (q > 0 && e0 + 8 <= cols) {
          *reinterpret_cast<uint4*>(d + e0) = shift8(lo[u], hi[u], e);
        } else {
          const int64_t from = q == 0 ? 0 : e0, to = q == 0 ? min(static_cast<int64_t>(lead), cols) : cols;
          for (int64_t i = from; i < to; ++i) d[i] = p[i];
        }
      }
    }
  }
}

// ------------------------------------------------------------ host side

struct Problem {
  const void* x;
  int64_t ldx;
  const void* w;
  int64_t ldw;
  int64_t tokens, vocab, dim;
  kairo_dtype dt;
  Targets ids;
  float scale;
  int reduction;
};

bool rows_aligned(const void* p, int64_t ld, int64_t rows) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (ld % 8 == 0 || rows <= 1);
}

int64_t tiles(int64_t n) { return ceil_div64(n, kPairTileN); }

// Columns of one piece of the backward pass: pieces of equal size, whole tiles.
int64_t piece_cols(int64_t tokens, int64_t vocab) {
  const int64_t most = std::max<int64_t>(1, kPieceBytes / (2 * std::max<int64_t>(1, tokens) * kPairTileN)) * kPairTileN;
  const int64_t pieces = ceil_div64(vocab, most);
  return tiles(ceil_div64(vocab, pieces)) * kPairTileN;
}

constexpr int64_t kFewTokens = FewStatsEpi<2>::TOKENS;  // of the forward pass with the table down the rows

struct LossWs {
  size_t ticket, target, each, part, x, w, total;
};

// Rows of a few tokens are read by every SM at the same time, all from the same few lines of L2: copies of them
// for different clusters bring 1 to 15 tokens of 131072 x 4096 from 237..261 us to what 16 take, 200.
constexpr int64_t kCopyRows = 64;
int64_t copies_of(int64_t tokens) { return tokens < 16 ? kCopyRows / tokens : 1; }

// Rows of copies begin on 128-byte lines: a box of 64 k of a row then touches one line, not two (4000 tokens, 50021 x
// 1000: 337 us, 302 with such a pitch; a copy of the table for that alone would cost what it saves).
int64_t copy_ld(int64_t dim) { return static_cast<int64_t>(align_up(static_cast<size_t>(dim), 64)); }

// Everything a call may need: the copies come last.
LossWs loss_ws(const Problem& p) {
  LossWs o{};
  size_t at = kWorkspaceHeaderBytes;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at = align_up(at + bytes, 256);
    return here;
  };
  o.ticket = 128;
  o.target = take(4 * static_cast<size_t>(p.tokens));
  o.each = take(4 * static_cast<size_t>(p.tokens));
  const int64_t slots =
      p.tokens <= kFewTokens ? 8 * std::min<int64_t>(kPairClusters, tiles(p.vocab)) : 2 * tiles(p.vocab);
  o.part = take(8 * static_cast<size_t>(p.tokens) * static_cast<size_t>(slots));
  const size_t ld = static_cast<size_t>(copy_ld(p.dim));
  const int64_t copies = copies_of(std::max<int64_t>(1, p.tokens));
  if (copies > 1 || !rows_aligned(p.x, p.ldx, p.tokens)) o.x = take(2 * ld * static_cast<size_t>(p.tokens * copies));
  if (!rows_aligned(p.w, p.ldw, p.vocab)) o.w = take(2 * ld * static_cast<size_t>(p.vocab));
  o.total = at;
  return o;
}

struct Results {
  void* dx;
  int64_t lddx;
  void* dw;
  int64_t lddw;
};

// Rows of G, of X beside it and of dX's sums for each token.  A single token's dW is its entries of G times its X, and a
// dX is mostly its target's row of the table: G's rounding then stands in the result at full size.  Up to 128 tokens, whose
// tiles have the rows and the k to spare, a second row holds what the first one's rounding left (bf16, 100000 x 1024: 16
// tokens 221 -> 230 us, 64 229 -> 248, 128 247 -> 287; the gradients' error 1.4 to 2 times that of one rounding -> 1.0).
int64_t halves(int64_t tokens) { return tokens <= kPairTileM / 2 ? 2 : 1; }

struct GradWs {
  size_t f, factor, acc_x, acc_w, x, w, g, out, total;
  int64_t rows, cols;  // of G
  int splits_x, splits_w;  // parts of the vocabulary piece for dX, of the tokens for dW
  bool direct_x;           // dX leaves from its product
};

// Parts of k for a product of rows x cols: tiles that fill the clusters' rounds evenly, against the fp32
// sums of each part, written and read once more.  In stages of one tile (about 0.27 us); a tile costs 8
// beside its k (filling the pipeline, the epilogue's end).
int splits_for(int64_t rows, int64_t cols, int64_t k) {
  const int64_t t = tiles(rows) * tiles(cols), steps = ceil_div64(k, kPairK);
  const double again = 8.0 * static_cast<double>(rows) * static_cast<double>(cols) / 6.5e12 / 0.27e-6;
  int best = 1;
  double least = 0.0;
  for (int s = 1; s <= 64 && s <= steps; ++s) {
    const double cost = static_cast<double>(ceil_div64(t * s, kPairClusters) * (ceil_div64(steps, s) + 8)) +
                        (s > 1 ? again * s + 10.0 : 0.0);
    if (s == 1 || cost < least) {
      least = cost;
      best = s;
    }
  }
  return best;
}

// A dX whose rows are not 16-byte aligned leaves as fp32 sums and k_join, such a dW through a copy.
GradWs grad_ws(const Problem& p, const Results& r) {
  GradWs o{};
  size_t at = kWorkspaceHeaderBytes;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at = align_up(at + bytes, 256);
    return here;
  };
  const size_t ld = static_cast<size_t>(copy_ld(p.dim));
  o.rows = halves(p.tokens) * p.tokens;
  o.cols = piece_cols(o.rows, p.vocab);
  o.factor = 128;
  o.f = take(4 * static_cast<size_t>(p.tokens));
  o.x = take(2 * ld * static_cast<size_t>(o.rows));
  o.splits_x = splits_for(o.rows, p.dim, std::min(o.cols, p.vocab));
  o.splits_w = splits_for(std::min(o.cols, p.vocab), p.dim, o.rows);
  o.direct_x = o.rows == p.tokens && o.cols >= p.vocab && o.splits_x == 1 && rows_aligned(r.dx, r.lddx, p.tokens);
  if (r.dx && !o.direct_x) o.acc_x = take(4 * ld * static_cast<size_t>(o.rows) * o.splits_x);
  if (r.dw && o.splits_w > 1) o.acc_w = take(4 * ld * static_cast<size_t>(std::min(o.cols, p.vocab)) * o.splits_w);
  if (!rows_aligned(p.w, p.ldw, p.vocab)) o.w = take(2 * ld * static_cast<size_t>(p.vocab));
  if (r.dw && o.splits_w == 1 && !rows_aligned(r.dw, r.lddw, p.vocab))
    o.out = take(2 * ld * static_cast<size_t>(std::min(o.cols, p.vocab)));
  o.g = take(2 * static_cast<size_t>(o.rows) * static_cast<size_t>(o.cols));
  o.total = at;
  return o;
}

kairo_status check_problem(const Problem& p) {
  if (p.tokens < 0 || p.vocab < 1 || p.dim < 1) return fail(KAIRO_STATUS_INVALID_VALUE, "invalid size");
  if (p.tokens > 0x7fffff00LL || p.vocab > 0x7fffff00LL || p.dim > 0x7fffff00LL ||
      tiles(p.tokens) * tiles(p.vocab) > 0x7fffffffLL || tiles(p.dim) * tiles(std::max(p.tokens, p.vocab)) > 0x7fffffffLL)
    return fail(KAIRO_STATUS_NOT_SUPPORTED, "sizes beyond 2^31 tiles");
  if (p.dt != KAIRO_DTYPE_F16 && p.dt != KAIRO_DTYPE_BF16)
    return fail(KAIRO_STATUS_INVALID_VALUE, "hidden states and table must be f16 or bf16");
  if (p.ldx < p.dim || p.ldw < p.dim) return fail(KAIRO_STATUS_INVALID_VALUE, "leading dimension too small");
  if (p.reduction < kNone || p.reduction > kMean) return fail(KAIRO_STATUS_INVALID_VALUE, "unknown reduction");
  if (p.ids.bytes != 4 && p.ids.bytes != 8) return fail(KAIRO_STATUS_INVALID_VALUE, "targets must be int32 or int64");
  return KAIRO_STATUS_SUCCESS;
}

kairo_status copy_rows(const void* src, int64_t ld, int64_t rows, int64_t cols, int64_t copies, uint8_t* dst,
                       Targets ids, int vocab, const PrepArgs& prep, cudaStream_t s) {
  const int64_t ldd = copy_ld(cols);
  const int64_t work = ceil_div64(rows * copies * (ldd / 8), 256);
  const int grid = static_cast<int>(std::min<int64_t>(work, device_sm_count(current_device()) * 16)) + (prep.f ? 1 : 0);
  k_rows<<<grid, 256, 0, s>>>(static_cast<const uint16_t*>(src), ld, rows, cols, rows * copies,
                              reinterpret_cast<uint16_t*>(dst), ldd, ids, vocab, prep);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? KAIRO_STATUS_SUCCESS : cuda_fail(e, "launch of the row copy");
}

// `src` with 16-byte aligned rows: itself, or a copy at `dst`.
kairo_status aligned_rows(const void** src, int64_t* ld, int64_t rows, int64_t cols, uint8_t* dst, cudaStream_t s) {
  if (rows_aligned(*src, *ld, rows)) return KAIRO_STATUS_SUCCESS;
  const kairo_status st = copy_rows(*src, *ld, rows, cols, 1, dst, Targets{nullptr, 8}, 0, PrepArgs{}, s);
  *src = dst;
  *ld = copy_ld(cols);
  return st;
}

// Rows of tiles visited together: their part of the row operand takes about a quarter of the L2.
int group_rows(int64_t tiles_m, int64_t k) {
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(tiles_m, (32LL << 20) / (kPairTileM * 2 * std::max<int64_t>(k, 64)))));
}

// Stages of a segment.  A loss is the difference of lse and a logit, a fraction of either: 384 k of a logit, and 128 or
// 256 for up to 64 or 128 tokens, which wait for the table all the same, leave a loss about as exact as fp32 products do
// (512 k: 3.5e-6 of the loss of a single token, which is rarely averaged out; 64 k: 64 tokens of 131072 x 4096 241 us
// instead of 197; 256 k: 1024 tokens 824 us, 512 k: 750).  Logits formed again for G: 512 k.  The gradients are
// rounded to 16 bits: 4096 k leave 1e-5.
constexpr int kSegLogits = 6, kSegFew = 2, kSegAgain = 8, kSegGrads = 64;

PairShape shape_of(int64_t rows, int64_t cols, int64_t k, int seg, int splits = 1) {
  PairShape s;
  s.seg = seg;
  s.splits = splits;
  s.copies = 1;
  s.copy_rows = 0;
  s.tiles_m = static_cast<int>(tiles(rows));
  s.tiles_n = static_cast<int>(tiles(cols));
  s.ksteps = static_cast<int>(ceil_div64(k, kPairK));
  s.group_m = group_rows(s.tiles_m, k);
  return s;
}

template <typename T>
kairo_status join(const float* acc, int64_t ldacc, int splits, int64_t rows, int64_t cols, const float* factor, T* out,
                  int64_t ldo, cudaStream_t s) {
  const int64_t groups = rows * ceil_div64(cols, 4);
  const int64_t most = device_sm_count(current_device()) * 16;
  if (splits >= 8)
    k_join<T, 8><<<static_cast<int>(std::min<int64_t>(ceil_div64(groups, 32), most)), 256, 0, s>>>(
        acc, ldacc, splits, rows, cols, factor, out, ldo);
  else
    k_join<T, 1><<<static_cast<int>(std::min<int64_t>(ceil_div64(groups, 256), most)), 256, 0, s>>>(
        acc, ldacc, splits, rows, cols, factor, out, ldo);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? KAIRO_STATUS_SUCCESS : cuda_fail(e, "launch of k_join");
}

template <typename T, int FMT>
kairo_status run_loss(Problem p, float* loss, float* lse, uint8_t* ws, unsigned* err, cudaStream_t s) {
  const LossWs o = loss_ws(p);
  const int64_t copies = copies_of(p.tokens);
  kairo_status st;
  if (copies > 1) {
    st = copy_rows(p.x, p.ldx, p.tokens, p.dim, copies, ws + o.x, Targets{nullptr, 8}, 0, PrepArgs{}, s);
    p.x = ws + o.x;
    p.ldx = copy_ld(p.dim);
  } else {
    st = aligned_rows(&p.x, &p.ldx, p.tokens, p.dim, ws + o.x, s);
  }
  if (st == KAIRO_STATUS_SUCCESS) st = aligned_rows(&p.w, &p.ldw, p.vocab, p.dim, ws + o.w, s);
  if (st) return st;
  unsigned* ticket = reinterpret_cast<unsigned*>(ws + o.ticket);
  float2* part = reinterpret_cast<float2*>(ws + o.part);
  float* target = reinterpret_cast<float*>(ws + o.target);
  const int tokens = static_cast<int>(p.tokens), vocab = static_cast<int>(p.vocab);
  const bool few = p.tokens <= kFewTokens;
  // tiles of 128 columns take as long as of 64, but draw more power: 64 tokens of 131072 x 4096, called one after
  // the other, 218 us against 185
  const bool half = p.tokens <= FewStatsEpi<1>::TOKENS;
  CUtensorMap mx, mw;
  st = pair_operand_map(&mx, p.x, p.dt, false, p.tokens * copies, p.dim, p.ldx, "hidden states",
                        few ? (half ? FewStatsEpi<1>::TOKENS : FewStatsEpi<2>::TOKENS) / 2 : kPairBoxRows);
  if (st == KAIRO_STATUS_SUCCESS) st = pair_operand_map(&mw, p.w, p.dt, false, p.vocab, p.dim, p.ldw, "vocabulary table");
  if (st) return st;
  int slots;
  if (few) {
    PairShape sh = shape_of(p.vocab, 1, p.dim, half ? kSegFew : 2 * kSegFew);
    sh.copies = static_cast<int>(copies);
    sh.copy_rows = tokens;
    slots = 8 * pair_clusters(sh.tiles_m);
    if (slots > 8 * kPairClusters) return fail(KAIRO_STATUS_NOT_SUPPORTED, "more SMs than the workspace is laid out for");
    auto go = [&](auto groups) {
      using Epi = FewStatsEpi<decltype(groups)::value>;
      const typename Epi::Args a{part, target, p.ids, tokens, vocab, p.scale, ticket};
      return launch_pair_gemm<FMT, false, false, Epi, Epi::TOKENS>(mw, mx, sh, err, a, s);
    };
    st = half ? go(std::integral_constant<int, 1>{}) : go(std::integral_constant<int, 2>{});
  } else {
    const PairShape sh = shape_of(p.tokens, p.vocab, p.dim, kSegLogits);
    const StatsEpi::Args a{part, target, p.ids, tokens, vocab, p.scale, sh.tiles_m == 1, ticket};
    slots = 2 * (a.by_cluster ? pair_clusters(sh.tiles_n) : sh.tiles_n);
    st = launch_pair_gemm<FMT, false, false, StatsEpi>(mx, mw, sh, err, a, s);
  }
  if (st) return st;
  k_lse<<<static_cast<int>(ceil_div64(p.tokens, 32)), 1024, 0, s>>>(
      part, slots, target, p.ids, tokens, vocab, p.scale, p.reduction,
      p.reduction == kNone ? loss : reinterpret_cast<float*>(ws + o.each), lse, loss, ticket);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? KAIRO_STATUS_SUCCESS : cuda_fail(e, "launch of k_lse");
}

template <typename T, int FMT>
kairo_status run_grad(Problem p, const float* grad, const float* lse, const Results& res, uint8_t* ws, unsigned* err,
                      cudaStream_t s) {
  const GradWs o = grad_ws(p, res);
  T *dx = static_cast<T*>(res.dx), *dw = static_cast<T*>(res.dw);
  const int64_t ld = copy_ld(p.dim);
  kairo_status st = aligned_rows(&p.w, &p.ldw, p.vocab, p.dim, ws + o.w, s);
  if (st) return st;
  float* f = reinterpret_cast<float*>(ws + o.f);
  float* factor = reinterpret_cast<float*>(ws + o.factor);
  void* x = ws + o.x;
  {
    PrepArgs pa{grad, p.ids, static_cast<int>(p.tokens), static_cast<int>(p.vocab), p.reduction, p.scale,
                FMT == 0 ? kHalfLift : 1.f, f, factor};
    st = copy_rows(p.x, p.ldx, p.tokens, p.dim, o.rows / p.tokens, ws + o.x, p.ids, static_cast<int>(p.vocab), pa, s);
    if (st) return st;
  }
  T* g = reinterpret_cast<T*>(ws + o.g);
  CUtensorMap mx, mxt, mg, mgt;
  st = pair_operand_map(&mx, x, p.dt, false, p.tokens, p.dim, ld, "hidden states");
  if (st == KAIRO_STATUS_SUCCESS) st = pair_operand_map(&mxt, x, p.dt, true, p.dim, o.rows, ld, "hidden states");
  if (st == KAIRO_STATUS_SUCCESS) st = pair_operand_map(&mg, g, p.dt, false, o.rows, o.cols, o.cols, "gradient of the logits");
  if (st == KAIRO_STATUS_SUCCESS) st = pair_operand_map(&mgt, g, p.dt, true, o.cols, o.rows, o.cols, "gradient of the logits");
  if (st) return st;
  for (int64_t v0 = 0; v0 < p.vocab; v0 += o.cols) {
    const int64_t n = std::min(o.cols, p.vocab - v0);
    const T* w = static_cast<const T*>(p.w) + v0 * p.ldw;
    CUtensorMap mw, mwt;
    st = pair_operand_map(&mw, w, p.dt, false, n, p.dim, p.ldw, "vocabulary table");
    if (st == KAIRO_STATUS_SUCCESS) st = pair_operand_map(&mwt, w, p.dt, true, p.dim, n, p.ldw, "vocabulary table");
    if (st) return st;
    auto form = [&](auto two) {
      using Epi = GradEpi<T, decltype(two)::value>;
      const typename Epi::Args ga{g, o.cols, lse, f, p.ids, static_cast<int>(p.tokens), static_cast<int>(p.vocab),
                                  static_cast<int>(v0), p.scale};
      return launch_pair_gemm<FMT, false, false, Epi>(mx, mw, shape_of(p.tokens, n, p.dim, kSegAgain), err, ga, s);
    };
    st = o.rows > p.tokens ? form(std::true_type{}) : form(std::false_type{});
    if (st) return st;
    if (dx) {
      // a last piece of few columns has fewer parts than the others: those it leaves out keep their sums
      const int splits = static_cast<int>(std::min<int64_t>(o.splits_x, ceil_div64(n, kPairK)));
      typename SumEpi<T>::Args sa{dx, res.lddx, o.direct_x ? nullptr : reinterpret_cast<float*>(ws + o.acc_x), ld,
                                  factor, static_cast<int>(o.rows), static_cast<int>(p.dim), v0 == 0};
      st = launch_pair_gemm<FMT, false, true, SumEpi<T>>(mg, mwt, shape_of(o.rows, p.dim, n, kSegGrads, splits), err,
                                                         sa, s);
      if (st == KAIRO_STATUS_SUCCESS && !o.direct_x && v0 + n == p.vocab)
        // a token's second row lies as another part's row of it would
        st = join<T>(sa.acc, ld, o.splits_x * static_cast<int>(o.rows / p.tokens), p.tokens, p.dim, factor, dx, res.lddx, s);
      if (st) return st;
    }
    if (dw) {
      T* out = dw + v0 * res.lddw;
      const bool copy = o.splits_w == 1 && !rows_aligned(dw, res.lddw, p.vocab);
      typename SumEpi<T>::Args sa{copy ? reinterpret_cast<T*>(ws + o.out) : out, copy ? ld : res.lddw,
                                  o.splits_w > 1 ? reinterpret_cast<float*>(ws + o.acc_w) : nullptr, ld,
                                  factor, static_cast<int>(n), static_cast<int>(p.dim), 1};
      st = launch_pair_gemm<FMT, true, true, SumEpi<T>>(mgt, mxt, shape_of(n, p.dim, o.rows, kSegGrads, o.splits_w),
                                                        err, sa, s);
      if (st == KAIRO_STATUS_SUCCESS && sa.acc) st = join<T>(sa.acc, ld, o.splits_w, n, p.dim, factor, out, res.lddw, s);
      if (st) return st;
      if (copy) {
        const int grid = static_cast<int>(std::min<int64_t>(ceil_div64(n, 8), device_sm_count(current_device()) * 16));
        k_rows_back<<<grid, 256, 0, s>>>(reinterpret_cast<const uint16_t*>(sa.out), ld, n, p.dim,
                                         reinterpret_cast<uint16_t*>(out), res.lddw);
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return cuda_fail(e, "launch of the row copy");
      }
    }
  }
  return KAIRO_STATUS_SUCCESS;
}

}  // namespace
}  // namespace kairo

using namespace kairo;

extern "C" kairo_status kairo_vocab_loss_workspace_size(const void* x, int64_t ldx, const void* w, int64_t ldw,
                                                        int64_t tokens, int64_t vocab, int64_t dim, size_t* bytes) {
  if (!bytes) return fail(KAIRO_STATUS_INVALID_VALUE, "null argument");
  const Problem p{x, ldx, w, ldw, tokens, vocab, dim, KAIRO_DTYPE_BF16, Targets{nullptr, 8}, 1.f, kNone};
  const kairo_status st = check_problem(p);
  if (st) return st;
  *bytes = loss_ws(p).total;
  return KAIRO_STATUS_SUCCESS;
}

extern "C" kairo_status kairo_vocab_loss_backward_workspace_size(const void* w, int64_t ldw, int64_t tokens,
                                                                 int64_t vocab, int64_t dim, void* dx, int64_t lddx,
                                                                 void* dw, int64_t lddw, size_t* bytes) {
  if (!bytes) return fail(KAIRO_STATUS_INVALID_VALUE, "null argument");
  const Problem p{nullptr, dim, w, ldw, tokens, vocab, dim, KAIRO_DTYPE_BF16, Targets{nullptr, 8}, 1.f, kNone};
  const kairo_status st = check_problem(p);
  if (st) return st;
  *bytes = grad_ws(p, Results{dx, lddx, dw, lddw}).total;
  return KAIRO_STATUS_SUCCESS;
}

extern "C" kairo_status kairo_vocab_loss(const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t tokens,
                                         int64_t vocab, int64_t dim, kairo_dtype dtype, const void* targets,
                                         int32_t target_bytes, float scale, int32_t reduction, float* loss, float* lse,
                                         void* workspace, size_t workspace_bytes, unsigned* error_word, void* stream) {
  const Problem p{x, ldx, w, ldw, tokens, vocab, dim, dtype, Targets{targets, target_bytes}, scale, reduction};
  kairo_status st = check_problem(p);
  if (st) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (tokens == 0) {
    if (reduction == kNone) return KAIRO_STATUS_SUCCESS;
    if (!loss) return fail(KAIRO_STATUS_INVALID_VALUE, "null pointer argument");
    const cudaError_t e = cudaMemsetAsync(loss, 0, sizeof(float), s);
    return e == cudaSuccess ? KAIRO_STATUS_SUCCESS : cuda_fail(e, "cudaMemsetAsync(loss)");
  }
  if (!x || !w || !targets || !loss || !lse || !workspace || !error_word)
    return fail(KAIRO_STATUS_INVALID_VALUE, "null pointer argument");
  if (reinterpret_cast<uintptr_t>(workspace) % 256) return fail(KAIRO_STATUS_INVALID_VALUE, "workspace must be 256-byte aligned");
  if (workspace_bytes < loss_ws(p).total) return fail(KAIRO_STATUS_WORKSPACE_TOO_SMALL, "loss workspace too small");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  return dtype == KAIRO_DTYPE_F16 ? run_loss<__half, 0>(p, loss, lse, ws, error_word, s)
                                  : run_loss<__nv_bfloat16, 1>(p, loss, lse, ws, error_word, s);
}

extern "C" kairo_status kairo_vocab_loss_backward(const float* grad, const void* x, int64_t ldx, const void* w,
                                                  int64_t ldw, int64_t tokens, int64_t vocab, int64_t dim,
                                                  kairo_dtype dtype, const void* targets, int32_t target_bytes,
                                                  float scale, int32_t reduction, const float* lse, void* dx,
                                                  int64_t lddx, void* dw, int64_t lddw, void* workspace,
                                                  size_t workspace_bytes, unsigned* error_word, void* stream) {
  const Problem p{x, ldx, w, ldw, tokens, vocab, dim, dtype, Targets{targets, target_bytes}, scale, reduction};
  kairo_status st = check_problem(p);
  if (st) return st;
  if ((dx && lddx < dim) || (dw && lddw < dim)) return fail(KAIRO_STATUS_INVALID_VALUE, "leading dimension too small");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (!dx && !dw) return KAIRO_STATUS_SUCCESS;
  if (tokens == 0) {
    if (!dw) return KAIRO_STATUS_SUCCESS;
    const cudaError_t e = cudaMemset2DAsync(dw, static_cast<size_t>(lddw) * 2, 0, static_cast<size_t>(dim) * 2,
                                            static_cast<size_t>(vocab), s);
    return e == cudaSuccess ? KAIRO_STATUS_SUCCESS : cuda_fail(e, "cudaMemset2DAsync(dW)");
  }
  if (!grad || !x || !w || !targets || !lse || !workspace || !error_word)
    return fail(KAIRO_STATUS_INVALID_VALUE, "null pointer argument");
  if (reinterpret_cast<uintptr_t>(workspace) % 256) return fail(KAIRO_STATUS_INVALID_VALUE, "workspace must be 256-byte aligned");
  const Results res{dx, lddx, dw, lddw};
  if (workspace_bytes < grad_ws(p, res).total) return fail(KAIRO_STATUS_WORKSPACE_TOO_SMALL, "loss workspace too small");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  return dtype == KAIRO_DTYPE_F16
             ? run_grad<__half, 0>(p, grad, lse, res, ws, error_word, s)
             : run_grad<__nv_bfloat16, 1>(p, grad, lse, res, ws, error_word, s);
}
