// Low-rank adapters of many requests in one batch, beside a shared projection.
//
//   low[t]  = scale_a * X[t] down_a^T            (rank values, fp32)
//   Y[t]    = base[t] + low[t] up_a              a = the adapter of token t
// with down (G, rank, K) and up (G, rank, N): both stored rank row by rank
// row, so that the backward pass is the same product with the two swapped
//   dlow[t] = scale_a * dY[t] up_a^T,   dX[t] = base_dX[t] + dlow[t] down_a
// and both weight gradients are one contraction over an adapter's tokens
//   ddown_a = sum_t dlow[t]^T X[t],     dup_a = sum_t low[t]^T dY[t].
// A token without an adapter keeps Y = base.
//
// The plan of a batch (kairo_adapter_plan_build) orders the tokens by adapter
// on the device; every layer of a model uses it.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "adapters_kernel.cuh"
#include "internal.h"

namespace kairo {
namespace {

// Plan memory, int32 words: the number of tiles of 16, 32 and 64 tokens, the
// token order (T), starts (G + 2: the tokens of adapter a are order[starts[a]
// .. starts[a + 1]), those without one order[starts[G] .. starts[G + 1])), for
// each tile size the first tile of every adapter (G + 2), and the tiles.
constexpr int kTileSizes = 3;
__host__ __device__ constexpr int tile_tokens(int which) { return 16 << which; }

struct Plan {
  int32_t* ntiles;
  int32_t* order;
  int32_t* starts;
  int32_t* first[kTileSizes];
  LowRankTile* tiles[kTileSizes];
};

// Tiles of `size` tokens that a batch can have: whole ones, and a rest per
// group of tokens (G adapters, and those without).
int64_t max_tiles(int64_t t, int64_t g, int size) { return t / size + std::min(t, g + 1); }

size_t carve_plan(void* mem, int64_t t, int64_t g, Plan* pl) {
  int32_t* p = static_cast<int32_t*>(mem);
  size_t at = 64;
  auto take = [&](int64_t words) {
    int32_t* q = p ? p + at : nullptr;
    at += align_up(static_cast<size_t>(words), 64);
    return q;
  };
  Plan q{};
  q.ntiles = p;
  q.order = take(t);
  q.starts = take(g + 2);
  for (int i = 0; i < kTileSizes; ++i) q.first[i] = take(g + 2);
  for (int i = 0; i < kTileSizes; ++i)
    q.tiles[i] = reinterpret_cast<LowRankTile*>(take(max_tiles(t, g, tile_tokens(i)) * 4));
  if (pl) *pl = q;
  return at * sizeof(int32_t);
}

// The tiles of one size (blockIdx.x) from the sorted ids: where each adapter's
// tokens start, how many tiles come before its own, and the tiles themselves.
__global__ void __launch_bounds__(1024) k_plan_tiles(const uint32_t* __restrict__ sorted, int64_t t, int64_t g,
                                                     Plan pl) {
  __shared__ int sums[32];
  __shared__ int carry;
  __shared__ int begins[1024 + 1];  // of the adapters of one turn
  const int which = blockIdx.x;
  const int size = tile_tokens(which);
  int32_t* first = which == 0 ? pl.first[0] : (which == 1 ? pl.first[1] : pl.first[2]);
  LowRankTile* tiles = which == 0 ? pl.tiles[0] : (which == 1 ? pl.tiles[1] : pl.tiles[2]);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto start_of = [&](int64_t a) {  // first position whose id is >= a
    int64_t lo = 0, hi = t;
    while (lo < hi) {
      const int64_t mid = (lo + hi) >> 1;
      if (sorted[mid] < static_cast<uint32_t>(a)) lo = mid + 1;
      else hi = mid;
    }
    return static_cast<int>(lo);
  };
  if (threadIdx.x == 0) carry = 0;
  __syncthreads();
  for (int64_t base = 0; base <= g; base += 1024) {
    const int64_t a = base + threadIdx.x;  // g: tokens without an adapter
    int v = 0;
    begins[threadIdx.x] = a <= g ? start_of(a) : static_cast<int>(t);
    if (threadIdx.x == 1023) begins[1024] = a < g ? start_of(a + 1) : static_cast<int>(t);
    __syncthreads();
    if (a <= g) {
      const int p0 = begins[threadIdx.x], p1 = begins[threadIdx.x + 1];
      v = (p1 - p0 + size - 1) / size;
      if (which == 0) {
        pl.starts[a] = p0;
        if (a == g) pl.starts[g + 1] = p1;
      }
    }
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) sums[warp] = x;
    __syncthreads();
    if (warp == 0) {
      int w = sums[lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += y;
      }
      sums[lane] = w;
    }
    __syncthreads();
    const int incl = carry + x + (warp ? sums[warp - 1] : 0);
    if (a <= g) first[a] = incl - v;
    __syncthreads();
    if (threadIdx.x == 1023) carry = incl;
    __syncthreads();
  }
  const int n = carry;
  if (threadIdx.x == 0) {
    first[g + 1] = n;
    pl.ntiles[which] = n;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += 1024) {
    int64_t lo = 0, hi = g;  // the adapter a with first[a] <= i < first[a + 1]
    while (lo < hi) {
      const int64_t mid = (lo + hi) >> 1;
      if (first[mid + 1] <= i) lo = mid + 1;
      else hi = mid;
    }
    // the last turn's are still there
    const int64_t turn = g / 1024 * 1024;
    const int p0 = lo >= turn ? begins[lo - turn] : start_of(lo);
    const int p1 = lo >= turn ? begins[lo - turn + 1] : start_of(lo + 1);
    LowRankTile tile;
    tile.adapter = lo < g ? static_cast<int32_t>(lo) : -1;
    tile.begin = p0 + (i - first[lo]) * size;
    tile.count = min(size, p1 - tile.begin);
    tile.pad = 0;
    tiles[i] = tile;
  }
}

constexpr int64_t kMaxAdapters = 65535;
constexpr int64_t kMaxRank = 128;
constexpr int kCluster = 8;        // CTAs that share a tile
constexpr int kChunkTokens = 64;   // tokens of one step of the weight gradient

kairo_status check_low_rank(int64_t t, int64_t k, int64_t n, int64_t rank, int64_t g, kairo_dtype dtype) {
  if (t < 0 || k <= 0 || n <= 0 || rank <= 0 || g < 0) return fail(KAIRO_STATUS_INVALID_VALUE, "invalid size");
  if (dtype != KAIRO_DTYPE_F16 && dtype != KAIRO_DTYPE_BF16)
    return fail(KAIRO_STATUS_INVALID_VALUE, "adapters must be f16 or bf16");
  if (rank > kMaxRank) return fail(KAIRO_STATUS_NOT_SUPPORTED, "rank above 128");
  if (g > kMaxAdapters) return fail(KAIRO_STATUS_NOT_SUPPORTED, "more than 65535 adapters");
  if (t > (int64_t(1) << 24)) return fail(KAIRO_STATUS_NOT_SUPPORTED, "more than 2^24 tokens");
  if (k > (int64_t(1) << 22) || n > (int64_t(1) << 22)) return fail(KAIRO_STATUS_NOT_SUPPORTED, "features above 2^22");
  return KAIRO_STATUS_SUCCESS;
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Tokens per tile.  Small batches want many short tiles (one CTA cluster each)
// for latency; long ones want tiles as tall as the accumulators allow,
// because every tile reads its adapter's weights from L2 once.  Best clusters, 8
// adapters, 4096 features: rank 16, 1024 tokens 9.1 us with tiles of 16 and
// 13.0 with 64, 2048 tokens 12.8 and 14.0, 4096 tokens 22.8 and 22.4; rank 32,
// 2048 tokens 17.3 and 17.6 (with 32), and 8192 tokens of 8192 features 117
// and 96; rank 64, 1024 tokens 19.0 and 24.2, 4096 tokens 48.5 and 39.6; rank 128,
// 4096 tokens 94.8 and 75.5 (with 32).  An fp32 base takes twice the room of
// its loads, one CTA per SM instead of two for the tall tiles of small ranks, and
// more time than the weights: 8192 features, 4096 tokens of 4 adapters, rank 16
// 82 us with tiles of 16 and 88 with 64, rank 32 88 and 94 (with 32), rank 64
// 119 and 96 (with 32); 2100 tokens of 4096 features, rank 16 29 and 49.
// Contractions that are summed in parts have tiles of 16 only: 4096 tokens, rank 16,
// 131080 features 334 us (with 64, in one sum, 258), 262144 455 (801).
int pick_tile(int64_t t, int64_t k, int64_t rank, bool vec, bool base_f32) {
  if (!vec || t <= 2048 || k > lowrank::kLongFeatures) return 16;
  if (base_f32) return rank > 32 && rank <= 64 ? 32 : 16;
  if (rank <= 16) return 64;
  if (rank <= 32) return 32;
  return rank <= 64 ? 64 : 32;
}

// CTAs per tile, a power of two up to 8.  As many as the GPU holds at once (two
// CTAs per SM; one where the low tile is large) gives the shortest calls: 96 tokens in 71 tiles of 8192
// features took 20.2, 12.8, 12.3 and 15.7 us with clusters of 1, 2, 4 and 8;
// 8192 tokens in 260 tiles 96, 103, 101 and 124 us. But no more than leave
// every warp a turn of 64 features (777 tokens, 1000 features: 6.1 us with
// two, 12.3 with eight), and where the contraction is so long that a warp has
// 32 turns, more, shorter CTAs even out the SMs (8192 tokens, 32768 features:
// 142 us with two, 139 with four).
int pick_cluster(int64_t t, int64_t g, int tile, int64_t k, int64_t n, int64_t rank) {
  // Half a tile is lost per adapter where one has several tokens for a tile; the
  // bound on their number is too many then (4369 tokens of 11 adapters: 74
  // against 80, and the difference between two CTAs per tile and one: 53 us and 87).
  const int64_t tiles = t >= tile * (g + 1) ? t / tile + (g + 1) / 2 : max_tiles(t, g, tile);
  const int64_t room = (tile * rank > 1024 ? 1 : 2) * device_sm_count(current_device());
  int c = 1;
  while (c < kCluster && (tiles * 2 * c <= room || k >= int64_t(32) * 8 * 64 * c) &&
         int64_t(2) * c * 8 * 64 <= std::max(k, n) + 511)
    c *= 2;
  return c;
}

// CTAs that share out an adapter's tokens.  Requests differ in length, so up to
// twice what the GPU holds at once: the CTAs of short adapters make room early.
// Both gradients of 8192 packed tokens of 4 adapters, 8192 features: rank 32
// (one CTA per SM) 127, 95, 99 and 143 us with 1, 2, 4 and 8; rank 16 (two) 94,
// 79, 63 and 67.  No more than leave the average adapter's CTAs a chunk of 64
// tokens each, and two to spare (777 tokens of 5 adapters: 14.5, 10.0, 8.2 and
// 9.1 us).
int pick_wgrad_cluster(int64_t ntokens, int64_t nadapters, int64_t k, int64_t rank) {
  const int64_t cols = rank <= 32 ? 512 : (rank <= 64 ? 256 : 128);  // features of a CTA
  const int64_t room = (rank <= 16 ? 2 : 1) * device_sm_count(current_device());
  const int64_t ctas = ceil_div64(k, cols) * nadapters;
  int c = 1;
  while (c < kCluster && ctas * 2 * c <= 2 * room && 2 * c * kChunkTokens <= ntokens / nadapters + 2 * kChunkTokens)
    c *= 2;
  return c;
}

}  // namespace
}  // namespace kairo

using namespace kairo;

extern "C" kairo_status kairo_adapter_plan_size(int64_t ntokens, int64_t nadapters, size_t* plan, size_t* workspace) {
  if (!plan || !workspace) return fail(KAIRO_STATUS_INVALID_VALUE, "null argument");
  const kairo_status st = check_low_rank(ntokens, 1, 1, 1, nadapters, KAIRO_DTYPE_F16);
  if (st) return st;
  size_t sort = 0;
  const kairo_status ss = kairo_token_sort_workspace_size(ntokens, nadapters, &sort);
  if (ss) return ss;
  *plan = carve_plan(nullptr, ntokens, nadapters, nullptr);
  *workspace = align_up(static_cast<size_t>(ntokens) * sizeof(int32_t), 256) + sort;
  return KAIRO_STATUS_SUCCESS;
}

extern "C" kairo_status kairo_adapter_plan_build(const void* ids, int32_t id_bytes, int64_t ntokens, int64_t nadapters,
                                                 void* plan, size_t plan_size, void* workspace, size_t workspace_bytes,
                                                 void* stream) {
  size_t need = 0, ws_need = 0;
  kairo_status st = kairo_adapter_plan_size(ntokens, nadapters, &need, &ws_need);
  if (st) return st;
  if (id_bytes != 4 && id_bytes != 8) return fail(KAIRO_STATUS_INVALID_VALUE, "ids must be int32 or int64");
  if (!plan || !workspace || (ntokens > 0 && !ids)) return fail(KAIRO_STATUS_INVALID_VALUE, "null pointer argument");
  if (!aligned16(plan) || !aligned16(workspace))
    return fail(KAIRO_STATUS_INVALID_VALUE, "plan and workspace must be 16-byte aligned");
  if (plan_size < need) return fail(KAIRO_STATUS_INVALID_VALUE, "plan memory too small");
  if (workspace_bytes < ws_need) return fail(KAIRO_STATUS_WORKSPACE_TOO_SMALL, "adapter plan workspace too small");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  Plan pl;
  carve_plan(plan, ntokens, nadapters, &pl);
  int32_t* sorted = static_cast<int32_t*>(workspace);
  const size_t col = align_up(static_cast<size_t>(ntokens) * sizeof(int32_t), 256);
  st = kairo_token_sort(ids, id_bytes, ntokens, nadapters, sorted, pl.order, static_cast<uint8_t*>(workspace) + col,
                        workspace_bytes - col, stream);
  if (st) return st;
  k_plan_tiles<<<kTileSizes, 1024, 0, s>>>(reinterpret_cast<const uint32_t*>(sorted), ntokens, nadapters, pl);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "launch of the adapter plan");
  return KAIRO_STATUS_SUCCESS;
}

extern "C" kairo_status kairo_low_rank_apply(const void* x, int64_t ldx, int64_t k, const void* down, const void* up,
                                             int64_t n, int64_t rank, kairo_dtype dtype, const float* scale,
                                             const void* plan, int64_t ntokens, int64_t nadapters, const void* base,
                                             int64_t ldb, kairo_dtype base_dtype, void* y, int64_t ldy,
                                             kairo_dtype y_dtype, float* low, void* stream) {
  const kairo_status st = check_low_rank(ntokens, k, n, rank, nadapters, dtype);
  if (st) return st;
  if ((base && base_dtype != KAIRO_DTYPE_F32 && base_dtype != dtype) ||
      (y && y_dtype != KAIRO_DTYPE_F32 && y_dtype != dtype))
    return fail(KAIRO_STATUS_INVALID_VALUE, "base and y must be fp32 or the adapters' dtype");
  if (ldx < k || (y && ldy < n) || (base && ldb < n))
    return fail(KAIRO_STATUS_INVALID_VALUE, "leading dimension too small");
  if (ntokens == 0) return KAIRO_STATUS_SUCCESS;
  if (!x || !plan || (!y && !low) || (nadapters > 0 && (!down || (y && !up))))
    return fail(KAIRO_STATUS_INVALID_VALUE, "null pointer argument");
  Plan pl;
  carve_plan(const_cast<void*>(plan), ntokens, nadapters, &pl);
  const int64_t e = 2;
  const int64_t eb = base_dtype == KAIRO_DTYPE_F32 ? 4 : 2, ey = y_dtype == KAIRO_DTYPE_F32 ? 4 : 2;
  const bool vec = k % 8 == 0 && n % 8 == 0 && ldx * e % 16 == 0 && aligned16(x) && aligned16(down) && aligned16(up) &&
                   (!base || (ldb * eb % 16 == 0 && aligned16(base))) && (!y || (ldy * ey % 16 == 0 && aligned16(y)));
  const int tile = pick_tile(ntokens, k, rank, vec, base && base_dtype == KAIRO_DTYPE_F32);
  const int which = tile == 16 ? 0 : (tile == 32 ? 1 : 2);
  LowRankApplyArgs a{};
  a.x = x;
  a.down = down;
  a.up = up;
  a.base = base;
  a.y = y;
  a.low = low;
  a.scale = scale;
  a.order = pl.order;
  a.tiles = pl.tiles[which];
  a.ntiles = pl.ntiles + which;
  a.ldx = ldx;
  a.ldb = ldb;
  a.ldy = ldy;
  a.k = static_cast<int32_t>(k);
  a.n = static_cast<int32_t>(n);
  a.rank = static_cast<int32_t>(rank);
  a.base_f32 = base && base_dtype == KAIRO_DTYPE_F32;
  const int64_t clusters = max_tiles(ntokens, nadapters, tile);
  const int cluster = pick_cluster(ntokens, nadapters, tile, k, n, rank);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool yf = y && y_dtype == KAIRO_DTYPE_F32;
  const cudaError_t err = dtype == KAIRO_DTYPE_F16
                              ? launch_low_rank_apply<__half>(a, yf, vec, tile, clusters, cluster, s)
                              : launch_low_rank_apply<__nv_bfloat16>(a, yf, vec, tile, clusters, cluster, s);
  if (err != cudaSuccess) return cuda_fail(err, "launch of the low-rank product");
  return KAIRO_STATUS_SUCCESS;
}

namespace {

// One contraction over tokens: z in its own type, or codes and steps.
struct Grad {
  const float* low;
  const void* z;
  int64_t ldz;
  const int8_t* codes;
  int64_t ldq;
  const float* steps;
  int64_t lds;
  int64_t k;
  void* grad;
};

kairo_status check_grad(const Grad& p, int64_t rank, kairo_dtype dtype, const void* plan, int64_t ntokens,
                        int64_t nadapters, kairo_dtype grad_dtype) {
  const kairo_status st = check_low_rank(ntokens, p.k, 1, rank, nadapters, dtype);
  if (st) return st;
  if (grad_dtype != KAIRO_DTYPE_F32 && grad_dtype != dtype)
    return fail(KAIRO_STATUS_INVALID_VALUE, "the gradient must be fp32 or the adapters' dtype");
  if (nadapters == 0) return KAIRO_STATUS_SUCCESS;
  if (!plan || !p.grad || (ntokens > 0 && !p.low)) return fail(KAIRO_STATUS_INVALID_VALUE, "null pointer argument");
  return KAIRO_STATUS_SUCCESS;
}

// 16-byte accesses to z and the gradient; an 8-bit z always has them, and its gradient is stored value by value.
bool grad_aligned(const Grad& p) {
  return p.codes || (p.k % 8 == 0 && p.ldz % 8 == 0 && aligned16(p.z) && aligned16(p.grad));
}

// One or two of them in one launch (two: neither in 8 bits).
kairo_status run_grads(const Grad* p, int count, int64_t rank, kairo_dtype dtype, const void* plan, int64_t ntokens,
                       int64_t nadapters, kairo_dtype grad_dtype, void* stream) {
  if (nadapters == 0) return KAIRO_STATUS_SUCCESS;
  Plan pl;
  carve_plan(const_cast<void*>(plan), ntokens, nadapters, &pl);
  LowRankWgradArgs a{};
  bool vec = true;
  int64_t widest = 0, total = 0;
  for (int i = 0; i < count; ++i) {
    LowRankWgradArgs::One& o = a.one[i];
    o.s = p[i].low;
    o.z = p[i].z;
    o.codes = p[i].codes;
    o.steps = p[i].steps;
    o.grad = p[i].grad;
    o.ldz = p[i].ldz;
    o.ldq = p[i].ldq;
    o.lds = p[i].lds;
    o.k = static_cast<int32_t>(p[i].k);
    vec = vec && grad_aligned(p[i]);
    widest = std::max(widest, p[i].k);
    total += p[i].k;
  }
  a.order = pl.order;
  a.starts = pl.starts;
  a.tokens = ntokens;
  a.rank = static_cast<int32_t>(rank);
  a.count = count;
  a.widest = static_cast<int32_t>(widest);
  const int cluster = pick_wgrad_cluster(ntokens, nadapters, total, rank);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool gf = grad_dtype == KAIRO_DTYPE_F32;
  const cudaError_t err = dtype == KAIRO_DTYPE_F16
                              ? launch_low_rank_wgrad<__half>(a, gf, vec, nadapters, cluster, s)
                              : launch_low_rank_wgrad<__nv_bfloat16>(a, gf, vec, nadapters, cluster, s);
  if (err != cudaSuccess) return cuda_fail(err, "launch of the adapter gradient");
  return KAIRO_STATUS_SUCCESS;
}

}  // namespace

extern "C" kairo_status kairo_low_rank_wgrad(const float* low, int64_t rank, const void* z, int64_t ldz, int64_t k,
                                             kairo_dtype dtype, const void* plan, int64_t ntokens, int64_t nadapters,
                                             void* grad, kairo_dtype grad_dtype, void* stream) {
  if (ldz < k) return fail(KAIRO_STATUS_INVALID_VALUE, "leading dimension too small");
  if (ntokens > 0 && nadapters > 0 && !z) return fail(KAIRO_STATUS_INVALID_VALUE, "null pointer argument");
  const Grad p{low, z, ldz, nullptr, 0, nullptr, 0, k, grad};
  const kairo_status st = check_grad(p, rank, dtype, plan, ntokens, nadapters, grad_dtype);
  return st ? st : run_grads(&p, 1, rank, dtype, plan, ntokens, nadapters, grad_dtype, stream);
}

extern "C" kairo_status kairo_low_rank_wgrad_q8(const float* low, int64_t rank, const int8_t* codes, int64_t ldq,
                                                const float* steps, int64_t lds, int64_t k, kairo_dtype dtype,
                                                const void* plan, int64_t ntokens, int64_t nadapters, void* grad,
                                                kairo_dtype grad_dtype, void* stream) {
  kairo_status st = q8_check(ntokens, k, codes, ldq, steps, lds);
  if (st) return st;
  const Grad p{low, nullptr, 0, codes, ldq, steps, lds, k, grad};
  st = check_grad(p, rank, dtype, plan, ntokens, nadapters, grad_dtype);
  return st ? st : run_grads(&p, 1, rank, dtype, plan, ntokens, nadapters, grad_dtype, stream);
}

extern "C" kairo_status kairo_low_rank_wgrads(const float* dlow, const float* low, int64_t rank, const void* x,
                                              int64_t ldx, int64_t k, const void* dy, int64_t lddy, int64_t n,
                                              kairo_dtype dtype, const void* plan, int64_t ntokens, int64_t nadapters,
                                              void* d_down, void* d_up, kairo_dtype grad_dtype, void* stream) {
  if (ldx < k || lddy < n) return fail(KAIRO_STATUS_INVALID_VALUE, "leading dimension too small");
  if (ntokens > 0 && nadapters > 0 && (!x || !dy)) return fail(KAIRO_STATUS_INVALID_VALUE, "null pointer argument");
  const Grad p[2] = {{dlow, x, ldx, nullptr, 0, nullptr, 0, k, d_down},
                     {low, dy, lddy, nullptr, 0, nullptr, 0, n, d_up}};
  for (const Grad& q : p) {
    const kairo_status st = check_grad(q, rank, dtype, plan, ntokens, nadapters, grad_dtype);
    if (st) return st;
  }
  return run_grads(p, 2, rank, dtype, plan, ntokens, nadapters, grad_dtype, stream);
}
