// Embedding lookup with scaling, and the table's gradient by sorted tokens.
//
// lookup  out[t, :] = scale * weight[id_t, :], one rounding; a zero row for
//         an id outside [0, n_rows).
// sort    the token positions ordered by id, equal ids in token order (an
//         LSD radix sort of 8 bits a pass: counts per tile, one scan, a stable
//         scatter).  Ids outside [0, n_rows) become n_rows and end up last.
// grad    grad_weight[r, :] = scale * sum of grad_output[t, :] over id_t == r.
//         The sorted positions are cut into chunks of equal length whatever
//         the ids, so that a frequent token costs no more time than rare ones.
//         A thread owns a few columns of one chunk and walks its positions
//         in order.  A row whose tokens all lie in the chunk is written at once;
//         the head and the tail of a run that crosses chunks go to fp32
//         partial rows, which a second kernel adds up in chunk order.  All
//         sums are fp32 in an order that depends on the ids alone, so that
//         equal calls give equal bits.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "convert.cuh"
#include "internal.h"

namespace kairo {
namespace {

// ------------------------------------------------------------------ lookup

constexpr int kLookupThreads = 256;

// `tpr` threads (a power of two) share a row; VE elements per access.
template <typename TI, typename TO, typename ID, int VE>
__global__ void __launch_bounds__(kLookupThreads) k_lookup(const TI* __restrict__ weight, int64_t n_rows, int64_t dim,
                                                           int64_t ldw, const ID* __restrict__ ids, int64_t nids,
                                                           float scale, TO* __restrict__ out, int tpr_log2) {
  const int64_t rows_per_cta = kLookupThreads >> tpr_log2;
  const int lane = threadIdx.x & ((1 << tpr_log2) - 1);
  const int64_t step = static_cast<int64_t>(VE) << tpr_log2;
  for (int64_t t = blockIdx.x * rows_per_cta + (threadIdx.x >> tpr_log2); t < nids;
       t += static_cast<int64_t>(gridDim.x) * rows_per_cta) {
    const int64_t id = static_cast<int64_t>(ids[t]);
    const bool ok = id >= 0 && id < n_rows;
    const TI* src = weight + (ok ? id : 0) * ldw;
    TO* dst = out + t * dim;
    for (int64_t d = static_cast<int64_t>(lane) * VE; d < dim; d += step) {
      float f[VE];
      if (ok) {
        load_f32<TI, VE>(src + d, f);
#pragma unroll
        for (int i = 0; i < VE; ++i) f[i] *= scale;
      } else {
#pragma unroll
        for (int i = 0; i < VE; ++i) f[i] = 0.f;
      }
      store_f32<TO, VE>(dst + d, f);
    }
  }
}

// ------------------------------------------------------------------ sort

constexpr int kSortThreads = 256;
constexpr int kSortItems = 8;  // keys per thread
constexpr int kSortTile = kSortThreads * kSortItems;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kBins = 256;

template <typename ID>
__device__ __forceinline__ uint32_t token_key(const ID* ids, int64_t i, int64_t n_rows) {
  const int64_t id = static_cast<int64_t>(ids[i]);
  return static_cast<uint32_t>((id >= 0 && id < n_rows) ? id : n_rows);
}

// Keys of the first pass come from the ids, later ones from the last pass.
template <typename ID>
__device__ __forceinline__ uint32_t sort_key(const ID* ids, const uint32_t* keys, int64_t i, int64_t n_rows) {
  return keys ? keys[i] : token_key(ids, i, n_rows);
}

template <typename ID>
__global__ void __launch_bounds__(kSortThreads) k_sort_count(const ID* __restrict__ ids,
                                                             const uint32_t* __restrict__ keys, int64_t n,
                                                             int64_t n_rows, int shift, int ntiles,
                                                             uint32_t* __restrict__ counts) {
  __shared__ uint32_t bins[kBins];
  for (int b = threadIdx.x; b < kBins; b += kSortThreads) bins[b] = 0;
  __syncthreads();
  const int64_t base = static_cast<int64_t>(blockIdx.x) * kSortTile;
  for (int j = 0; j < kSortItems; ++j) {
    const int64_t i = base + j * kSortThreads + threadIdx.x;
    if (i < n) atomicAdd(&bins[(sort_key(ids, keys, i, n_rows) >> shift) & (kBins - 1)], 1u);
  }
  __syncthreads();
  for (int b = threadIdx.x; b < kBins; b += kSortThreads)
    counts[static_cast<int64_t>(b) * ntiles + blockIdx.x] = bins[b];
}

// Exclusive scan of n counts in place, one CTA.
__global__ void __launch_bounds__(1024) k_sort_scan(uint32_t* __restrict__ counts, int64_t n) {
  __shared__ uint32_t sums[32];
  __shared__ uint32_t carry;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) carry = 0;
  __syncthreads();
  for (int64_t base = 0; base < n; base += 1024) {
    const int64_t i = base + threadIdx.x;
    const uint32_t v = i < n ? counts[i] : 0u;
    uint32_t x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) sums[warp] = x;
    __syncthreads();
    if (warp == 0) {
      uint32_t s = sums[lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += y;
      }
      sums[lane] = s;
    }
    __syncthreads();
    const uint32_t incl = carry + x + (warp ? sums[warp - 1] : 0u);
    if (i < n) counts[i] = incl - v;
    __syncthreads();
    if (threadIdx.x == 1023) carry = incl;
    __syncthreads();
  }
}

// Stable scatter of one digit.  A warp owns 32 * kSortItems consecutive keys
// and takes them 32 at a time in order; lanes with equal digits rank
// themselves by a match of the warp.
template <typename ID>
__global__ void __launch_bounds__(kSortThreads) k_sort_scatter(
    const ID* __restrict__ ids, const uint32_t* __restrict__ keys, const int32_t* __restrict__ vals, int64_t n,
    int64_t n_rows, int shift, int ntiles, const uint32_t* __restrict__ offsets, uint32_t* __restrict__ keys_out,
    int32_t* __restrict__ vals_out) {
  __shared__ uint32_t where[kSortWarps][kBins];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int b = threadIdx.x; b < kSortWarps * kBins; b += kSortThreads) (&where[0][0])[b] = 0;
  __syncthreads();
  const int64_t base = static_cast<int64_t>(blockIdx.x) * kSortTile + warp * (32 * kSortItems) + lane;
  uint32_t key[kSortItems], rank[kSortItems];
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) {
    const int64_t i = base + j * 32;
    const bool ok = i < n;
    key[j] = ok ? sort_key(ids, keys, i, n_rows) : 0u;
    // keys past the end share a digit of their own that is never counted
    const uint32_t d = ok ? (key[j] >> shift) & (kBins - 1) : kBins;
    const uint32_t same = __match_any_sync(0xffffffffu, d);
    const int leader = __ffs(same) - 1;
    uint32_t first = 0;
    if (lane == leader && ok) {
      first = where[warp][d];
      where[warp][d] = first + __popc(same);
    }
    first = __shfl_sync(0xffffffffu, first, leader);
    rank[j] = first + __popc(same & ((1u << lane) - 1u));
    __syncwarp();
  }
  __syncthreads();
  for (int b = threadIdx.x; b < kBins; b += kSortThreads) {
    uint32_t at = offsets[static_cast<int64_t>(b) * ntiles + blockIdx.x];
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) {
      const uint32_t c = where[w][b];
      where[w][b] = at;
      at += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) {
    const int64_t i = base + j * 32;
    if (i < n) {
      const uint32_t to = where[warp][(key[j] >> shift) & (kBins - 1)] + rank[j];
      keys_out[to] = key[j];
      vals_out[to] = vals ? vals[i] : static_cast<int32_t>(i);
    }
  }
}

int sort_passes(int64_t n_rows) {
  int bits = 1;
  while (bits < 31 && (int64_t(1) << bits) <= n_rows) ++bits;
  return (bits + 7) / 8;
}

int64_t sort_tiles(int64_t n) { return std::max<int64_t>(1, ceil_div64(n, kSortTile)); }

// Workspace: one spare copy of keys and positions, then the counts.
size_t sort_ws_bytes(int64_t n) {
  return 2 * align_up(static_cast<size_t>(n) * 4, 256) + align_up(static_cast<size_t>(sort_tiles(n)) * kBins * 4, 256);
}

template <typename ID>
kairo_status sort_launch(const ID* ids, int64_t n, int64_t n_rows, uint32_t* sorted, int32_t* perm, void* ws,
                         cudaStream_t s) {
  const size_t col = align_up(static_cast<size_t>(n) * 4, 256);
  uint32_t* keys_b = static_cast<uint32_t*>(ws);
  int32_t* vals_b = reinterpret_cast<int32_t*>(static_cast<uint8_t*>(ws) + col);
  uint32_t* counts = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(ws) + 2 * col);
  const int tiles = static_cast<int>(sort_tiles(n));
  const int passes = sort_passes(n_rows);
  const uint32_t* keys = nullptr;
  const int32_t* vals = nullptr;
  for (int p = 0; p < passes; ++p) {
    // the last pass writes the caller's arrays
    const bool own = ((passes - 1 - p) & 1) == 0;
    uint32_t* keys_out = own ? sorted : keys_b;
    int32_t* vals_out = own ? perm : vals_b;
    k_sort_count<ID><<<tiles, kSortThreads, 0, s>>>(ids, keys, n, n_rows, 8 * p, tiles, counts);
    k_sort_scan<<<1, 1024, 0, s>>>(counts, static_cast<int64_t>(tiles) * kBins);
    k_sort_scatter<ID><<<tiles, kSortThreads, 0, s>>>(ids, keys, vals, n, n_rows, 8 * p, tiles, counts, keys_out,
                                                      vals_out);
    keys = keys_out;
    vals = vals_out;
  }
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "launch of the token sort");
  return KAIRO_STATUS_SUCCESS;
}

// ------------------------------------------------------------------ gradient

constexpr int kGradThreads = 128;
constexpr int kGradChunk = 32;  // sorted positions per chunk

template <typename TO, int VE>
__device__ __forceinline__ void emit_row(TO* dst, float (&acc)[VE], float scale, bool accumulate) {
  float f[VE];
  if (accumulate) load_f32<TO, VE>(dst, f);
#pragma unroll
  for (int i = 0; i < VE; ++i) f[i] = accumulate ? f[i] + acc[i] * scale : acc[i] * scale;
  store_f32<TO, VE>(dst, f);
}

template <int VE>
__device__ __forceinline__ void store_partial(float* dst, const float (&acc)[VE]) {
#pragma unroll
  for (int i = 0; i < VE; ++i) dst[i] = acc[i];
}

// Partial rows: 2 * chunk is the part of a run that began before the chunk,
// 2 * chunk + 1 the part of a run that begins in it and goes on behind it.
template <typename TI, typename TO, int VE>
__global__ void __launch_bounds__(kGradThreads) k_grad_chunks(
    const TI* __restrict__ grad, int64_t ldg, const uint32_t* __restrict__ sorted, const int32_t* __restrict__ perm,
    int64_t n, int64_t n_rows, int64_t dim, float scale, TO* __restrict__ out, int64_t ldo, bool accumulate,
    float* __restrict__ partial) {
  const int64_t col = (static_cast<int64_t>(blockIdx.y) * kGradThreads + threadIdx.x) * VE;
  if (col >= dim) return;
  const int64_t chunk = blockIdx.x;
  const int64_t p0 = chunk * kGradChunk, p1 = min(n, p0 + kGradChunk);
  bool open_left = p0 > 0 && sorted[p0 - 1] == sorted[p0];
  float acc[VE];
#pragma unroll
  for (int i = 0; i < VE; ++i) acc[i] = 0.f;
  for (int64_t p = p0; p < p1; ++p) {
    const uint32_t key = sorted[p];
    if (key >= n_rows) break;  // ids out of range come last
    const int32_t t = perm[p];
    if (t < 0 || t >= n) break;  // not a permutation: read nothing
    float f[VE];
    load_f32<TI, VE>(grad + static_cast<int64_t>(t) * ldg + col, f);
#pragma unroll
    for (int i = 0; i < VE; ++i) acc[i] += f[i];
    const bool last = p + 1 == n || sorted[p + 1] != key;
    if (last || p + 1 == p1) {
      if (open_left) store_partial<VE>(partial + (2 * chunk) * dim + col, acc);
      else if (!last) store_partial<VE>(partial + (2 * chunk + 1) * dim + col, acc);
      else emit_row<TO, VE>(out + static_cast<int64_t>(key) * ldo + col, acc, scale, accumulate);
      open_left = false;
#pragma unroll
      for (int i = 0; i < VE; ++i) acc[i] = 0.f;
    }
  }
}

// The chunk in which a run begins that goes on behind it adds up the run's
// parts in order.
template <typename TO, int VE>
__global__ void __launch_bounds__(kGradThreads) k_grad_join(const uint32_t* __restrict__ sorted, int64_t n,
                                                            int64_t n_rows, int64_t dim, float scale,
                                                            TO* __restrict__ out, int64_t ldo, bool accumulate,
                                                            const float* __restrict__ partial) {
  const int64_t col = (static_cast<int64_t>(blockIdx.y) * kGradThreads + threadIdx.x) * VE;
  if (col >= dim) return;
  const int64_t chunk = blockIdx.x;
  const int64_t p0 = chunk * kGradChunk, p1 = p0 + kGradChunk;
  if (p1 >= n) return;
  const uint32_t key = sorted[p1 - 1];
  if (key >= n_rows || sorted[p1] != key) return;
  if (p0 > 0 && sorted[p0] == key && sorted[p0 - 1] == key) return;  // began earlier
  float acc[VE];
#pragma unroll
  for (int i = 0; i < VE; ++i) acc[i] = partial[(2 * chunk + 1) * dim + col + i];
  for (int64_t c = chunk + 1; c * kGradChunk < n && sorted[c * kGradChunk] == key; ++c) {
#pragma unroll
    for (int i = 0; i < VE; ++i) acc[i] += partial[(2 * c) * dim + col + i];
  }
  emit_row<TO, VE>(out + static_cast<int64_t>(key) * ldo + col, acc, scale, accumulate);
}

size_t grad_ws_bytes(int64_t n, int64_t dim) {
  return static_cast<size_t>(2 * ceil_div64(std::max<int64_t>(n, 1), kGradChunk)) * dim * sizeof(float);
}

template <typename TI, typename TO, int VE>
void grad_launch(const void* grad, int64_t ldg, const int32_t* sorted, const int32_t* perm, int64_t n, int64_t n_rows,
                 int64_t dim, float scale, void* out, int64_t ldo, bool accumulate, float* partial, cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>(ceil_div64(n, kGradChunk)),
                  static_cast<unsigned>(ceil_div64(dim, static_cast<int64_t>(kGradThreads) * VE)));
  const uint32_t* keys = reinterpret_cast<const uint32_t*>(sorted);
  k_grad_chunks<TI, TO, VE><<<grid, kGradThreads, 0, s>>>(static_cast<const TI*>(grad), ldg, keys, perm, n, n_rows,
                                                         dim, scale, static_cast<TO*>(out), ldo, accumulate, partial);
  if (grid.x > 1)
    k_grad_join<TO, VE><<<grid, kGradThreads, 0, s>>>(keys, n, n_rows, dim, scale, static_cast<TO*>(out), ldo,
                                                      accumulate, partial);
}

template <typename TI, typename TO>
void grad_pick(int ve, const void* grad, int64_t ldg, const int32_t* sorted, const int32_t* perm, int64_t n,
               int64_t n_rows, int64_t dim, float scale, void* out, int64_t ldo, bool accumulate, float* partial,
               cudaStream_t s) {
  if (ve == 4)
    grad_launch<TI, TO, 4>(grad, ldg, sorted, perm, n, n_rows, dim, scale, out, ldo, accumulate, partial, s);
  else
    grad_launch<TI, TO, 1>(grad, ldg, sorted, perm, n, n_rows, dim, scale, out, ldo, accumulate, partial, s);
}

bool aligned(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % static_cast<uintptr_t>(bytes) == 0; }

template <typename TI, typename TO, typename ID>
void lookup_pick(const void* weight, int64_t n_rows, int64_t dim, int64_t ldw, const void* ids, int64_t nids,
                 float scale, void* out, cudaStream_t s) {
  const TI* w = static_cast<const TI*>(weight);
  TO* o = static_cast<TO*>(out);
  const ID* id = static_cast<const ID*>(ids);
  const bool vec = dim % 4 == 0 && ldw % 4 == 0 && aligned(weight, 4 * sizeof(TI)) && aligned(out, 4 * sizeof(TO));
  const int64_t per_row = vec ? dim / 4 : dim;
  int l2 = 0;
  while (l2 < 8 && (int64_t(1) << l2) < per_row) ++l2;
  const int64_t rows = kLookupThreads >> l2;
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(ceil_div64(nids, rows), 148 * 64));
  if (vec) k_lookup<TI, TO, ID, 4><<<grid, kLookupThreads, 0, s>>>(w, n_rows, dim, ldw, id, nids, scale, o, l2);
  else k_lookup<TI, TO, ID, 1><<<grid, kLookupThreads, 0, s>>>(w, n_rows, dim, ldw, id, nids, scale, o, l2);
}

template <typename TI, typename TO>
void lookup_ids(const void* weight, int64_t n_rows, int64_t dim, int64_t ldw, const void* ids, bool ids64,
                int64_t nids, float scale, void* out, cudaStream_t s) {
  if (ids64) lookup_pick<TI, TO, int64_t>(weight, n_rows, dim, ldw, ids, nids, scale, out, s);
  else lookup_pick<TI, TO, int32_t>(weight, n_rows, dim, ldw, ids, nids, scale, out, s);
}

constexpr int64_t kMaxTokens = 0x7fffffffLL - 4096;
constexpr int64_t kMaxRows = 0x7ffffffeLL;

// Calls fn with one value of each C++ element type of (in, out).
template <typename F>
void for_types(kairo_dtype in, kairo_dtype out, F&& fn) {
  auto with = [&](auto ti) {
    if (out == KAIRO_DTYPE_F32) fn(ti, float{});
    else if (out == KAIRO_DTYPE_F16) fn(ti, __half{});
    else fn(ti, __nv_bfloat16{});
  };
  if (in == KAIRO_DTYPE_F32) with(float{});
  else if (in == KAIRO_DTYPE_F16) with(__half{});
  else with(__nv_bfloat16{});
}

}  // namespace
}  // namespace kairo

using namespace kairo;

extern "C" kairo_status kairo_embedding_lookup(const void* weight, int64_t n_rows, int64_t dim, int64_t ldw,
                                               kairo_dtype dtype, const void* ids, int32_t id_bytes, int64_t nids,
                                               float scale, void* out, kairo_dtype out_dtype, void* stream) {
  if (n_rows < 0 || dim <= 0 || nids < 0) return fail(KAIRO_STATUS_INVALID_VALUE, "invalid size");
  if (ldw < dim) return fail(KAIRO_STATUS_INVALID_VALUE, "leading dimension smaller than dim");
  if (!known_dtype(dtype) || !known_dtype(out_dtype)) return fail(KAIRO_STATUS_INVALID_VALUE, "unknown dtype");
  if (id_bytes != 4 && id_bytes != 8) return fail(KAIRO_STATUS_INVALID_VALUE, "ids must be int32 or int64");
  if (nids == 0) return KAIRO_STATUS_SUCCESS;
  if ((!weight && n_rows > 0) || !ids || !out) return fail(KAIRO_STATUS_INVALID_VALUE, "null pointer argument");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  for_types(dtype, out_dtype, [&](auto ti, auto to) {
    lookup_ids<decltype(ti), decltype(to)>(weight, n_rows, dim, ldw, ids, id_bytes == 8, nids, scale, out, s);
  });
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "launch of the embedding lookup");
  return KAIRO_STATUS_SUCCESS;
}

extern "C" kairo_status kairo_token_sort_workspace_size(int64_t nids, int64_t n_rows, size_t* bytes) {
  if (!bytes || nids < 0 || n_rows < 0) return fail(KAIRO_STATUS_INVALID_VALUE, "invalid argument");
  if (nids > kMaxTokens || n_rows > kMaxRows) return fail(KAIRO_STATUS_NOT_SUPPORTED, "too many tokens or rows");
  *bytes = sort_ws_bytes(nids);
  return KAIRO_STATUS_SUCCESS;
}

extern "C" kairo_status kairo_token_sort(const void* ids, int32_t id_bytes, int64_t nids, int64_t n_rows,
                                         int32_t* sorted, int32_t* perm, void* workspace, size_t workspace_bytes,
                                         void* stream) {
  size_t need = 0;
  const kairo_status st = kairo_token_sort_workspace_size(nids, n_rows, &need);
  if (st) return st;
  if (id_bytes != 4 && id_bytes != 8) return fail(KAIRO_STATUS_INVALID_VALUE, "ids must be int32 or int64");
  if (nids == 0) return KAIRO_STATUS_SUCCESS;
  if (!ids || !sorted || !perm || !workspace) return fail(KAIRO_STATUS_INVALID_VALUE, "null pointer argument");
  if (workspace_bytes < need) return fail(KAIRO_STATUS_WORKSPACE_TOO_SMALL, "token sort workspace too small");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  uint32_t* keys = reinterpret_cast<uint32_t*>(sorted);
  return id_bytes == 8 ? sort_launch(static_cast<const int64_t*>(ids), nids, n_rows, keys, perm, workspace, s)
                       : sort_launch(static_cast<const int32_t*>(ids), nids, n_rows, keys, perm, workspace, s);
}

extern "C" kairo_status kairo_embedding_grad_workspace_size(int64_t nids, int64_t dim, size_t* bytes) {
  if (!bytes || nids < 0 || dim <= 0) return fail(KAIRO_STATUS_INVALID_VALUE, "invalid argument");
  *bytes = grad_ws_bytes(nids, dim);
  return KAIRO_STATUS_SUCCESS;
}

extern "C" kairo_status kairo_embedding_grad(const void* grad_output, int64_t ldg, kairo_dtype dtype,
                                             const int32_t* sorted, const int32_t* perm, int64_t nids, int64_t n_rows,
                                             int64_t dim, float scale, void* grad_weight, int64_t ldo,
                                             kairo_dtype out_dtype, int32_t accumulate, void* workspace,
                                             size_t workspace_bytes, void* stream) {
  if (n_rows < 0 || dim <= 0 || nids < 0) return fail(KAIRO_STATUS_INVALID_VALUE, "invalid size");
  if (nids > kMaxTokens || n_rows > kMaxRows) return fail(KAIRO_STATUS_NOT_SUPPORTED, "too many tokens or rows");
  if (dim > static_cast<int64_t>(65535) * kGradThreads) return fail(KAIRO_STATUS_NOT_SUPPORTED, "dim too large");
  if (ldg < dim || ldo < dim) return fail(KAIRO_STATUS_INVALID_VALUE, "leading dimension smaller than dim");
  if (!known_dtype(dtype) || !known_dtype(out_dtype)) return fail(KAIRO_STATUS_INVALID_VALUE, "unknown dtype");
  if (n_rows == 0) return KAIRO_STATUS_SUCCESS;
  if (!grad_weight) return fail(KAIRO_STATUS_INVALID_VALUE, "null grad_weight");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t ob = element_bytes(out_dtype);
  if (!accumulate) {
    const cudaError_t e = cudaMemset2DAsync(grad_weight, static_cast<size_t>(ldo * ob), 0,
                                            static_cast<size_t>(dim * ob), static_cast<size_t>(n_rows), s);
    if (e != cudaSuccess) return cuda_fail(e, "cudaMemset2DAsync(grad_weight)");
  }
  if (nids == 0) return KAIRO_STATUS_SUCCESS;
  if (!grad_output || !sorted || !perm || !workspace) return fail(KAIRO_STATUS_INVALID_VALUE, "null pointer argument");
  if (workspace_bytes < grad_ws_bytes(nids, dim))
    return fail(KAIRO_STATUS_WORKSPACE_TOO_SMALL, "embedding gradient workspace too small");
  const int64_t ib = element_bytes(dtype);
  const int ve = (dim % 4 == 0 && ldg % 4 == 0 && ldo % 4 == 0 && aligned(grad_output, 4 * ib) &&
                  aligned(grad_weight, 4 * ob)) ? 4 : 1;
  for_types(dtype, out_dtype, [&](auto ti, auto to) {
    grad_pick<decltype(ti), decltype(to)>(ve, grad_output, ldg, sorted, perm, nids, n_rows, dim, scale, grad_weight,
                                          ldo, accumulate != 0, static_cast<float*>(workspace), s);
  });
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "launch of the embedding gradient");
  return KAIRO_STATUS_SUCCESS;
}
