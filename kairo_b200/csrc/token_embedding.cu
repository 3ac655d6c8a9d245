// Embedding lookup with scaling, and the table's gradient by sorted tokens.
//
// lookup  out[t, :] = scale * weight[id_t, :], one rounding; a zero row for
//         an id outside [0, n_rows).
// sort    the token positions ordered by id, equal ids in token order (an
//         LSD radix sort).  Ids outside [0, n_rows) become n_rows and end up
//         last.  Lists of up to 4096 tokens (2048 where ids are below 512) are
//         ranked by counting; up to 65536 are sorted by one cluster, keys and
//         positions staying in its distributed shared memory between the
//         passes, both in one launch; longer lists take three launches a pass
//         (65536 tokens of 131072 rows 35 us, 65537 64, 10^6 332).
// grad    grad_weight[r, :] = scale * sum of grad_output[t, :] over id_t == r.
//         The sorted positions are cut into chunks of equal length whatever
//         the ids, so that a frequent token costs no more time than rare ones.
//         A thread owns a few columns of one chunk and walks its positions
//         in order.  A row whose tokens all lie in the chunk is written at once;
//         the head and the tail of a run that crosses chunks go to fp32
//         partial rows, which a second kernel adds up in chunk order.  All
//         sums are fp32 in an order that depends on the ids alone, so that
//         equal calls give equal bits.  Rows without tokens are zeroed by
//         further CTAs of the first kernel; the last rows of a large table are
//         zeroed beside the cluster's sort, and those of them that have tokens
//         written again.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "convert.cuh"
#include "internal.h"

namespace kairo {
namespace {

// ------------------------------------------------------------------ lookup

constexpr int kLookupThreads = 256;

// `tpr` threads (a power of two) share a row; VE elements per access, U rows of
// each thread under way.  Bound by memory: 32768 rows of 4096 bf16 82 us (6.5
// TB/s), 65536 of 128 fp32 to bf16 7.1 us (parts of it stay in L2).
template <typename TI, typename TO, typename ID, int VE, int U>
__global__ void __launch_bounds__(kLookupThreads) k_lookup(const TI* __restrict__ weight, int64_t n_rows, int64_t dim,
                                                           int64_t ldw, const ID* __restrict__ ids, int64_t nids,
                                                           float scale, TO* __restrict__ out, int tpr_log2) {
  const int64_t rows = kLookupThreads >> tpr_log2;  // of the CTA at a time
  const int lane = threadIdx.x & ((1 << tpr_log2) - 1);
  const int64_t first = (static_cast<int64_t>(blockIdx.y) << tpr_log2) + lane;  // slices of the columns
  const int64_t step = (static_cast<int64_t>(VE) << tpr_log2) * gridDim.y;
  for (int64_t t0 = blockIdx.x * rows * U + (threadIdx.x >> tpr_log2); t0 < nids;
       t0 += static_cast<int64_t>(gridDim.x) * rows * U) {
    int64_t id[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      id[u] = t0 + u * rows < nids ? static_cast<int64_t>(ids[t0 + u * rows]) : -1;
      if (id[u] >= n_rows) id[u] = -1;
    }
    for (int64_t d = first * VE; d < dim; d += step) {
      Raw<TI, VE> f[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (id[u] >= 0) f[u].load(weight + id[u] * ldw + d);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (t0 + u * rows >= nids) break;
        float v[VE];
#pragma unroll
        for (int i = 0; i < VE; ++i) v[i] = id[u] >= 0 ? f[u][i] * scale : 0.f;
        store_f32<TO, VE>(out + (t0 + u * rows) * dim + d, v);
      }
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

// Lanes that hold the same `bits`-bit digit as this one, among those with ok.  A
// vote per bit: with the warp's match instruction the cluster sort of 32768
// tokens of 131072 rows took 26.4 us instead of 22.6.
__device__ __forceinline__ uint32_t same_digit(uint32_t d, bool ok, int bits) {
  uint32_t same = __ballot_sync(0xffffffffu, ok);
  for (int b = 0; b < bits; ++b) {
    const bool one = (d >> b) & 1u;
    const uint32_t vote = __ballot_sync(0xffffffffu, one);
    same &= one ? vote : ~vote;
  }
  return same;
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
// themselves by a vote per bit.
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
    const uint32_t d = (key[j] >> shift) & (kBins - 1);
    const uint32_t same = same_digit(d, ok, 8);
    const int leader = ok ? __ffs(same) - 1 : lane;
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

int key_bits(int64_t n_rows) {  // of the keys 0 .. n_rows
  int bits = 1;
  while (bits < 31 && (int64_t(1) << bits) <= n_rows) ++bits;
  return bits;
}

int sort_passes(int64_t n_rows) { return (key_bits(n_rows) + 7) / 8; }

// The whole sort in one cluster.  CTA c holds positions c * per ..; in a pass
// every warp ranks its share of them in order, the digit counts of all CTAs
// are read over distributed shared memory, the CTA brings its keys into digit
// order, and each is stored straight into the shared memory of the CTA that
// holds its place (the last pass: into the result), equal digits side by side.
//
// Clusters behind the first zero rows of the gradient meanwhile, which the
// other SMs have time for.
constexpr int kClusterThreads = 1024;
constexpr int kClusterWarps = kClusterThreads / 32;
constexpr int kClusterItems = 8;   // positions per thread at most
constexpr int kClusterMax = 8;     // CTAs
constexpr int kMaxDigit = 9;       // bits of a pass
constexpr int kMaxBins = 1 << kMaxDigit;
constexpr int64_t kClusterTokens = int64_t(kClusterMax) * kClusterItems * kClusterThreads;

size_t cluster_sort_smem(int per) {
  return static_cast<size_t>(per) * 16 + static_cast<size_t>(kClusterWarps * kMaxBins + 3 * kMaxBins + 64) * 4;
}

// Rows to zero: `vecs` 16-byte vectors each, `pitch` of them apart.
struct ZeroRows {
  uint4* first;
  int64_t rows, vecs, pitch;
};

__device__ __forceinline__ uint32_t cta_of(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void all_ctas() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

// Exclusive scan of v over the CTA's threads.
__device__ __forceinline__ uint32_t scan_cta(uint32_t v, uint32_t* sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
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
  const uint32_t out = x - v + (warp ? sums[warp - 1] : 0u);
  __syncthreads();
  return out;
}

template <typename ID>
__global__ void __launch_bounds__(kClusterThreads) k_sort_cluster(const ID* __restrict__ ids, int n, int64_t n_rows,
                                                                  int per, int passes, int digit,
                                                                  uint32_t* __restrict__ sorted,
                                                                  int32_t* __restrict__ perm, const ZeroRows zero) {
  extern __shared__ __align__(16) uint32_t sm[];
  uint32_t* keys = sm;                              // [2][per]
  uint32_t* vals = keys + 2 * per;                  // [2][per]
  uint32_t* where = vals + 2 * per;                 // [kClusterWarps][bins]
  uint32_t* total = where + kClusterWarps * kMaxBins;  // [bins]: this CTA's count of every digit
  uint32_t* local = total + kMaxBins;               // [bins]: first of a digit in the CTA's own order
  uint32_t* base = local + kMaxBins;                // [bins]: place of that one in the whole order
  uint32_t* sums = base + kMaxBins;                 // [32]
  uint32_t crank, csize;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(crank));
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(csize));
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (blockIdx.x >= csize) {  // not the sorting cluster
    const int64_t warps = static_cast<int64_t>(gridDim.x - csize) * kClusterWarps;
    for (int64_t r = static_cast<int64_t>(blockIdx.x - csize) * kClusterWarps + warp; r < zero.rows; r += warps)
      for (int64_t v = lane; v < zero.vecs; v += 32) zero.first[r * zero.pitch + v] = make_uint4(0u, 0u, 0u, 0u);
    return;
  }
  const int bins = 1 << digit;
  const int first = static_cast<int>(crank) * per;
  const int have = max(0, min(per, n - first));     // positions of this CTA
  const int share = per / kClusterWarps;            // consecutive positions of a warp
  for (int i = threadIdx.x; i < have; i += kClusterThreads) {
    keys[i] = token_key(ids, first + i, n_rows);
    vals[i] = static_cast<uint32_t>(first + i);
  }
  for (int p = 0; p < passes; ++p) {
    const int shift = p * digit;
    uint32_t* from_k = keys + (p & 1) * per;
    uint32_t* from_v = vals + (p & 1) * per;
    for (int i = threadIdx.x; i < kClusterWarps * bins; i += kClusterThreads) where[i] = 0;
    __syncthreads();
    uint32_t key[kClusterItems], val[kClusterItems], rank[kClusterItems];
    uint32_t* mine = where + warp * bins;
#pragma unroll
    for (int j = 0; j < kClusterItems; ++j) {
      if (j * 32 < share) {
        const int i = warp * share + j * 32 + lane;
        const bool ok = i < have;
        key[j] = ok ? from_k[i] : 0u;
        val[j] = ok ? from_v[i] : 0u;
        const uint32_t d = (key[j] >> shift) & (bins - 1);
        const uint32_t same = same_digit(d, ok, digit);
        const int leader = ok ? __ffs(same) - 1 : lane;
        uint32_t at = 0;
        if (lane == leader && ok) {
          at = mine[d];
          mine[d] = at + __popc(same);
        }
        at = __shfl_sync(0xffffffffu, at, leader);
        rank[j] = at + __popc(same & ((1u << lane) - 1u));
        __syncwarp();
      }
    }
    __syncthreads();
    uint32_t here = 0;
    if (threadIdx.x < bins) {
#pragma unroll 8
      for (int w = 0; w < kClusterWarps; ++w) {
        const uint32_t c = where[w * bins + threadIdx.x];
        where[w * bins + threadIdx.x] = here;
        here += c;
      }
      total[threadIdx.x] = here;
    }
    const uint32_t before_here = scan_cta(here, sums);
    if (threadIdx.x < bins) local[threadIdx.x] = before_here;
    all_ctas();
    // Keys of smaller digits anywhere, and of this digit in CTAs before this one.
    uint32_t all = 0, before = 0;
    if (threadIdx.x < bins) {
      const uint32_t addr = static_cast<uint32_t>(__cvta_generic_to_shared(total + threadIdx.x));
      uint32_t c[kClusterMax];
#pragma unroll
      for (uint32_t r = 0; r < kClusterMax; ++r) {
        c[r] = 0;
        if (r < csize) asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(c[r]) : "r"(cta_of(addr, r)));
      }
#pragma unroll
      for (uint32_t r = 0; r < kClusterMax; ++r) {
        all += c[r];
        if (r < crank) before += c[r];
      }
    }
    const uint32_t smaller = scan_cta(all, sums);
    if (threadIdx.x < bins) base[threadIdx.x] = smaller + before;
    // This CTA's keys in the order of their digits.
#pragma unroll
    for (int j = 0; j < kClusterItems; ++j) {
      if (j * 32 < share && warp * share + j * 32 + lane < have) {
        const uint32_t d = (key[j] >> shift) & (bins - 1);
        const uint32_t at = local[d] + mine[d] + rank[j];
        from_k[at] = key[j];
        from_v[at] = val[j];
      }
    }
    __syncthreads();
    const bool last = p + 1 == passes;
    const uint32_t to_k = static_cast<uint32_t>(__cvta_generic_to_shared(keys + ((p + 1) & 1) * per));
    const uint32_t to_v = static_cast<uint32_t>(__cvta_generic_to_shared(vals + ((p + 1) & 1) * per));
    for (int i = threadIdx.x; i < have; i += kClusterThreads) {
      const uint32_t k = from_k[i], v = from_v[i];
      const uint32_t d = (k >> shift) & (bins - 1);
      const uint32_t at = base[d] + (static_cast<uint32_t>(i) - local[d]);
      if (last) {
        sorted[at] = k;
        perm[at] = static_cast<int32_t>(v);
      } else {
        const uint32_t cta = at / static_cast<uint32_t>(per), off = 4u * (at - cta * per);
        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cta_of(to_k + off, cta)), "r"(k) : "memory");
        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cta_of(to_v + off, cta)), "r"(v) : "memory");
      }
    }
    all_ctas();  // the next pass reads what the others stored here
  }
}

// A list of kRankTokens at most: the place of a token is the number of smaller
// ids and of equal ones before it.  A warp counts for one token, 32 tokens to
// a CTA; one pass, no exchange.  1024 tokens 3.1 us, 4096 6.7 and 8192 20; the
// cluster's sort takes 10.8 us for 4097 tokens and 11.3 for 8192.
constexpr int kRankTokens = 4096;
template <typename ID>
__global__ void __launch_bounds__(1024) k_sort_ranks(const ID* __restrict__ ids, int n, int64_t n_rows,
                                                     uint32_t* __restrict__ sorted, int32_t* __restrict__ perm) {
  __shared__ uint32_t keys[kRankTokens];
  for (int i = threadIdx.x; i < n; i += 1024) keys[i] = token_key(ids, i, n_rows);
  __syncthreads();
  const int lane = threadIdx.x & 31, t = blockIdx.x * 32 + (threadIdx.x >> 5);
  if (t >= n) return;
  const uint32_t mine = keys[t];
  int place = 0;
  for (int i = lane; i < n; i += 32) {
    const uint32_t k = keys[i];
    place += k < mine || (k == mine && i < t);
  }
  place = __reduce_add_sync(0xffffffffu, place);
  if (lane == 0) {
    sorted[place] = mine;
    perm[place] = t;
  }
}

template <typename ID>
kairo_status sort_in_cluster(const ID* ids, int64_t n, int64_t n_rows, uint32_t* sorted, int32_t* perm,
                             const ZeroRows& zero, cudaStream_t s) {
  int ctas = 1;
  while (ctas < kClusterMax && ctas * kClusterThreads < n) ctas *= 2;
  const int per = static_cast<int>(ceil_div64(ceil_div64(n, ctas), kClusterThreads)) * kClusterThreads;
  const int bits = key_bits(n_rows);
  const int passes = (bits + kMaxDigit - 1) / kMaxDigit;
  auto* fn = &k_sort_cluster<ID>;
  const size_t smem = cluster_sort_smem(per);
  cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       static_cast<int>(cluster_sort_smem(kClusterItems * kClusterThreads)));
  if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(token sort)");
  // As many zeroing clusters as leave room for the sort, and one at least: the
  // caller counts on these rows.
  const int spare = zero.rows > 0 ? std::max(1, device_sm_count(current_device()) / ctas - 2) : 0;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas * (1 + spare)));
  cfg.blockDim = dim3(kClusterThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = static_cast<unsigned>(ctas);
  at.val.clusterDim.y = 1;
  at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, fn, ids, static_cast<int>(n), n_rows, per, passes, (bits + passes - 1) / passes, sorted,
                         perm, zero);
  if (e != cudaSuccess) return cuda_fail(e, "launch of the token sort");
  return KAIRO_STATUS_SUCCESS;
}

int64_t sort_tiles(int64_t n) { return std::max<int64_t>(1, ceil_div64(n, kSortTile)); }

// Workspace: one spare copy of keys and positions, then the counts.
size_t sort_ws_bytes(int64_t n) {
  if (n <= kClusterTokens) return 256;  // nothing: the cluster's shared memory holds it all
  return 2 * align_up(static_cast<size_t>(n) * 4, 256) + align_up(static_cast<size_t>(sort_tiles(n)) * kBins * 4, 256);
}

template <typename ID>
kairo_status sort_launch(const ID* ids, int64_t n, int64_t n_rows, uint32_t* sorted, int32_t* perm, void* ws,
                         const ZeroRows& zero, cudaStream_t s) {
  // half as many where the cluster needs one pass only (ids below 512): 4096 tokens 5.9 us, counted 6.7
  if (n <= (key_bits(n_rows) <= kMaxDigit ? kRankTokens / 2 : kRankTokens)) {
    k_sort_ranks<ID><<<static_cast<unsigned>(ceil_div64(n, 32)), 1024, 0, s>>>(ids, static_cast<int>(n), n_rows, sorted,
                                                                              perm);
    const cudaError_t e = cudaGetLastError();
    return e != cudaSuccess ? cuda_fail(e, "launch of the token sort") : KAIRO_STATUS_SUCCESS;
  }
  if (n <= kClusterTokens) return sort_in_cluster(ids, n, n_rows, sorted, perm, zero, s);
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
constexpr int kGradChunk = 32;   // sorted positions per chunk
constexpr int kGradAhead = 8;    // rows under way per thread
constexpr int kFewRows = 32;     // rows of a CTA that takes a short list

template <typename TO, int VE>
__device__ __forceinline__ void emit_row(TO* dst, float (&acc)[VE], float scale, bool accumulate) {
  float f[VE];
  if (accumulate) load_f32<TO, VE>(dst, f);
#pragma unroll
  for (int i = 0; i < VE; ++i) f[i] = accumulate ? f[i] + acc[i] * scale : acc[i] * scale;
  store_f32<TO, VE>(dst, f);
}

// Rows r0 .. r0 + kZeroCtaRows - 1: zeros where no token has the row's id.  A
// thread per row looks its id up in the sorted list; the more rows share that
// wait (some 15 dependent reads), the less of the time it is.
constexpr int kZeroCtaRows = 64;
template <typename TO, int VE>
__device__ __forceinline__ void zero_rows(const uint32_t* __restrict__ sorted, int64_t n, int64_t n_rows, int64_t dim,
                                          TO* __restrict__ out, int64_t ldo, int64_t r0) {
  __shared__ uint32_t masks[kZeroCtaRows / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x < kZeroCtaRows) {
    const int64_t row = r0 + threadIdx.x;
    int64_t lo = 0, hi = n;  // first position whose id is >= row
    while (lo < hi) {
      const int64_t mid = (lo + hi) >> 1;
      if (sorted[mid] < row) lo = mid + 1;
      else hi = mid;
    }
    const uint32_t mask = __ballot_sync(0xffffffffu, row < n_rows && !(lo < n && sorted[lo] == row));
    if (lane == 0) masks[warp] = mask;
  }
  __syncthreads();
  float zero[VE];
#pragma unroll
  for (int i = 0; i < VE; ++i) zero[i] = 0.f;
  for (int r = warp; r < kZeroCtaRows; r += kGradThreads / 32) {
    if (!((masks[r >> 5] >> (r & 31)) & 1u)) continue;
    TO* dst = out + (r0 + r) * ldo;
    for (int64_t c = static_cast<int64_t>(lane) * VE; c < dim; c += 32 * VE) store_f32<TO, VE>(dst + c, zero);
  }
}

// CTAs 0 .. chunks * slices - 1: one chunk and one slice of the columns each;
// those behind them zero the rows without tokens.  Partial rows: 2 * chunk is
// the part of a run that began before the chunk, 2 * chunk + 1 the part of a
// run that begins in it and goes on behind it.
//
// Bound by memory: 32768 x 2048 bf16 tokens of some 20000 ids into 131072 rows are
// 134 MB read and 537 MB written, of which zeros alone take 90 us (a memset of
// the table takes 136).
template <typename TI, typename TO, int VE, bool ADD>
__global__ void __launch_bounds__(kGradThreads, 8) k_grad_chunks(
    const TI* __restrict__ grad, int64_t ldg, const uint32_t* __restrict__ sorted, const int32_t* __restrict__ perm,
    int64_t n, int64_t n_rows, int64_t dim, float scale, TO* __restrict__ out, int64_t ldo,
    float* __restrict__ partial, int64_t chunks, int slices, int64_t zero_rows_end) {
  if (static_cast<int64_t>(blockIdx.x) >= chunks * slices) {
    zero_rows<TO, VE>(sorted, n, zero_rows_end, dim, out, ldo, (blockIdx.x - chunks * slices) * kZeroCtaRows);
    return;
  }
  // The chunk's ids with their neighbours on both sides (n_rows + 1: none), and its tokens.
  __shared__ uint32_t key[kGradChunk + 2];
  __shared__ int tok[kGradChunk];
  const int64_t chunk = blockIdx.x / slices;
  const int64_t p0 = chunk * kGradChunk;
  if (threadIdx.x < kGradChunk + 2) {
    const int64_t p = p0 + threadIdx.x - 1;
    key[threadIdx.x] = p >= 0 && p < n ? sorted[p] : static_cast<uint32_t>(n_rows + 1);
  } else if (threadIdx.x >= 64 && threadIdx.x < 64 + kGradChunk) {
    const int64_t p = p0 + threadIdx.x - 64;
    const int t = p < n ? perm[p] : -1;
    tok[threadIdx.x - 64] = t < n ? t : -1;
  }
  __syncthreads();
  const int64_t col = (static_cast<int64_t>(blockIdx.x - chunk * slices) * kGradThreads + threadIdx.x) * VE;
  if (col >= dim) return;
  const int have = static_cast<int>(min(static_cast<int64_t>(kGradChunk), n - p0));
  bool open_left = key[0] == key[1];
  constexpr int AHEAD = ADD ? kGradAhead / 2 : kGradAhead;
  float acc[VE];
#pragma unroll
  for (int i = 0; i < VE; ++i) acc[i] = 0.f;
#pragma unroll 1
  for (int q0 = 0; q0 < have; q0 += AHEAD) {
    Raw<TI, VE> f[AHEAD];
    Raw<TO, VE> old[ADD ? AHEAD : 1];  // of the rows that end here
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int q = q0 + u;
      if (q < have && key[q + 1] < n_rows && tok[q] >= 0) {
        f[u].load(grad + static_cast<int64_t>(tok[q]) * ldg + col);
        if (ADD && key[q + 1] != key[q + 2]) old[u].load(out + static_cast<int64_t>(key[q + 1]) * ldo + col);
      }
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int q = q0 + u;
      if (q >= have || key[q + 1] >= n_rows) break;  // ids out of range come last
      if (tok[q] >= 0) {
#pragma unroll
        for (int i = 0; i < VE; ++i) acc[i] += f[u][i];
      }
      const bool last = key[q + 1] != key[q + 2];
      if (last || q + 1 == have) {
        if (open_left) {
          store_f32<float, VE>(partial + (2 * chunk) * dim + col, acc);
        } else if (!last) {
          store_f32<float, VE>(partial + (2 * chunk + 1) * dim + col, acc);
        } else if (!ADD || tok[q] >= 0) {
          float v[VE];
#pragma unroll
          for (int i = 0; i < VE; ++i) v[i] = ADD ? old[ADD ? u : 0][i] + acc[i] * scale : acc[i] * scale;
          store_f32<TO, VE>(out + static_cast<int64_t>(key[q + 1]) * ldo + col, v);
        }
        open_left = false;
#pragma unroll
        for (int i = 0; i < VE; ++i) acc[i] = 0.f;
      }
    }
  }
}

// The chunk in which a run begins that goes on behind it adds up the run's
// parts: kJoinGroups groups of threads take turns of kGradAhead parts each, in
// order, and their sums are added in the order of the groups.
constexpr int kJoinGroups = 2;
template <typename TO, int VE>
__global__ void __launch_bounds__(kGradThreads * kJoinGroups) k_grad_join(const uint32_t* __restrict__ sorted,
                                                                          int64_t n, int64_t n_rows, int64_t dim,
                                                                          float scale, TO* __restrict__ out,
                                                                          int64_t ldo, bool accumulate,
                                                                          const float* __restrict__ partial) {
  __shared__ float sums[kJoinGroups][kGradThreads * VE];
  const int64_t chunk = blockIdx.x;
  const int64_t p0 = chunk * kGradChunk, p1 = p0 + kGradChunk;
  if (p1 >= n) return;
  const uint32_t key = sorted[p1 - 1], after = sorted[p1], start = sorted[p0], before = sorted[p0 > 0 ? p0 - 1 : 0];
  if (key >= n_rows || after != key) return;
  if (p0 > 0 && start == key && before == key) return;  // began earlier
  const int group = threadIdx.x / kGradThreads, thread = threadIdx.x % kGradThreads;
  const int64_t col = (static_cast<int64_t>(blockIdx.y) * kGradThreads + thread) * VE;
  const bool live = col < dim;
  float acc[VE];
#pragma unroll
  for (int i = 0; i < VE; ++i) acc[i] = 0.f;
  if (group == 0 && live) load_f32<float, VE>(partial + (2 * chunk + 1) * dim + col, acc);
  bool more = true;
  for (int64_t c0 = chunk + 1 + group * kGradAhead; more; c0 += kJoinGroups * kGradAhead) {
    float f[kGradAhead][VE];
    bool in[kGradAhead];
#pragma unroll
    for (int u = 0; u < kGradAhead; ++u) {
      const int64_t p = (c0 + u) * kGradChunk;
      in[u] = p < n && sorted[p] == key;
      // read before it is known to be wanted: a chunk that does not begin with
      // this id has another part there, or none
      if (p < n && live) load_f32<float, VE>(partial + 2 * (c0 + u) * dim + col, f[u]);
    }
#pragma unroll
    for (int u = 0; u < kGradAhead; ++u) {
      more = in[u];
      if (!more) break;
#pragma unroll
      for (int i = 0; i < VE; ++i) acc[i] += f[u][i];
    }
  }
#pragma unroll
  for (int i = 0; i < VE; ++i) sums[group][thread * VE + i] = acc[i];
  __syncthreads();
  if (group == 0 && live) {
#pragma unroll
    for (int g = 1; g < kJoinGroups; ++g)
#pragma unroll
      for (int i = 0; i < VE; ++i) acc[i] += sums[g][thread * VE + i];
    emit_row<TO, VE>(out + static_cast<int64_t>(key) * ldo + col, acc, scale, accumulate);
  }
}

// A short list (kFewTokens at most) needs no sorted order: every CTA takes 32
// rows and a slice of the columns, picks the rows' tokens out of the whole list,
// groups them by row in token order, and sums them.  One launch instead of
// three.  A row's place in the sorted order is the number of smaller ids, so the
// sum is cut where the chunks would cut it: the parts are the warps' items,
// and those of one row are added as the join adds them, to the same bits.
// This kernel and the three, 256 tokens (spread and skewed ids), cold: 10000 x 64
// fp32 10 / 14 and 16 / 18 us, 8874 x 512 bf16 12 / 16 and 18 / 21, 8874 x 1024 fp32
// 25 / 27 and 21 / 23, 131072 x 2048 180 / 178 and 176 / 176.  Each CTA groups its
// rows' tokens before its first load and a frequent row is not spread over the
// GPU, so wide rows of middling tables lose: 8874 x 2888 43 / 45 and 39 / 41
// (bf16 33 / 33 and 25 / 27); the length alone decides, because a call that comes
// from the host saves two launches.  An accumulating call looks through
// the list for every 32 rows of the table all the same: 256 tokens into 10^6 x
// 64 take 123 us, 257 through the sort 20.
constexpr int kFewTokens = 256;
constexpr int kFewThreads = 256;
constexpr int kFewWarps = kFewThreads / 32;
constexpr int kFewChunks = kFewTokens / kGradChunk + 1;        // that the tokens of a CTA can have places in
constexpr int kFewItems = kFewRows + kFewChunks;               // parts of the rows of a CTA at most
static_assert(kFewRows == 32 && kJoinGroups == 2, "a lane per row; parts go to the groups in turns of kGradAhead");
template <typename TI, typename TO, typename ID, int VE>
__global__ void __launch_bounds__(kFewThreads) k_grad_few(const TI* __restrict__ grad, int64_t ldg,
                                                          const ID* __restrict__ ids, int n, int64_t n_rows,
                                                          int64_t dim, float scale, TO* __restrict__ out, int64_t ldo,
                                                          bool accumulate, int turns) {
  __shared__ uint16_t tok[kFewTokens], grouped[kFewTokens];  // tokens of these rows, in order; then row by row
  __shared__ uint8_t of[kFewTokens];                         // the row of each of tok, less the first
  __shared__ int counts[2][kFewWarps];
  __shared__ int row_count[kFewRows], row_start[kFewRows], item_row[kFewItems], nitems;
  // Parts of rows of several: in a chunk, one that goes on from before it and one
  // that goes on behind it.
  __shared__ float parts[2 * kFewChunks][32 * VE];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * kFewRows;
  // A warp looks through its share of the list.
  constexpr int TURNS = kFewTokens / kFewThreads;
  const int t0 = warp * (32 * TURNS);
  int64_t id[TURNS];
  int mine = 0, less = 0;
#pragma unroll
  for (int j = 0; j < TURNS; ++j) {
    const int t = t0 + j * 32 + lane;
    id[j] = t < n ? static_cast<int64_t>(ids[t]) : -1;
    if (id[j] >= n_rows) id[j] = -1;
  }
#pragma unroll
  for (int j = 0; j < TURNS; ++j) {
    mine += __popc(__ballot_sync(0xffffffffu, id[j] >= r0 && id[j] < r0 + kFewRows));
    less += __popc(__ballot_sync(0xffffffffu, id[j] >= 0 && id[j] < r0));
  }
  if (lane == 0) {
    counts[0][warp] = mine;
    counts[1][warp] = less;
  }
  __syncthreads();
  int have = 0, before = 0, at = 0;  // tokens of these rows, of smaller ids, of these rows in the warps before
#pragma unroll
  for (int w = 0; w < kFewWarps; ++w) {
    if (w < warp) at += counts[0][w];
    have += counts[0][w];
    before += counts[1][w];
  }
#pragma unroll
  for (int j = 0; j < TURNS; ++j) {
    const bool in = id[j] >= r0 && id[j] < r0 + kFewRows;
    const uint32_t vote = __ballot_sync(0xffffffffu, in);
    if (in) {
      const int to = at + __popc(vote & ((1u << lane) - 1u));
      tok[to] = static_cast<uint16_t>(t0 + j * 32 + lane);
      of[to] = static_cast<uint8_t>(id[j] - r0);
    }
    at += __popc(vote);
  }
  __syncthreads();
  for (int r = warp; r < kFewRows; r += kFewWarps) {
    int c = 0;
    for (int q = lane; q < have; q += 32) c += of[q] == r;
    c = __reduce_add_sync(0xffffffffu, c);
    if (lane == 0) row_count[r] = c;
  }
  __syncthreads();
  if (warp == 0) {
    const int c = row_count[lane];
    int x = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    row_start[lane] = x - c;
    // Parts of the row: the chunks that it has places in.
    const int place = before + x - c;
    const int np = c ? (place + c - 1) / kGradChunk - place / kGradChunk + 1 : 0;
    int y = np;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int z = __shfl_up_sync(0xffffffffu, y, o);
      if (lane >= o) y += z;
    }
    for (int i = 0; i < np; ++i) item_row[y - np + i] = lane | (i << 8);
    if (lane == 31) nitems = y;
  }
  __syncthreads();
  for (int r = warp; r < kFewRows; r += kFewWarps) {
    int to = row_start[r];
    if (!row_count[r]) continue;
    for (int q0 = 0; q0 < have; q0 += 32) {
      const bool in = q0 + lane < have && of[q0 + lane] == r;
      const uint32_t vote = __ballot_sync(0xffffffffu, in);
      if (in) grouped[to + __popc(vote & ((1u << lane) - 1u))] = tok[q0 + lane];
      to += __popc(vote);
    }
  }
  __syncthreads();
#pragma unroll 1
  for (int turn = 0; turn < turns; ++turn) {
    const int64_t c0 = (static_cast<int64_t>(blockIdx.y) * turns + turn) * (32 * VE);
    if (c0 >= dim) break;
    const int64_t c = c0 + static_cast<int64_t>(lane) * VE;
    const bool live = c < dim;
    float acc[VE];
    for (int i = warp; i < nitems; i += kFewWarps) {
      const int r = item_row[i] & 255, part = item_row[i] >> 8;
      const int count = row_count[r], place = before + row_start[r];
      // places of the part, counted from the row's first
      const int p0 = part ? (place / kGradChunk + part) * kGradChunk - place : 0;
      const int p1 = min(count, (place / kGradChunk + part + 1) * kGradChunk - place);
      const uint16_t* list = grouped + row_start[r];
#pragma unroll
      for (int e = 0; e < VE; ++e) acc[e] = 0.f;
      for (int q = p0; q < p1; q += kGradAhead) {
        Raw<TI, VE> f[kGradAhead];
#pragma unroll
        for (int u = 0; u < kGradAhead; ++u)
          if (live && q + u < p1) f[u].load(grad + static_cast<int64_t>(list[q + u]) * ldg + c);
#pragma unroll
        for (int u = 0; u < kGradAhead; ++u) {
          if (!live || q + u >= p1) break;
#pragma unroll
          for (int e = 0; e < VE; ++e) acc[e] += f[u][e];
        }
      }
      if (p0 == 0 && p1 == count) {
        if (live) emit_row<TO, VE>(out + (r0 + r) * ldo + c, acc, scale, accumulate);
      } else {
        const int slot = 2 * (place / kGradChunk + part - before / kGradChunk) + (part == 0);
#pragma unroll
        for (int e = 0; e < VE; ++e) parts[slot][lane * VE + e] = acc[e];
      }
    }
    if (!accumulate) {
#pragma unroll
      for (int e = 0; e < VE; ++e) acc[e] = 0.f;
      for (int r = warp; r < kFewRows && r0 + r < n_rows; r += kFewWarps)
        if (!row_count[r] && live) store_f32<TO, VE>(out + (r0 + r) * ldo + c, acc);
    }
    __syncthreads();
    // Rows of several parts: the first to group 0, then kGradAhead to each group in turn.
    for (int i = warp; i < nitems; i += kFewWarps) {
      const int r = item_row[i] & 255;
      if (item_row[i] >> 8 || i + 1 >= nitems || (item_row[i + 1] & 255) != r) continue;
      const int chunk = (before + row_start[r]) / kGradChunk - before / kGradChunk;
      float group[kJoinGroups][VE];
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        group[0][e] = parts[2 * chunk + 1][lane * VE + e];
        group[1][e] = 0.f;
      }
      for (int k = 1; i + k < nitems && (item_row[i + k] & 255) == r; ++k) {
        const bool second = ((k - 1) / kGradAhead) & 1;
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          const float v = parts[2 * (chunk + k)][lane * VE + e];
          if (second) group[1][e] += v;
          else group[0][e] += v;
        }
      }
#pragma unroll
      for (int e = 0; e < VE; ++e) acc[e] = group[0][e] + group[1][e];
      if (live) emit_row<TO, VE>(out + (r0 + r) * ldo + c, acc, scale, accumulate);
    }
    __syncthreads();
  }
}

size_t grad_ws_bytes(int64_t n, int64_t dim) {
  return static_cast<size_t>(2 * ceil_div64(std::max<int64_t>(n, 1), kGradChunk)) * dim * sizeof(float);
}

template <typename TI, typename TO, int VE>
void grad_launch(const void* grad, int64_t ldg, const int32_t* sorted, const int32_t* perm, int64_t n, int64_t n_rows,
                 int64_t dim, float scale, void* out, int64_t ldo, bool accumulate, float* partial,
                 int64_t zero_rows_end, cudaStream_t s) {
  const int64_t chunks = ceil_div64(n, kGradChunk);
  const int64_t slices = ceil_div64(dim, static_cast<int64_t>(kGradThreads) * VE);
  const int64_t zeros = ceil_div64(zero_rows_end, kZeroCtaRows);
  const uint32_t* keys = reinterpret_cast<const uint32_t*>(sorted);
  TO* o = static_cast<TO*>(out);
  auto* fn = accumulate ? &k_grad_chunks<TI, TO, VE, true> : &k_grad_chunks<TI, TO, VE, false>;
  fn<<<static_cast<unsigned>(chunks * slices + zeros), kGradThreads, 0, s>>>(
      static_cast<const TI*>(grad), ldg, keys, perm, n, n_rows, dim, scale, o, ldo, partial, chunks,
      static_cast<int>(slices), zero_rows_end);
  if (chunks > 1)
    k_grad_join<TO, VE><<<dim3(static_cast<unsigned>(chunks), static_cast<unsigned>(slices)),
                          kGradThreads * kJoinGroups, 0, s>>>(
        keys, n, n_rows, dim, scale, o, ldo, accumulate, partial);
}

// What a gradient call reads and writes.
struct GradArgs {
  const void* grad;
  int64_t ldg;
  const int32_t* sorted;
  const int32_t* perm;
  const void* ids;  // of a short list, instead of sorted and perm
  bool ids64;
  int64_t n, n_rows, dim;
  float scale;
  void* out;
  int64_t ldo;
  bool accumulate;
  float* partial;
  int64_t zero_rows_end;  // rows below it are zeroed where they have no token
};

template <typename TI, typename TO, int VE>
void grad_with(const GradArgs& a, cudaStream_t s) {
  if (!a.ids) {
    grad_launch<TI, TO, VE>(a.grad, a.ldg, a.sorted, a.perm, a.n, a.n_rows, a.dim, a.scale, a.out, a.ldo, a.accumulate,
                            a.partial, a.zero_rows_end, s);
    return;
  }
  // Slices of the columns, in turns of 32 * VE.  Each CTA looks through the whole
  // list, but one that has a frequent id is not to have many columns of it: 256
  // skewed tokens, 8874 x 2888 fp32, take 45 us with two turns (the rule), 53 with
  // one or six and 143 with all; 131072 x 2048 320, 219, 170 and 178 (the rule: all).
  const int64_t groups = ceil_div64(a.n_rows, kFewRows), all = ceil_div64(a.dim, static_cast<int64_t>(32) * VE);
  const int64_t room = 32 * device_sm_count(current_device());
  const int turns = static_cast<int>(ceil_div64(all, std::min(all, std::max<int64_t>(1, room / groups))));
  const dim3 grid(static_cast<unsigned>(groups), static_cast<unsigned>(ceil_div64(all, turns)));
  auto go = [&](auto* ids) {
    using ID = typename std::remove_const<typename std::remove_pointer<decltype(ids)>::type>::type;
    k_grad_few<TI, TO, ID, VE><<<grid, kFewThreads, 0, s>>>(static_cast<const TI*>(a.grad), a.ldg, ids,
                                                           static_cast<int>(a.n), a.n_rows, a.dim, a.scale,
                                                           static_cast<TO*>(a.out), a.ldo, a.accumulate, turns);
  };
  if (a.ids64) go(static_cast<const int64_t*>(a.ids));
  else go(static_cast<const int32_t*>(a.ids));
}

template <typename TI, typename TO>
void grad_pick(int ve, const GradArgs& a, cudaStream_t s) {
  if constexpr (sizeof(TI) == 2 && sizeof(TO) == 2) {
    if (ve == 8) return grad_with<TI, TO, 8>(a, s);
  }
  if (ve >= 4) grad_with<TI, TO, 4>(a, s);
  else if (ve == 2) grad_with<TI, TO, 2>(a, s);
  else grad_with<TI, TO, 1>(a, s);
}

bool aligned(const void* p, int64_t bytes) {
  return reinterpret_cast<uintptr_t>(p) % static_cast<uintptr_t>(bytes) == 0;
}

template <typename TI, typename TO, typename ID>
void lookup_pick(const void* weight, int64_t n_rows, int64_t dim, int64_t ldw, const void* ids, int64_t nids,
                 float scale, void* out, cudaStream_t s) {
  const TI* w = static_cast<const TI*>(weight);
  TO* o = static_cast<TO*>(out);
  const ID* id = static_cast<const ID*>(ids);
  auto go = [&](auto width) {
    constexpr int VE = decltype(width)::value;
    const int64_t per_row = dim / VE;
    int l2 = 0;
    while (l2 < 8 && (int64_t(1) << l2) < per_row) ++l2;
    const int64_t rows = kLookupThreads >> l2;
    // Four rows under way where that leaves every SM a CTA (bf16 rows of 4096: 1024
    // tokens 3.8 us and 4.1 one by one, 8192 22.2 and 33.9); below that a row is cut
    // as long as there are SMs without a CTA (64 tokens: 2.2 us and 2.4).  More CTAs
    // than needed cost time (1024 tokens with every row cut in two: 5.0 us).
    const int64_t sms = device_sm_count(current_device());
    if (nids >= rows * 4 * sms) {
      const unsigned grid = static_cast<unsigned>(std::min<int64_t>(ceil_div64(nids, rows * 4), 1 << 20));
      k_lookup<TI, TO, ID, VE, 4><<<grid, kLookupThreads, 0, s>>>(w, n_rows, dim, ldw, id, nids, scale, o, l2);
    } else {
      const int64_t ctas = ceil_div64(nids, rows);
      const int64_t slices = std::min(ceil_div64(per_row, int64_t(1) << l2), std::max<int64_t>(1, sms / ctas));
      const dim3 grid(static_cast<unsigned>(ctas), static_cast<unsigned>(slices));
      k_lookup<TI, TO, ID, VE, 1><<<grid, kLookupThreads, 0, s>>>(w, n_rows, dim, ldw, id, nids, scale, o, l2);
    }
  };
  auto fits = [&](int64_t ve) {
    return dim % ve == 0 && ldw % ve == 0 && aligned(weight, ve * sizeof(TI)) && aligned(out, ve * sizeof(TO));
  };
  if constexpr (sizeof(TI) == 2 && sizeof(TO) == 2) {
    if (fits(8)) return go(std::integral_constant<int, 8>{});
  }
  if (fits(4)) go(std::integral_constant<int, 4>{});
  else if (fits(2)) go(std::integral_constant<int, 2>{});
  else go(std::integral_constant<int, 1>{});
}

template <typename TI, typename TO>
void lookup_ids(const void* weight, int64_t n_rows, int64_t dim, int64_t ldw, const void* ids, bool ids64,
                int64_t nids, float scale, void* out, cudaStream_t s) {
  if (ids64) lookup_pick<TI, TO, int64_t>(weight, n_rows, dim, ldw, ids, nids, scale, out, s);
  else lookup_pick<TI, TO, int32_t>(weight, n_rows, dim, ldw, ids, nids, scale, out, s);
}

kairo_status sort_tokens(const void* ids, int32_t id_bytes, int64_t n, int64_t n_rows, uint32_t* sorted, int32_t* perm,
                         const ZeroRows& zero, void* ws, cudaStream_t s) {
  return id_bytes == 8 ? sort_launch(static_cast<const int64_t*>(ids), n, n_rows, sorted, perm, ws, zero, s)
                       : sort_launch(static_cast<const int32_t*>(ids), n, n_rows, sorted, perm, ws, zero, s);
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
  if (!ids || !sorted || !perm || !workspace)
    return fail(KAIRO_STATUS_INVALID_VALUE, "null pointer argument");
  if (!aligned(workspace, 16)) return fail(KAIRO_STATUS_INVALID_VALUE, "workspace must be 16-byte aligned");
  if (workspace_bytes < need) return fail(KAIRO_STATUS_WORKSPACE_TOO_SMALL, "token sort workspace too small");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  uint32_t* keys = reinterpret_cast<uint32_t*>(sorted);
  return sort_tokens(ids, id_bytes, nids, n_rows, keys, perm, ZeroRows{}, workspace, s);
}

namespace {

// Workspace: the partial rows, and for a call with ids the sorted order and the
// sort's own.
size_t order_bytes(int64_t n) { return 2 * align_up(static_cast<size_t>(n) * 4, 256); }

kairo_status run_grad(const void* grad_output, int64_t ldg, kairo_dtype dtype, const int32_t* sorted,
                      const int32_t* perm, const void* ids, int32_t id_bytes, int64_t nids, int64_t n_rows,
                      int64_t dim, float scale, void* grad_weight, int64_t ldo, kairo_dtype out_dtype,
                      int32_t accumulate, void* workspace, size_t workspace_bytes, void* stream) {
  if (n_rows < 0 || dim <= 0 || nids < 0) return fail(KAIRO_STATUS_INVALID_VALUE, "invalid size");
  if (nids > kMaxTokens || n_rows > kMaxRows) return fail(KAIRO_STATUS_NOT_SUPPORTED, "too many tokens or rows");
  if (dim > static_cast<int64_t>(65535) * kGradThreads ||
      ceil_div64(nids, kGradChunk) * ceil_div64(dim, kGradThreads) + ceil_div64(n_rows, kFewRows) > 0x7fffffffLL)
    return fail(KAIRO_STATUS_NOT_SUPPORTED, "too many tokens for this width");
  if (ldg < dim || ldo < dim) return fail(KAIRO_STATUS_INVALID_VALUE, "leading dimension smaller than dim");
  if (!known_dtype(dtype) || !known_dtype(out_dtype)) return fail(KAIRO_STATUS_INVALID_VALUE, "unknown dtype");
  if (id_bytes != 4 && id_bytes != 8) return fail(KAIRO_STATUS_INVALID_VALUE, "ids must be int32 or int64");
  if (n_rows == 0) return KAIRO_STATUS_SUCCESS;
  if (!grad_weight) return fail(KAIRO_STATUS_INVALID_VALUE, "null grad_weight");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t ob = element_bytes(out_dtype);
  if (nids == 0) {
    if (accumulate) return KAIRO_STATUS_SUCCESS;
    const cudaError_t e = cudaMemset2DAsync(grad_weight, static_cast<size_t>(ldo * ob), 0,
                                            static_cast<size_t>(dim * ob), static_cast<size_t>(n_rows), s);
    if (e != cudaSuccess) return cuda_fail(e, "cudaMemset2DAsync(grad_weight)");
    return KAIRO_STATUS_SUCCESS;
  }
  if (!grad_output || (!ids && (!sorted || !perm))) return fail(KAIRO_STATUS_INVALID_VALUE, "null pointer argument");
  size_t need = grad_ws_bytes(nids, dim);
  const size_t order_at = align_up(need, 256);
  if (ids) need = nids <= kFewTokens ? 0 : order_at + order_bytes(nids) + sort_ws_bytes(nids);
  if (need > 0 && !workspace) return fail(KAIRO_STATUS_INVALID_VALUE, "null pointer argument");
  if (need > 0 && !aligned(workspace, 16))
    return fail(KAIRO_STATUS_INVALID_VALUE, "workspace must be 16-byte aligned");
  if (workspace_bytes < need) return fail(KAIRO_STATUS_WORKSPACE_TOO_SMALL, "embedding gradient workspace too small");
  GradArgs a{};
  a.grad = grad_output;
  a.ldg = ldg;
  a.sorted = sorted;
  a.perm = perm;
  a.n = nids;
  a.n_rows = n_rows;
  a.dim = dim;
  a.scale = scale;
  a.out = grad_weight;
  a.ldo = ldo;
  a.accumulate = accumulate != 0;
  a.partial = static_cast<float*>(workspace);
  a.zero_rows_end = accumulate ? 0 : n_rows;
  if (ids && nids <= kFewTokens) {
    a.ids = ids;
    a.ids64 = id_bytes == 8;
  } else if (ids) {
    uint8_t* p = static_cast<uint8_t*>(workspace) + order_at;
    int32_t* order = reinterpret_cast<int32_t*>(p);
    int32_t* tokens = reinterpret_cast<int32_t*>(p + order_bytes(nids) / 2);
    // While one cluster sorts, the other SMs zero the last rows, tokens or not:
    // about what they can write in that time (a sort of n tokens takes some 10 us
    // and 0.4 us per 1024, 5 MB are written per us).  Frequent ids are small in
    // most vocabularies, so few of these rows are written again.
    ZeroRows zero{};
    if (!accumulate && nids > kRankTokens && nids <= kClusterTokens && dim * ob % 16 == 0 && ldo * ob % 16 == 0 &&
        aligned(grad_weight, 16)) {
      const int64_t bytes = (int64_t(40) << 20) + nids * 2048;
      zero.rows = std::min(n_rows, bytes / (dim * ob));
      zero.vecs = dim * ob / 16;
      zero.pitch = ldo * ob / 16;
      a.zero_rows_end = n_rows - zero.rows;
      zero.first = reinterpret_cast<uint4*>(static_cast<uint8_t*>(grad_weight) + a.zero_rows_end * ldo * ob);
    }
    const kairo_status st = sort_tokens(ids, id_bytes, nids, n_rows, reinterpret_cast<uint32_t*>(order), tokens, zero,
                                        p + order_bytes(nids), s);
    if (st) return st;
    a.sorted = order;
    a.perm = tokens;
  }
  const int64_t ib = element_bytes(dtype);
  auto fits = [&](int64_t ve) {
    return dim % ve == 0 && ldg % ve == 0 && ldo % ve == 0 && aligned(grad_output, ve * ib) &&
           aligned(grad_weight, ve * ob);
  };
  const int ve = ib == 2 && ob == 2 && fits(8) ? 8 : (fits(4) ? 4 : (fits(2) ? 2 : 1));
  for_types(dtype, out_dtype, [&](auto ti, auto to) { grad_pick<decltype(ti), decltype(to)>(ve, a, s); });
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "launch of the embedding gradient");
  return KAIRO_STATUS_SUCCESS;
}

}  // namespace

extern "C" kairo_status kairo_embedding_grad_workspace_size(int64_t nids, int64_t dim, int32_t sorted, size_t* bytes) {
  if (!bytes || nids < 0 || dim <= 0) return fail(KAIRO_STATUS_INVALID_VALUE, "invalid argument");
  if (sorted) *bytes = grad_ws_bytes(nids, dim);
  else if (nids <= kFewTokens) *bytes = 0;
  else *bytes = align_up(grad_ws_bytes(nids, dim), 256) + order_bytes(nids) + sort_ws_bytes(nids);
  return KAIRO_STATUS_SUCCESS;
}

extern "C" kairo_status kairo_embedding_grad(const void* grad_output, int64_t ldg, kairo_dtype dtype, const void* ids,
                                             int32_t id_bytes, int64_t nids, int64_t n_rows, int64_t dim, float scale,
                                             void* grad_weight, int64_t ldo, kairo_dtype out_dtype, int32_t accumulate,
                                             void* workspace, size_t workspace_bytes, void* stream) {
  if (nids > 0 && n_rows > 0 && !ids) return fail(KAIRO_STATUS_INVALID_VALUE, "null pointer argument");
  return run_grad(grad_output, ldg, dtype, nullptr, nullptr, ids, id_bytes, nids, n_rows, dim, scale, grad_weight, ldo,
                  out_dtype, accumulate, workspace, workspace_bytes, stream);
}

extern "C" kairo_status kairo_embedding_grad_sorted(const void* grad_output, int64_t ldg, kairo_dtype dtype,
                                                    const int32_t* sorted, const int32_t* perm, int64_t nids,
                                                    int64_t n_rows, int64_t dim, float scale, void* grad_weight,
                                                    int64_t ldo, kairo_dtype out_dtype, int32_t accumulate,
                                                    void* workspace, size_t workspace_bytes, void* stream) {
  return run_grad(grad_output, ldg, dtype, sorted, perm, nullptr, 4, nids, n_rows, dim, scale, grad_weight, ldo,
                  out_dtype, accumulate, workspace, workspace_bytes, stream);
}
