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

#include "convert.cuh"
#include "internal.h"

namespace kairo {
namespace {

// Plan memory, int32 words: the token order (T), then starts (G + 2): the
// tokens of adapter a are order[starts[a] .. starts[a + 1]), those without one
// order[starts[G] .. starts[G + 1]).
struct Plan {
  int32_t* order;
  int32_t* starts;
};

Plan carve_plan(void* mem, int64_t t) {
  int32_t* p = static_cast<int32_t*>(mem);
  return Plan{p, p + align_up(static_cast<size_t>(t), 64)};
}

size_t plan_bytes(int64_t t, int64_t g) {
  return (align_up(static_cast<size_t>(t), 64) + align_up(static_cast<size_t>(g + 2), 64)) * sizeof(int32_t);
}

__global__ void k_plan_starts(const uint32_t* __restrict__ sorted, int64_t t, int64_t g, int32_t* __restrict__ starts) {
  for (int64_t a = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; a < g + 2;
       a += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    int64_t lo = 0, hi = t;  // first position whose key is >= a
    while (lo < hi) {
      const int64_t mid = (lo + hi) >> 1;
      if (sorted[mid] < static_cast<uint32_t>(a)) lo = mid + 1;
      else hi = mid;
    }
    starts[a] = static_cast<int32_t>(lo);
  }
}

// The adapter of a position of the order (g: none).
__device__ __forceinline__ int64_t adapter_at(const int32_t* starts, int64_t g, int64_t p) {
  int64_t lo = 0, hi = g;  // last a with starts[a] <= p and tokens behind it
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (starts[mid + 1] <= p) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

// One warp per (position, rank row).
template <typename T>
__global__ void __launch_bounds__(256) k_low(const T* __restrict__ x, int64_t ldx, int64_t k,
                                             const T* __restrict__ down, int64_t rank,
                                             const float* __restrict__ scale, const int32_t* __restrict__ order,
                                             const int32_t* __restrict__ starts, int64_t t, int64_t g,
                                             float* __restrict__ low) {
  const int lane = threadIdx.x & 31;
  const int64_t w = (blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x) >> 5;
  const int64_t p = w / rank, r = w - p * rank;
  if (p >= t) return;
  const int64_t tok = order[p];
  const int64_t a = adapter_at(starts, g, p);
  float acc = 0.f;
  if (a < g) {
    const T* xr = x + tok * ldx;
    const T* dr = down + (a * rank + r) * k;
    for (int64_t c = lane; c < k; c += 32) acc += to_f32<T>(xr[c]) * to_f32<T>(dr[c]);
    for (int o = 16; o; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
    if (scale) acc *= scale[a];
  }
  if (lane == 0) low[tok * rank + r] = acc;
}

template <typename T, typename TB, typename TY>
__global__ void __launch_bounds__(256) k_expand(const float* __restrict__ low, int64_t rank,
                                                const T* __restrict__ up, int64_t n, const TB* base, int64_t ldb,
                                                TY* y, int64_t ldy, const int32_t* __restrict__ order,
                                                const int32_t* __restrict__ starts, int64_t t, int64_t g) {
  const int64_t p = blockIdx.x;
  const int64_t tok = order[p];
  const int64_t a = adapter_at(starts, g, p);
  for (int64_t c = static_cast<int64_t>(blockIdx.y) * blockDim.x + threadIdx.x; c < n;
       c += static_cast<int64_t>(gridDim.y) * blockDim.x) {
    float acc = base ? to_f32<TB>(base[tok * ldb + c]) : 0.f;
    if (a < g) {
      float d = 0.f;
      for (int64_t r = 0; r < rank; ++r) d += low[tok * rank + r] * to_f32<T>(up[(a * rank + r) * n + c]);
      acc += d;
    }
    y[tok * ldy + c] = from_f32<TY>(acc);
  }
}

// grad[a, r, c] = sum over the adapter's tokens of s[t, r] * z[t, c].
template <typename T, typename TG>
__global__ void __launch_bounds__(128) k_low_wgrad(const float* __restrict__ s, int64_t rank,
                                                   const T* __restrict__ z, int64_t ldz, int64_t k,
                                                   const int32_t* __restrict__ order,
                                                   const int32_t* __restrict__ starts, TG* __restrict__ grad) {
  const int64_t c = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int64_t a = blockIdx.y;
  if (c >= k) return;
  const int p0 = starts[a], p1 = starts[a + 1];
  for (int64_t r0 = 0; r0 < rank; r0 += 8) {
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int p = p0; p < p1; ++p) {
      const int64_t tok = order[p];
      const float v = to_f32<T>(z[tok * ldz + c]);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (r0 + i < rank) acc[i] += s[tok * rank + r0 + i] * v;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (r0 + i < rank) grad[(a * rank + r0 + i) * k + c] = from_f32<TG>(acc[i]);
  }
}

constexpr int64_t kMaxAdapters = 65535;
constexpr int64_t kMaxRank = 128;

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

template <typename T, typename TB, typename TY>
void apply_launch(const void* x, int64_t ldx, int64_t k, const void* down, const void* up, int64_t n, int64_t rank,
                  const float* scale, const Plan& pl, int64_t t, int64_t g, const void* base, int64_t ldb, void* y,
                  int64_t ldy, float* low, cudaStream_t s) {
  k_low<T><<<static_cast<unsigned>(ceil_div64(t * rank, 8)), 256, 0, s>>>(
      static_cast<const T*>(x), ldx, k, static_cast<const T*>(down), rank, scale, pl.order, pl.starts, t, g, low);
  if (!y) return;
  const dim3 grid(static_cast<unsigned>(t), static_cast<unsigned>(std::min<int64_t>(ceil_div64(n, 256), 64)));
  k_expand<T, TB, TY><<<grid, 256, 0, s>>>(low, rank, static_cast<const T*>(up), n, static_cast<const TB*>(base), ldb,
                                          static_cast<TY*>(y), ldy, pl.order, pl.starts, t, g);
}

template <typename T>
void apply_types(kairo_dtype base_dtype, kairo_dtype y_dtype, const void* x, int64_t ldx, int64_t k, const void* down,
                 const void* up, int64_t n, int64_t rank, const float* scale, const Plan& pl, int64_t t, int64_t g,
                 const void* base, int64_t ldb, void* y, int64_t ldy, float* low, cudaStream_t s) {
  const bool bf = base_dtype == KAIRO_DTYPE_F32, yf = y_dtype == KAIRO_DTYPE_F32;
  if (bf && yf)
    apply_launch<T, float, float>(x, ldx, k, down, up, n, rank, scale, pl, t, g, base, ldb, y, ldy, low, s);
  else if (bf)
    apply_launch<T, float, T>(x, ldx, k, down, up, n, rank, scale, pl, t, g, base, ldb, y, ldy, low, s);
  else if (yf)
    apply_launch<T, T, float>(x, ldx, k, down, up, n, rank, scale, pl, t, g, base, ldb, y, ldy, low, s);
  else
    apply_launch<T, T, T>(x, ldx, k, down, up, n, rank, scale, pl, t, g, base, ldb, y, ldy, low, s);
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
  *plan = plan_bytes(ntokens, nadapters);
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
  if (plan_size < need) return fail(KAIRO_STATUS_INVALID_VALUE, "plan memory too small");
  if (workspace_bytes < ws_need) return fail(KAIRO_STATUS_WORKSPACE_TOO_SMALL, "adapter plan workspace too small");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const Plan pl = carve_plan(plan, ntokens);
  int32_t* sorted = static_cast<int32_t*>(workspace);
  const size_t col = align_up(static_cast<size_t>(ntokens) * sizeof(int32_t), 256);
  st = kairo_token_sort(ids, id_bytes, ntokens, nadapters, sorted, pl.order, static_cast<uint8_t*>(workspace) + col,
                        workspace_bytes - col, stream);
  if (st) return st;
  k_plan_starts<<<static_cast<unsigned>(ceil_div64(nadapters + 2, 256)), 256, 0, s>>>(
      reinterpret_cast<const uint32_t*>(sorted), ntokens, nadapters, pl.starts);
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
  if (ldx < k || (y && ldy < n) || (base && ldb < n)) return fail(KAIRO_STATUS_INVALID_VALUE, "leading dimension too small");
  if (ntokens == 0) return KAIRO_STATUS_SUCCESS;
  if (!x || !plan || !low || (nadapters > 0 && (!down || (y && !up))))
    return fail(KAIRO_STATUS_INVALID_VALUE, "null pointer argument");
  const Plan pl = carve_plan(const_cast<void*>(plan), ntokens);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (!base) base_dtype = dtype;
  if (dtype == KAIRO_DTYPE_F16)
    apply_types<__half>(base_dtype, y_dtype, x, ldx, k, down, up, n, rank, scale, pl, ntokens, nadapters, base, ldb, y,
                        ldy, low, s);
  else
    apply_types<__nv_bfloat16>(base_dtype, y_dtype, x, ldx, k, down, up, n, rank, scale, pl, ntokens, nadapters, base,
                               ldb, y, ldy, low, s);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "launch of the low-rank product");
  return KAIRO_STATUS_SUCCESS;
}

extern "C" kairo_status kairo_low_rank_wgrad(const float* low, int64_t rank, const void* z, int64_t ldz, int64_t k,
                                             kairo_dtype dtype, const void* plan, int64_t ntokens, int64_t nadapters,
                                             void* grad, kairo_dtype grad_dtype, void* stream) {
  const kairo_status st = check_low_rank(ntokens, k, 1, rank, nadapters, dtype);
  if (st) return st;
  if (grad_dtype != KAIRO_DTYPE_F32 && grad_dtype != dtype)
    return fail(KAIRO_STATUS_INVALID_VALUE, "the gradient must be fp32 or the adapters' dtype");
  if (ldz < k) return fail(KAIRO_STATUS_INVALID_VALUE, "leading dimension too small");
  if (nadapters == 0) return KAIRO_STATUS_SUCCESS;
  if (!plan || !grad || (ntokens > 0 && (!low || !z))) return fail(KAIRO_STATUS_INVALID_VALUE, "null pointer argument");
  const Plan pl = carve_plan(const_cast<void*>(plan), ntokens);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(ceil_div64(k, 128)), static_cast<unsigned>(nadapters));
  auto go = [&](auto zt, auto gt) {
    using T = decltype(zt);
    using TG = decltype(gt);
    k_low_wgrad<T, TG><<<grid, 128, 0, s>>>(low, rank, static_cast<const T*>(z), ldz, k, pl.order, pl.starts,
                                           static_cast<TG*>(grad));
  };
  if (dtype == KAIRO_DTYPE_F16) grad_dtype == KAIRO_DTYPE_F32 ? go(__half{}, float{}) : go(__half{}, __half{});
  else grad_dtype == KAIRO_DTYPE_F32 ? go(__nv_bfloat16{}, float{}) : go(__nv_bfloat16{}, __nv_bfloat16{});
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "launch of the adapter gradient");
  return KAIRO_STATUS_SUCCESS;
}
