// Activations kept in 8 bits for the backward pass.
//
// Every 64 columns of a row share a step.  With a = max |x| of the group,
//   inv  = 127 * (1 / a),  step = a * (1 / 127),     (every operation in fp32)
//   code = round_half_even(x * inv)        (int8, -127 .. 127),
//   x^   = T(code * step)                  in the activation's own type T.
// x * inv is rounded once: fma(x, inv, 1.5 * 2^23) leaves the integer in the
// low bits of the sum, so the product never passes through fp32 and its ties.
// A group with a < 2^-100 keeps zeros (1 / a must not overflow); a group that
// holds an infinity or a NaN gets a NaN step and reads back as NaN, so that a
// broken activation stays visible in the gradient.
//
// Steps are stored column group by column group, (k / 64, n): the weight
// gradient reads the steps of 64 consecutive rows of one group.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "convert.cuh"
#include "internal.h"

namespace kairo {
namespace {

constexpr int kQThreads = 256;
constexpr int kQGroup = 64;   // columns per step
constexpr int kQLanes = 8;    // lanes per group, 8 columns each
constexpr int kQRows = kQThreads / kQLanes;  // rows per CTA
constexpr int kQGroups = 4;   // groups of a row per thread

template <typename T>
__device__ __forceinline__ void load8(const T* p, int64_t left, bool vec, float (&f)[8]) {
  if (vec && left >= 8) {
    if constexpr (sizeof(T) == 4) {
      float lo[4], hi[4];
      load_f32<T, 4>(p, lo);
      load_f32<T, 4>(p + 4, hi);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f[i] = lo[i];
        f[4 + i] = hi[i];
      }
    } else {
      load_f32<T, 8>(p, f);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = i < left ? to_f32<T>(p[i]) : 0.f;
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, int64_t left, bool vec, const float (&f)[8]) {
  if (vec && left >= 8) {
    if constexpr (sizeof(T) == 4) {
      float lo[4] = {f[0], f[1], f[2], f[3]}, hi[4] = {f[4], f[5], f[6], f[7]};
      store_f32<T, 4>(p, lo);
      store_f32<T, 4>(p + 4, hi);
    } else {
      store_f32<T, 8>(p, f);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) p[i] = from_f32<T>(f[i]);
  }
}

template <typename T>
__global__ void __launch_bounds__(kQThreads) k_quantize(const T* __restrict__ x, int64_t n, int64_t k, int64_t ldx,
                                                        bool vec, int8_t* __restrict__ codes, int64_t ldq,
                                                        float* __restrict__ steps, int64_t lds) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kQRows + threadIdx.x / kQLanes;
  const int sub = threadIdx.x % kQLanes;
  const int64_t g0 = static_cast<int64_t>(blockIdx.y) * kQGroups;
  if (row >= n) return;  // whole groups of kQLanes lanes leave together
  const unsigned lanes = 0xffu << (threadIdx.x & 24);
  float f[kQGroups][8];
#pragma unroll
  for (int u = 0; u < kQGroups; ++u) {
    const int64_t c = (g0 + u) * kQGroup + sub * 8;
    load8<T>(x + row * ldx + c, k - c, vec, f[u]);
  }
#pragma unroll
  for (int u = 0; u < kQGroups; ++u) {
    const int64_t c = (g0 + u) * kQGroup + sub * 8;
    if ((g0 + u) * kQGroup >= k) break;
    // magnitudes order as integers, with infinities and NaN on top
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(f[u][i]) & 0x7fffffffu);
#pragma unroll
    for (int o = 1; o < kQLanes; o <<= 1) m = max(m, __shfl_xor_sync(lanes, m, o));
    const float a = __uint_as_float(m);
    const bool broken = m >= 0x7f800000u;
    const bool live = !broken && a >= 0x1p-100f;
    const float inv = live ? __fmul_rn(127.f, __frcp_rn(a)) : 0.f;
    const float step = broken ? __uint_as_float(0x7fffffffu) : (live ? __fmul_rn(a, 1.f / 127.f) : 0.f);
    unsigned w[2] = {0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float s = __fmaf_rn(live ? f[u][i] : 0.f, inv, 12582912.f);
      w[i >> 2] |= (__float_as_uint(s) & 0xffu) << (8 * (i & 3));
    }
    if (c < k) *reinterpret_cast<uint2*>(codes + row * ldq + c) = make_uint2(w[0], w[1]);
    if (sub == 0) steps[(g0 + u) * lds + row] = step;
  }
}

template <typename T>
__global__ void __launch_bounds__(kQThreads) k_dequantize(const int8_t* __restrict__ codes, int64_t ldq,
                                                          const float* __restrict__ steps, int64_t lds, int64_t n,
                                                          int64_t k, T* __restrict__ x, int64_t ldx, bool vec) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kQRows + threadIdx.x / kQLanes;
  const int sub = threadIdx.x % kQLanes;
  const int64_t g0 = static_cast<int64_t>(blockIdx.y) * kQGroups;
  if (row >= n) return;
  uint2 q[kQGroups];
  float step[kQGroups];
#pragma unroll
  for (int u = 0; u < kQGroups; ++u) {
    const int64_t c = (g0 + u) * kQGroup + sub * 8;
    q[u] = make_uint2(0u, 0u);
    step[u] = 0.f;
    if (c < k) {
      q[u] = *reinterpret_cast<const uint2*>(codes + row * ldq + c);
      step[u] = steps[(g0 + u) * lds + row];
    }
  }
#pragma unroll
  for (int u = 0; u < kQGroups; ++u) {
    const int64_t c = (g0 + u) * kQGroup + sub * 8;
    if (c >= k) break;
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const unsigned word = i < 4 ? q[u].x : q[u].y;
      f[i] = static_cast<float>(static_cast<int8_t>(word >> (8 * (i & 3)))) * step[u];
    }
    store8<T>(x + row * ldx + c, k - c, vec, f);
  }
}

kairo_status check_q8(int64_t n, int64_t k, int64_t ldx, kairo_dtype dtype, const void* codes, int64_t ldq,
                      const void* steps, int64_t lds) {
  if (n < 0 || k < 0) return fail(KAIRO_STATUS_INVALID_VALUE, "invalid size");
  if (!known_dtype(dtype)) return fail(KAIRO_STATUS_INVALID_VALUE, "unknown dtype");
  if (ldx < k || ldq < k || lds < n) return fail(KAIRO_STATUS_INVALID_VALUE, "leading dimension too small");
  if (ldq % 16 != 0) return fail(KAIRO_STATUS_INVALID_VALUE, "ldq must be a multiple of 16");
  if (k > int64_t(65535) * kQGroups * kQGroup || n > int64_t(0x7fffffff) * kQRows)
    return fail(KAIRO_STATUS_NOT_SUPPORTED, "activation too large");
  if (n > 0 && k > 0) {
    if (!codes || !steps) return fail(KAIRO_STATUS_INVALID_VALUE, "null pointer argument");
    if (reinterpret_cast<uintptr_t>(codes) % 16) return fail(KAIRO_STATUS_INVALID_VALUE, "codes must be 16-byte aligned");
  }
  return KAIRO_STATUS_SUCCESS;
}

dim3 q8_grid(int64_t n, int64_t k) {
  return dim3(static_cast<unsigned>(ceil_div64(n, kQRows)),
              static_cast<unsigned>(ceil_div64(k, static_cast<int64_t>(kQGroups) * kQGroup)));
}

// 16-byte accesses to x: rows and base aligned.
bool q8_vec(const void* x, int64_t ldx, kairo_dtype dtype) {
  return (ldx * element_bytes(dtype)) % 16 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
}

}  // namespace
}  // namespace kairo

using namespace kairo;

extern "C" kairo_status kairo_quantize_q8(const void* x, int64_t n, int64_t k, int64_t ldx, kairo_dtype dtype,
                                          int8_t* codes, int64_t ldq, float* steps, int64_t lds, void* stream) {
  const kairo_status st = check_q8(n, k, ldx, dtype, codes, ldq, steps, lds);
  if (st) return st;
  if (n == 0 || k == 0) return KAIRO_STATUS_SUCCESS;
  if (!x) return fail(KAIRO_STATUS_INVALID_VALUE, "null pointer argument");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const dim3 g = q8_grid(n, k);
  const bool vec = q8_vec(x, ldx, dtype);
  if (dtype == KAIRO_DTYPE_F32)
    k_quantize<float><<<g, kQThreads, 0, s>>>(static_cast<const float*>(x), n, k, ldx, vec, codes, ldq, steps, lds);
  else if (dtype == KAIRO_DTYPE_F16)
    k_quantize<__half><<<g, kQThreads, 0, s>>>(static_cast<const __half*>(x), n, k, ldx, vec, codes, ldq, steps, lds);
  else
    k_quantize<__nv_bfloat16><<<g, kQThreads, 0, s>>>(static_cast<const __nv_bfloat16*>(x), n, k, ldx, vec, codes, ldq,
                                                      steps, lds);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "launch of the 8-bit quantisation");
  return KAIRO_STATUS_SUCCESS;
}

extern "C" kairo_status kairo_dequantize_q8(const int8_t* codes, int64_t ldq, const float* steps, int64_t lds,
                                            int64_t n, int64_t k, void* x, int64_t ldx, kairo_dtype dtype,
                                            void* stream) {
  const kairo_status st = check_q8(n, k, ldx, dtype, codes, ldq, steps, lds);
  if (st) return st;
  if (n == 0 || k == 0) return KAIRO_STATUS_SUCCESS;
  if (!x) return fail(KAIRO_STATUS_INVALID_VALUE, "null pointer argument");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const dim3 g = q8_grid(n, k);
  const bool vec = q8_vec(x, ldx, dtype);
  if (dtype == KAIRO_DTYPE_F32)
    k_dequantize<float><<<g, kQThreads, 0, s>>>(codes, ldq, steps, lds, n, k, static_cast<float*>(x), ldx, vec);
  else if (dtype == KAIRO_DTYPE_F16)
    k_dequantize<__half><<<g, kQThreads, 0, s>>>(codes, ldq, steps, lds, n, k, static_cast<__half*>(x), ldx, vec);
  else
    k_dequantize<__nv_bfloat16><<<g, kQThreads, 0, s>>>(codes, ldq, steps, lds, n, k, static_cast<__nv_bfloat16*>(x),
                                                        ldx, vec);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "launch of the 8-bit dequantisation");
  return KAIRO_STATUS_SUCCESS;
}

namespace {

// The read-back activation of the weight gradient, rows padded to 16 bytes.
int64_t back_ld(const kairo_bsr* a) { return ceil_div64(a->cols, 8) * 8; }
size_t back_bytes(const kairo_bsr* a, int64_t n) {
  return align_up(static_cast<size_t>(n) * back_ld(a) * element_bytes(a->dtype), 256);
}

}  // namespace

extern "C" kairo_status kairo_bsr_sddmm_q8_workspace_size(const kairo_bsr* a, int64_t n, size_t* bytes) {
  if (!a || !bytes || n < 0) return fail(KAIRO_STATUS_INVALID_VALUE, "invalid argument");
  size_t base = 0;
  const kairo_status st = kairo_bsr_sddmm_workspace_size(a, &base);
  if (st) return st;
  *bytes = align_up(base, 256) + back_bytes(a, n);
  return KAIRO_STATUS_SUCCESS;
}

extern "C" kairo_status kairo_bsr_sddmm_q8(const kairo_bsr* a, const int32_t* row_ptr_t, const int32_t* col_idx_t,
                                           const int32_t* perm_t, const void* dy, int64_t lddy, const int8_t* codes,
                                           int64_t ldq, const float* steps, int64_t lds, int64_t n, void* dblocks,
                                           kairo_dtype out_dtype, void* workspace, size_t workspace_bytes,
                                           void* stream) {
  size_t need = 0, base = 0;
  kairo_status st = kairo_bsr_sddmm_q8_workspace_size(a, n, &need);
  if (st) return st;
  st = check_q8(n, a->cols, a->cols, a->dtype, codes, ldq, steps, lds);
  if (st) return st;
  st = sddmm_check(a, row_ptr_t, col_idx_t, perm_t, dy, lddy, codes, a->cols, n, dblocks, out_dtype, workspace);
  if (st) return st;
  if (a->nnzb == 0) return KAIRO_STATUS_SUCCESS;
  if (!workspace) return fail(KAIRO_STATUS_INVALID_VALUE, "null pointer argument");
  if (workspace_bytes < need) return fail(KAIRO_STATUS_WORKSPACE_TOO_SMALL, "SDDMM workspace too small");
  st = kairo_bsr_sddmm_workspace_size(a, &base);
  if (st) return st;
  uint8_t* back = static_cast<uint8_t*>(workspace) + align_up(base, 256);
  st = kairo_dequantize_q8(codes, ldq, steps, lds, n, a->cols, back, back_ld(a), a->dtype, stream);
  if (st) return st;
  return kairo_bsr_sddmm(a, row_ptr_t, col_idx_t, perm_t, dy, lddy, back, back_ld(a), n, dblocks, out_dtype, workspace,
                         base, stream);
}
