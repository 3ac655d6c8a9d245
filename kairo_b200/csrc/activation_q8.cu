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
#include "q8.cuh"

namespace kairo {
namespace {

constexpr int kQThreads = 256;
constexpr int kQWarps = kQThreads / 32;
constexpr int kQGroup = 64;   // columns per step
constexpr int kQLanes = 8;    // lanes per group, 8 columns each
constexpr int kQCols = 4 * kQGroup;  // columns of a warp: 512 contiguous bytes of a 16-bit row
constexpr int kQRows = 8;     // rows of a warp, all in flight; their steps fill a sector

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

// Eight values of a row as they are stored, and their largest magnitude as the
// bits of a float (magnitudes order as integers, with infinities and NaN on
// top; 16-bit ones two at a time).
template <typename T>
struct Row8 {
  uint32_t w[2 * sizeof(T)];
  __device__ __forceinline__ void load(const T* p, int64_t left, bool vec) {
    if (vec && left >= 8) {
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) {
        const uint4 v = reinterpret_cast<const uint4*>(p)[i];
        w[4 * i] = v.x;
        w[4 * i + 1] = v.y;
        w[4 * i + 2] = v.z;
        w[4 * i + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2 * static_cast<int>(sizeof(T)); ++i) w[i] = 0u;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (i < left) {
          if constexpr (sizeof(T) == 4) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
          else w[i >> 1] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(p)[i]) << (16 * (i & 1));
        }
      }
    }
  }
  __device__ __forceinline__ float value(int i) const {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(w[i]);
    } else {
      const uint16_t b = static_cast<uint16_t>(w[i >> 1] >> (16 * (i & 1)));
      return to_f32<T>(*reinterpret_cast<const T*>(&b));
    }
  }
  __device__ __forceinline__ uint32_t max_bits() const {
    if constexpr (sizeof(T) == 4) {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max(m, w[i] & 0x7fffffffu);
#pragma unroll
      for (int o = 1; o < kQLanes; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
      return m;
    } else {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
#pragma unroll
      for (int o = 1; o < kQLanes; o <<= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
      const uint16_t b = static_cast<uint16_t>(max(m >> 16, m & 0xffffu));
      return __float_as_uint(to_f32<T>(*reinterpret_cast<const T*>(&b)));
    }
  }
};

// A warp takes 256 columns of 8 rows: 32 groups, of which each lane computes
// the two quotients of one.  Bound by memory when that is done (3.06 bytes a
// value of a 16-bit activation; 8192 x 32768 in 128 us, 6.4 TB/s); with the quotients computed by all lanes for
// every row, and the largest magnitude one value at a time, the instructions
// bound it: 8192 x 32768 took 276 us.
template <typename T>
__global__ void __launch_bounds__(kQThreads) k_quantize(const T* __restrict__ x, int64_t n, int64_t k, int64_t ldx,
                                                        bool vec, int8_t* __restrict__ codes, int64_t ldq,
                                                        float* __restrict__ steps, int64_t lds) {
  const int lane = threadIdx.x & 31;
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * kQRows;
  const int64_t c0 = (static_cast<int64_t>(blockIdx.y) * kQWarps + (threadIdx.x >> 5)) * kQCols;
  const int64_t c = c0 + lane * 8;
  if (c0 >= k) return;
  Row8<T> f[kQRows];
#pragma unroll
  for (int u = 0; u < kQRows; ++u) f[u].load(x + (r0 + u) * ldx + c, r0 + u < n ? k - c : 0, vec);
  uint32_t mine = 0;  // largest magnitude of row r0 + lane % 8, group of lane / 8
#pragma unroll
  for (int u = 0; u < kQRows; ++u) {
    const uint32_t m = f[u].max_bits();
    if ((lane & 7) == u) mine = m;
  }
  const float a = __uint_as_float(mine);
  const bool broken = mine >= 0x7f800000u;
  const bool live = !broken && a >= 0x1p-100f;
  const float inv = live ? __fmul_rn(127.f, __frcp_rn(a)) : 0.f;
  const int64_t group = (c0 >> 6) + (lane >> 3), row = r0 + (lane & 7);
  if (group * kQGroup < k && row < n)
    steps[group * lds + row] = broken ? __uint_as_float(0x7fffffffu) : (live ? __fmul_rn(a, 1.f / 127.f) : 0.f);
#pragma unroll
  for (int u = 0; u < kQRows; ++u) {
    const float s = __shfl_sync(0xffffffffu, inv, (lane & 24) + u);
    unsigned w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      unsigned q[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) q[i] = __float_as_uint(__fmaf_rn(f[u].value(4 * h + i), s, 12582912.f));
      w[h] = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
      if (s == 0.f) w[h] = 0u;  // no code of an infinity or NaN
    }
    if (c < k && r0 + u < n) *reinterpret_cast<uint2*>(codes + (r0 + u) * ldq + c) = make_uint2(w[0], w[1]);
  }
}

template <typename T>
__global__ void __launch_bounds__(kQThreads) k_dequantize(const int8_t* __restrict__ codes, int64_t ldq,
                                                          const float* __restrict__ steps, int64_t lds, int64_t n,
                                                          int64_t k, T* __restrict__ x, int64_t ldx, bool vec) {
  const int lane = threadIdx.x & 31;
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * kQRows;
  const int64_t c0 = (static_cast<int64_t>(blockIdx.y) * kQWarps + (threadIdx.x >> 5)) * kQCols;
  const int64_t c = c0 + lane * 8;
  if (c0 >= k) return;
  const int64_t group = (c0 >> 6) + (lane >> 3), row = r0 + (lane & 7);
  const float mine = group * kQGroup < k && row < n ? steps[group * lds + row] : 0.f;
  uint2 q[kQRows];
#pragma unroll
  for (int u = 0; u < kQRows; ++u) {
    q[u] = make_uint2(0u, 0u);
    if (c < k && r0 + u < n) q[u] = *reinterpret_cast<const uint2*>(codes + (r0 + u) * ldq + c);
  }
#pragma unroll
  for (int u = 0; u < kQRows; ++u) {
    const float step = __shfl_sync(0xffffffffu, mine, (lane & 24) + u);
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = code_value(i < 4 ? q[u].x : q[u].y, i & 3) * step;
    store8<T>(x + (r0 + u) * ldx + c, r0 + u < n ? k - c : 0, vec, f);
  }
}

kairo_status check_q8(int64_t n, int64_t k, int64_t ldx, kairo_dtype dtype, const void* codes, int64_t ldq,
                      const void* steps, int64_t lds) {
  if (!known_dtype(dtype)) return fail(KAIRO_STATUS_INVALID_VALUE, "unknown dtype");
  if (ldx < k) return fail(KAIRO_STATUS_INVALID_VALUE, "leading dimension too small");
  const kairo_status st = q8_check(n, k, codes, ldq, steps, lds);
  if (st) return st;
  if (k > int64_t(65535) * kQWarps * kQCols || n > int64_t(0x7fffffff) * kQRows)
    return fail(KAIRO_STATUS_NOT_SUPPORTED, "activation too large");
  return KAIRO_STATUS_SUCCESS;
}

dim3 q8_grid(int64_t n, int64_t k) {
  return dim3(static_cast<unsigned>(ceil_div64(n, kQRows)),
              static_cast<unsigned>(ceil_div64(k, static_cast<int64_t>(kQWarps) * kQCols)));
}

// 16-byte accesses to x: rows and base aligned.
bool q8_vec(const void* x, int64_t ldx, kairo_dtype dtype) {
  return (ldx * element_bytes(dtype)) % 16 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
}

}  // namespace

kairo_status q8_check(int64_t n, int64_t k, const void* codes, int64_t ldq, const void* steps, int64_t lds) {
  if (n < 0 || k < 0) return fail(KAIRO_STATUS_INVALID_VALUE, "invalid size");
  if (ldq < k || lds < n) return fail(KAIRO_STATUS_INVALID_VALUE, "leading dimension too small");
  if (ldq % 16 != 0) return fail(KAIRO_STATUS_INVALID_VALUE, "ldq must be a multiple of 16");
  if (n > 0 && k > 0) {
    if (!codes || !steps) return fail(KAIRO_STATUS_INVALID_VALUE, "null pointer argument");
    if (reinterpret_cast<uintptr_t>(codes) % 16)
      return fail(KAIRO_STATUS_INVALID_VALUE, "codes must be 16-byte aligned");
  }
  return KAIRO_STATUS_SUCCESS;
}

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

extern "C" kairo_status kairo_bsr_sddmm_q8_workspace_size(const kairo_bsr* a, int64_t n, size_t* bytes) {
  if (!a || !bytes || n < 0) return fail(KAIRO_STATUS_INVALID_VALUE, "invalid argument");
  return kairo_bsr_sddmm_workspace_size(a, bytes);
}
