// Conversions between the element types of the C ABI and fp32, and short
// vectors of them: 16- or 8-byte loads and stores with every value held in
// fp32 in between.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "../../include/kairo_spmm.h"

namespace kairo {

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

// One rounding (to nearest, ties to even) from fp32.
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// The words of N elements of T, aligned to their whole size.
template <int BYTES>
struct Words;
template <>
struct Words<2> { using type = uint16_t; };
template <>
struct Words<4> { using type = uint32_t; };
template <>
struct Words<8> { using type = uint2; };
template <>
struct Words<16> { using type = uint4; };

template <typename T, int N>
struct Pack {
  union {
    typename Words<N * static_cast<int>(sizeof(T))>::type raw;
    T v[N];
  };
  __device__ __forceinline__ Pack() {}
};

// N elements at p, in pieces of up to 16 bytes; p is aligned to a piece.
template <typename T, int N>
__device__ __forceinline__ void load_f32(const T* p, float (&f)[N]) {
  constexpr int P = N * static_cast<int>(sizeof(T)) > 16 ? 16 / static_cast<int>(sizeof(T)) : N;
#pragma unroll
  for (int q = 0; q < N; q += P) {
    Pack<T, P> k;
    k.raw = *reinterpret_cast<const decltype(k.raw)*>(p + q);
#pragma unroll
    for (int i = 0; i < P; ++i) f[q + i] = to_f32<T>(k.v[i]);
  }
}

template <typename T, int N>
__device__ __forceinline__ void store_f32(T* p, const float (&f)[N]) {
  constexpr int P = N * static_cast<int>(sizeof(T)) > 16 ? 16 / static_cast<int>(sizeof(T)) : N;
#pragma unroll
  for (int q = 0; q < N; q += P) {
    Pack<T, P> k;
#pragma unroll
    for (int i = 0; i < P; ++i) k.v[i] = from_f32<T>(f[q + i]);
    *reinterpret_cast<decltype(k.raw)*>(p + q) = k.raw;
  }
}

// The same N elements as they are stored, converted when they are used: half the
// registers of fp32 values while 16-bit loads are under way.
template <typename T, int N>
struct Raw {
  static constexpr int P = N * static_cast<int>(sizeof(T)) > 16 ? 16 / static_cast<int>(sizeof(T)) : N;
  Pack<T, P> piece[N / P];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int q = 0; q < N / P; ++q) piece[q].raw = *reinterpret_cast<const decltype(piece[q].raw)*>(p + q * P);
  }
  __device__ __forceinline__ float operator[](int i) const { return to_f32<T>(piece[i / P].v[i % P]); }
};

inline int element_bytes(kairo_dtype d) { return d == KAIRO_DTYPE_F32 ? 4 : 2; }
inline bool known_dtype(kairo_dtype d) {
  return d == KAIRO_DTYPE_F32 || d == KAIRO_DTYPE_F16 || d == KAIRO_DTYPE_BF16;
}

}  // namespace kairo
