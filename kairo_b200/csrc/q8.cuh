// Reading 8-bit activations back (activation_q8.cu has their definition).
#pragma once

#include "convert.cuh"

namespace kairo {

// Two fp32 values rounded to T, the first in the low half.
template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack_pair<__half>(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack_pair<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Code `i` of four as a float.  With its sign bit flipped it is the low byte of
// the float 2^23 + 128 + code: one byte permutation and one exact subtraction, both
// at the full rate that a conversion instruction does not have.
__device__ __forceinline__ float code_value(uint32_t four, int i) {
  return __uint_as_float(__byte_perm(four ^ 0x80808080u, 0x4b000000u, 0x7650u + static_cast<unsigned>(i))) - 8388736.f;
}

// Eight codes times their step, rounded to T.
template <typename T>
__device__ __forceinline__ uint4 read_back(uint2 q, float step) {
  const uint32_t b[2] = {q.x, q.y};
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e)
    w[e] = pack_pair<T>(__fmul_rn(code_value(b[e >> 1], (e & 1) * 2), step),
                        __fmul_rn(code_value(b[e >> 1], (e & 1) * 2 + 1), step));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// The first `n` of eight 16-bit values, the others zero.
__device__ __forceinline__ uint4 keep_first(uint4 v, int n) {
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (n <= 2 * e) w[e] = 0u;
    else if (n == 2 * e + 1) w[e] &= 0xffffu;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

}  // namespace kairo
