// Rounding of activations to e4m3 with a power-of-two scale per 128 elements, shared by the quantiser and the products that round their rows themselves.
#pragma once
#include "common.cuh"
#include <cuda_fp8.h>

namespace mx {

constexpr int FP8_BLOCK = 128;   // elements of K per scale
constexpr int FP8_ROWS = 16;     // weight rows per scale

// Scale of a block with largest magnitude `amax`: the smallest power of two, 2^-100 at least, with amax <= 448 scale; 1 for zeros, NaN for infinities and NaN
// (the caller then writes zero codes).  *inv = 1 / scale, a power of two as well: x * inv is exact, so the codes are those of a division.
__device__ __forceinline__ float fp8_scale(float amax, float* inv) {
  const uint32_t bits = __float_as_uint(amax);
  *inv = 1.f;
  if (bits >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  if (bits == 0) return 1.f;
  int e = (int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u);      // biased: 448 = 1.75 * 2^8
  e = max(e, 27);
  *inv = __uint_as_float((uint32_t)(254 - e) << 23);
  return __uint_as_float((uint32_t)e << 23);
}
// max |v| as bits, NaN above infinity (magnitudes of floats order like their bits)
__device__ __forceinline__ uint32_t fp8_mag(float v) { return __float_as_uint(v) & 0x7fffffffu; }

__device__ __forceinline__ uint32_t fp8_pack4(float a, float b, float c, float d) {
  const __nv_fp8x2_storage_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const __nv_fp8x2_storage_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return (uint32_t)lo | ((uint32_t)hi << 16);
}

}  // namespace mx
