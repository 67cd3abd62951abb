// The 8-bit cache format and its conversions.
//
// K and V are e4m3 bytes (4 significant bits, largest value 448, least 2^-9, NaN
// 0x7F / 0xFF); for each block of tokens and KV head scales[block, head, 0 (K) or 1
// (V)] is the biased exponent e of a power of two, and a byte stands for
// e4m3 * 2^(e - 127). A power of two, because it costs e4m3 no precision (its
// relative step is the same at every scale), raising it later re-rounds only what
// gets subnormal, and every value is exact in bf16 (e >= kLeastExponent keeps it
// normal there).
#pragma once

#include "common.h"

namespace vrh {

constexpr int kLeastExponent = 27;  // 2^-100

// Biased exponent of the least power of two s with amax <= 448 s = 1.75 * 2^8 s.
__device__ __forceinline__ int q8_exponent(float amax) {
  const uint32_t u = __float_as_uint(amax);
  return max((int)(u >> 23) - 8 + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0), kLeastExponent);
}

// 2^(e - 127) for e in [0, 254]; e = 0 gives 0, 255 infinity.
__device__ __forceinline__ float q8_scale(int e) { return __uint_as_float((uint32_t)e << 23); }

// Four e4m3 bytes to floats (exact).
__device__ __forceinline__ void q8_unpack4(uint32_t x, float (&out)[4]) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)x, false);
  const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)x, true);
  out[0] = lo[0];
  out[1] = lo[1];
  out[2] = hi[0];
  out[3] = hi[1];
}

// Four floats to e4m3, to nearest even; NaN, infinities and values that would round
// past 448 become NaN.
__device__ __forceinline__ uint32_t q8_pack4(float a, float b, float c, float d) {
  int x = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  x = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, x, true);
  return (uint32_t)x;
}

__device__ __forceinline__ float q8_to_f32(uint8_t x) {
  return __builtin_amdgcn_cvt_f32_fp8((int)x, 0);
}
__device__ __forceinline__ uint8_t q8_from_f32(float x) {
  return (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(x, x, 0, false);
}

}  // namespace vrh
