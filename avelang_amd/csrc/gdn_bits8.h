// 8-bit codes with a scale per row: e4m3 (largest value 448) and integers
// (-127 .. 127), rounded to nearest with ties to even.
#pragma once

#include "gdn_common.h"
#include "../../include/gdn_attn.h"

namespace gdn {

// words at any byte
typedef uint32_t u32b __attribute__((aligned(1)));
typedef uint32_t u32x2b __attribute__((ext_vector_type(2), aligned(1)));

// |f|'s bits: their order is that of the values, infinity and NaN above all.
__device__ __forceinline__ uint32_t abs_bits(float f) { return __float_as_uint(f) & 0x7fffffffu; }
constexpr uint32_t kInfBits = 0x7f800000u;

__host__ __device__ constexpr float largest8(int code) { return code == GDN_DTYPE_E4M3 ? 448.f : 127.f; }

// Four values within the codes' range as four codes.
__device__ __forceinline__ uint32_t e4m3_4(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}
__device__ __forceinline__ uint32_t int8_1(float a) { return (uint32_t)(int)rintf(a) & 0xffu; }
__device__ __forceinline__ uint32_t int8_4(float a, float b, float c, float d) {
  return int8_1(a) | int8_1(b) << 8 | int8_1(c) << 16 | int8_1(d) << 24;
}

// Scale of a row from its largest |value|'s bits: max / M, 0 for a row of
// zeros, no less than that of 2^-100 (M / max and codes stay finite), NaN for
// one that is not finite (`also`: a sum of its squares that may have
// overflowed).  inv = M / max.
struct Row8 {
  float scale, inv;
};
__device__ __forceinline__ Row8 row8(uint32_t bits, int code, float also = 0.f) {
  const float M = largest8(code), m = fmaxf(__uint_as_float(bits), 0x1p-100f);
  if (bits >= kInfBits || abs_bits(also) >= kInfBits) return {__builtin_nanf(""), __builtin_nanf("")};
  return {bits ? m / M : 0.f, M / m};
}

}  // namespace gdn
