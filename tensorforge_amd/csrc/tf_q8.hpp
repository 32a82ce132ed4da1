// Conversions and geometry of the 8-bit paged KV cache (e4m3 codes with a
// power-of-two scale for each page and kv head).
#pragma once

#include "tf_common.hpp"

namespace tf {

constexpr int32_t kLowestExponent = -126;

inline int32_t check_q8_geometry(int32_t kv_heads, int32_t head_dim, int32_t num_blocks, int32_t block_size) {
  if (kv_heads <= 0 || head_dim <= 0 || num_blocks <= 0 || block_size <= 0)
    return fail(TF_ERROR_INVALID_ARGUMENT, "cache dimensions must be positive");
  if (head_dim % 16 != 0 || head_dim > 256)
    return fail(TF_ERROR_UNSUPPORTED, "the 8-bit cache takes head dimensions that are multiples of 16 up to 256");
  if (block_size % 16 != 0 || block_size > 1024)
    return fail(TF_ERROR_UNSUPPORTED, "the 8-bit cache takes pages of a multiple of 16 tokens up to 1024");
  return TF_SUCCESS;
}

// |x| as an ordered integer, 0 for infinities and NaN.
__device__ __forceinline__ uint32_t finite_bits(float x) {
  const uint32_t bits = __builtin_bit_cast(uint32_t, x) & 0x7fffffffu;
  return bits < 0x7f800000u ? bits : 0u;
}

// The smallest t >= -126 with x <= 448 * 2^t for the float with these bits:
// 448 = 1.75 * 2^8.  (Subnormal x: any t >= -126 will do.)
__device__ __forceinline__ int32_t smallest_exponent(uint32_t bits) {
  const int32_t t = static_cast<int32_t>(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return t < kLowestExponent ? kLowestExponent : t;
}

__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
#pragma unroll
  for (int offset = 32; offset > 0; offset >>= 1) v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), offset, 64)));
  return v;
}

// e4m3 of four values, |x| <= 448 or NaN, round to nearest even, in a word.
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
  const int low = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, low, true));
}

// x * 2^-exponent; infinities become NaN (e4m3 has no infinity).
__device__ __forceinline__ float scaled(float x, int32_t exponent) {
  const bool finite = (__builtin_bit_cast(uint32_t, x) & 0x7fffffffu) < 0x7f800000u;
  return finite ? ldexpf(x, -exponent) : __builtin_nanf("");
}

// The codes of four values under a scale of 2^exponent.
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d, int32_t exponent) {
  return pack4(scaled(a, exponent), scaled(b, exponent), scaled(c, exponent), scaled(d, exponent));
}

// Four codes times 2^exponent.
__device__ __forceinline__ void decode4(uint32_t codes, int32_t exponent, float *x) {
  const int word = static_cast<int>(codes);
  x[0] = ldexpf(__builtin_amdgcn_cvt_f32_fp8(word, 0), exponent);
  x[1] = ldexpf(__builtin_amdgcn_cvt_f32_fp8(word, 1), exponent);
  x[2] = ldexpf(__builtin_amdgcn_cvt_f32_fp8(word, 2), exponent);
  x[3] = ldexpf(__builtin_amdgcn_cvt_f32_fp8(word, 3), exponent);
}

// Four codes rounded to a scale 2^-exponent times theirs (exponent < 0).
__device__ __forceinline__ uint32_t rescale4(uint32_t codes, int32_t exponent) {
  float x[4];
  decode4(codes, exponent, x);
  return pack4(x[0], x[1], x[2], x[3]);
}

}  // namespace tf
