// 8-bit floats (e4m3: sign, four exponent bits, three mantissa bits, no infinity,
// magnitudes to 448) with a power of two for several values: a cache's type.
#pragma once

#include <type_traits>

#include "nibble_copy.h"

namespace nibble {

// The powers of two, biased by 127, under which 8-bit floats are values of a 16-bit
// type: the smallest of the first, 2^-9, is fp16's least step or bf16's least normal
// value; the last ends at 240 (kFloat8LastMax), beyond which the type does.
constexpr float kFloat8Max = 448.0f, kFloat8LastMax = 240.0f;
template <class E>
constexpr int kLowExponent = std::is_same_v<E, Half> ? 127 - 15 : 127 - 117;
template <class E>
constexpr int kHighExponent = std::is_same_v<E, Half> ? 127 + 8 : 127 + 120;
template <class E>
constexpr float kLargest = std::is_same_v<E, Half> ? 65504.0f : 0x1.fep127f;

// The least exponent for which top <= 448 2^(e - 127): 448 is 1.75 2^8.
template <class E>
__device__ __forceinline__ int exponent_for(float top) {
  const uint32_t bits = __builtin_bit_cast(uint32_t, top);
  const int e = static_cast<int>(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, kLowExponent<E>), kHighExponent<E>);
}
// 2^(e - 127) of a biased exponent, and its inverse.
__device__ __forceinline__ float power(int e) {
  return __builtin_bit_cast(float, static_cast<uint32_t>(e) << 23);
}

// Eight values of a 16-bit type from eight 8-bit floats and their power of two.
template <class E>
__device__ __forceinline__ typename E::vec8 from_float8(uint32_t lo, uint32_t hi, float slo,
                                                        float shi) {
  typename E::vec8 y;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int word = static_cast<int>(i < 2 ? lo : hi);
    const float s = i < 2 ? slo : shi;
    if constexpr (std::is_same_v<E, Half>) {
      const auto p = i & 1 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, s, true)
                           : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, s, false);
      y[2 * i] = p[0], y[2 * i + 1] = p[1];
    } else {
      const auto p = i & 1 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, s, true)
                           : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, s, false);
      y[2 * i] = p[0], y[2 * i + 1] = p[1];
    }
  }
  return y;
}

// Four 8-bit floats, each the nearest to its value, ties to even; what is not finite
// becomes NaN.  (Values are within the range already.)
__device__ __forceinline__ uint32_t to_float8(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true));
}

}  // namespace nibble
