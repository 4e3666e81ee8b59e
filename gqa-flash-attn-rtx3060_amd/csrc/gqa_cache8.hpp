// gqa_cache8.hpp — a paged K/V cache in 8 bits, as its kernels see it.
//
// A value is held as an e4m3 code (1 sign, 4 exponent, 3 mantissa bits; largest
// 448, least step 2^-9) times 2^e, with one whole exponent e for the tokens of a page
// and kv head, keys and values each.  e4m3 has an exponent of its own, so a power of
// two as the scale loses nothing against any other: the rounding is half a step of
// 2^-4 of the value wherever the scale lies, down to 2^-15 of the page's largest; and
// bringing a page's codes to a larger e rounds those alone that fall below 2^-6 of
// its unit, so a page can be filled token by token.  The products with it are
// exact, and the conversion instruction applies it: a code times 2^e is a number of
// bf16, and of fp16 where it is in its range.
#pragma once

#include "gqa_common.hpp"
#include "gqa_params.hpp"

namespace gqa {

constexpr int kExpMin = -126, kExpMax = 126;  // (2^e and 2^-e are normal numbers)
// Exponents are read from memory that a caller may have left as it came.
__device__ inline int clamp_exp(int e) { return min(max(e, kExpMin), kExpMax); }
__device__ inline float exp_scale(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// The least e with most <= 448 * 2^e = 1.75 * 2^(e + 8).
__device__ inline int exponent_of(float most) {
  const int e = (int)((__float_as_uint(most) + 0x1FFFFFu) >> 23) - 135;
  return clamp_exp(e);
}

// Two codes (the lower or upper half of w) times scale, a power of two, as two
// 16-bit values.
template <int DT, bool HI> __device__ inline uint32_t widen2(uint32_t w, float scale) {
  if constexpr (DT == 0) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HI));
  else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, HI));
}
// Eight codes, the first four of one scale and the others of another.
template <int DT> __device__ inline u32x4 widen8(uint32_t a, float sa, uint32_t b, float sb) {
  return u32x4{widen2<DT, false>(a, sa), widen2<DT, true>(a, sa), widen2<DT, false>(b, sb), widen2<DT, true>(b, sb)};
}

// Four values (at most 448 in size) as codes, to the nearest, ties to even.
__device__ inline uint32_t codes4(float a, float b, float c, float d) {
  uint32_t w = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, (int)w, true);
}

}  // namespace gqa
