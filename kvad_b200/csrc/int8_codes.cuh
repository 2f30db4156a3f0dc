// Numbers to 8-bit codes: c = x / s rounded to the nearest integer, halves to the even one, -127 .. 127, with s = max|x| / 127 of the row.
//
// The code is that of the correctly rounded quotient, which is what a reader of the definition computes; a division takes ten times a product, so the product with
// 1 / s decides wherever it is not within 2^-10 of a half (it is off by less than 2^-15), and the division where it is.
#pragma once
#include "common.cuh"

namespace kvad {

struct Scale {
  float s, inverse;      // inverse 0: a row without codes (zeros, or a number that is not finite)
  bool small;            // s is below the smallest normal number: divisions throughout
};

// `top`: the bits of the row's largest magnitude; NaN and infinity are above every finite number.
__device__ __forceinline__ Scale scale_of(uint32_t top) {
  Scale r;
  const bool finite = top < 0x7f800000u;
  r.s = finite ? __fmul_rn(__uint_as_float(top), 1.f / 127.f) : __uint_as_float(0x7fffffffu);
  r.small = r.s < 1.17549435e-38f;
  r.inverse = finite && r.s > 0.f ? __fdividef(1.f, r.small ? 1.f : r.s) : 0.f;
  return r;
}

// The code of one number, in the lowest byte.
__device__ __forceinline__ uint32_t code_of(float x, const Scale& k) {
  constexpr float M = 12582912.f;               // 1.5 x 2^23: what is added to it is rounded to a whole number, which its lowest bits then are
  if (k.inverse == 0.f) return 0u;
  const float q = x * k.inverse, m = q + M;
  if (!k.small && fabsf(q - (m - M)) <= 0.5f - 0x1p-10f) return __float_as_uint(m);
  return __float_as_uint(fminf(fmaxf(__fdiv_rn(x, k.s), -127.f), 127.f) + M);
}
// Four numbers' codes in a word.
__device__ __forceinline__ uint32_t codes_of(float a, float b, float c, float d, const Scale& k) {
  const uint32_t lo = __byte_perm(code_of(a, k), code_of(b, k), 0x0040), hi = __byte_perm(code_of(c, k), code_of(d, k), 0x0040);
  return __byte_perm(lo, hi, 0x5410);
}

}  // namespace kvad
