// Rotary positions with several axes:
//
//   angle(row, head, pair) = sum over axes a of position[row][a] frequency[a][head][pair]
//
// added in FP64 in the order of the axes (a product of two FP32 numbers is exact there),
// and its cosine and sine, each rounded to FP32 once. In FP32 the angle itself would be
// off by 2^-24 of it: 0.004 at position 65,536 of the fastest pair.
#pragma once

#include "focr_internal.hpp"

namespace focr {

constexpr int kMaxAxes = 4;

// {cos, sin} of an angle in FP64. With k the nearest whole number of quarter turns (the
// low bits of angle 2/pi + 1.5 2^52), r = angle - k pi/2 by two fused steps, pi/2 in two
// parts, so to about 2^-53; |r| <= pi/4, where the Taylor sums to r^15 and r^16 are off by
// less than 2^-53 too (the next terms: 5e-17 and 2e-18). Angles of 2^50 and more, an
// infinity and NaN give NaN.
__device__ __forceinline__ float2 cos_sin(double angle) {
  const double shift = 6755399441055744.0;  // 1.5 2^52
  const double t = __builtin_fma(angle, 0.63661977236758134308, shift);
  const double k = t - shift;
  const int quarter = static_cast<int>(__builtin_bit_cast(unsigned long long, t));
  double r = __builtin_fma(-k, 1.57079632679489661923, angle);
  r = __builtin_fma(-k, 6.123233995736765886e-17, r);
  const double z = r * r;
  double s = -1.0 / 1307674368000.0;
  s = __builtin_fma(s, z, 1.0 / 6227020800.0);
  s = __builtin_fma(s, z, -1.0 / 39916800.0);
  s = __builtin_fma(s, z, 1.0 / 362880.0);
  s = __builtin_fma(s, z, -1.0 / 5040.0);
  s = __builtin_fma(s, z, 1.0 / 120.0);
  s = __builtin_fma(s, z, -1.0 / 6.0);
  s = __builtin_fma(s * z, r, r);
  double c = 1.0 / 20922789888000.0;
  c = __builtin_fma(c, z, -1.0 / 87178291200.0);
  c = __builtin_fma(c, z, 1.0 / 479001600.0);
  c = __builtin_fma(c, z, -1.0 / 3628800.0);
  c = __builtin_fma(c, z, 1.0 / 40320.0);
  c = __builtin_fma(c, z, -1.0 / 720.0);
  c = __builtin_fma(c, z, 1.0 / 24.0);
  c = __builtin_fma(c, z, -0.5);
  c = __builtin_fma(c, z, 1.0);
  const uint32_t sine = __float_as_uint(static_cast<float>(s)), cosine = __float_as_uint(static_cast<float>(c));
  // A quarter turn: (cos, sin) to (-sin, cos).
  const uint32_t first = quarter & 1 ? sine : cosine, second = quarter & 1 ? cosine : sine;
  const float2 out = make_float2(__uint_as_float(first ^ ((quarter + 1) & 2) << 30), __uint_as_float(second ^ (quarter & 2) << 30));
  const bool fine = __builtin_fabs(angle) < 1125899906842624.0;
  return make_float2(fine ? out.x : __builtin_nanf(""), fine ? out.y : __builtin_nanf(""));
}

}  // namespace focr
