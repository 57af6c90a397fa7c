// Rotary positions shared by the rotary kernel and the page pool's write.
#pragma once

#include "si_common.h"

namespace si {

// The rotation of a launch: pair i of a token at position p turns by
// p * freq[i] turns (a turn is 2 pi), its values are scaled by `gain`. sign -1
// rotates the other way (the transpose).
struct Rotation {
  const double* freq;  // [pairs], device
  const void* pos;     // int64 or int32
  int pos64;
  int pairs;
  int interleaved;     // pairs (2i, 2i+1), otherwise (i, i + pairs)
  double gain;
  double sign;
};

inline Rotation to_rotation(const si_rotation& r, const void* positions, int positions64, bool transpose) {
  return {r.freq, positions, positions64, (int)r.pairs, r.interleaved ? 1 : 0, r.gain, transpose ? -1.0 : 1.0};
}

// cos and sin of t turns, times gain. The argument is reduced in 64 bits (the
// integer part of t and then its nearest quarter are subtracted exactly), so
// position 10^6 is as exact as position 1; |x| <= pi/4 is left, where the Taylor
// sums to x^13 and x^14 are within 3e-14. One rounding to fp32 at the end.
__device__ __forceinline__ float2 turn_cos_sin(double t, double gain) {
  t -= rint(t);
  const double q = rint(4.0 * t);
  const double x = (t - 0.25 * q) * 6.283185307179586;
  const double z = x * x;
  double s = 1.6059043836821613e-10;                // 1/13!
  s = __builtin_fma(s, z, -2.505210838544172e-08);  // 1/11!
  s = __builtin_fma(s, z, 2.7557319223985893e-06);
  s = __builtin_fma(s, z, -1.984126984126984e-04);
  s = __builtin_fma(s, z, 8.333333333333333e-03);
  s = __builtin_fma(s, z, -1.6666666666666666e-01);
  s = __builtin_fma(s * z, x, x);
  double c = -1.1470745597729725e-11;               // 1/14!
  c = __builtin_fma(c, z, 2.08767569878681e-09);
  c = __builtin_fma(c, z, -2.755731922398589e-07);
  c = __builtin_fma(c, z, 2.48015873015873e-05);
  c = __builtin_fma(c, z, -1.388888888888889e-03);
  c = __builtin_fma(c, z, 4.1666666666666664e-02);
  c = __builtin_fma(c, z, -0.5);
  c = __builtin_fma(c, z, 1.0);
  const int k = (int)q & 3;
  const double co = k == 0 ? c : k == 1 ? -s : k == 2 ? -c : s;
  const double si = k == 0 ? s : k == 1 ? c : k == 2 ? -s : -c;
  return make_float2((float)(co * gain), (float)(si * gain));
}

// cos and sin of pair i for the token whose position is element n of r.pos.
__device__ __forceinline__ float2 pair_cos_sin(const Rotation& r, int64_t n, int i) {
  const double p = r.pos64 ? (double)reinterpret_cast<const int64_t*>(r.pos)[n]
                           : (double)reinterpret_cast<const int32_t*>(r.pos)[n];
  return turn_cos_sin(p * (r.sign * r.freq[i]), r.gain);
}

// The pair (a, b) turned, in fp32; each value is rounded to the row's type once
// by the caller.
__device__ __forceinline__ void rotate_pair(float2 cs, float& a, float& b) {
  const float x = a, y = b;
  a = __builtin_fmaf(-y, cs.y, x * cs.x);
  b = __builtin_fmaf(x, cs.y, y * cs.x);
}

}  // namespace si
