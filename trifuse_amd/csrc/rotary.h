// Sine and cosine of rotary angles.
#pragma once

#include "tfm_device.h"

namespace tfm {

constexpr double kTurnsPerRadian = 0.15915494309189533577;  // 1 / (2 pi)

// scale * (cos, sin) of 2 pi * turns. Whole turns are taken off in 64 bits: a far position's
// angle has millions of them, of which fp32 keeps nothing. What is left, at most half a turn,
// is right to 2^-26 of one in fp32; less its quarters, |a| <= pi / 4, it takes the Taylor
// polynomials of degree 9 and 10 (next terms below 2e-9).
__device__ __forceinline__ float2 turn_cos_sin(double turns, float scale) {
  const float part = (float)(turns - __builtin_rint(turns));  // [-1/2, 1/2]
  const float quarter = __builtin_rintf(4.0f * part);
  const float a = (part - 0.25f * quarter) * 6.283185307179586f;
  const int q = (int)quarter;  // -2 .. 2
  const float z = a * a;
  float s = 2.7557319e-6f;
  s = __builtin_fmaf(s, z, -1.9841270e-4f);
  s = __builtin_fmaf(s, z, 8.3333333e-3f);
  s = __builtin_fmaf(s, z, -1.6666667e-1f);
  s = __builtin_fmaf(s * z, a, a);
  float c = -2.7557319e-7f;
  c = __builtin_fmaf(c, z, 2.4801587e-5f);
  c = __builtin_fmaf(c, z, -1.3888889e-3f);
  c = __builtin_fmaf(c, z, 4.1666667e-2f);
  c = __builtin_fmaf(c, z, -0.5f);
  c = __builtin_fmaf(c, z, 1.0f);
  // A quarter turn takes (cos, sin) to (-sin, cos).
  const float x = q & 1 ? s : c, y = q & 1 ? c : s;
  const bool nx = (q + 4) % 4 == 1 || (q + 4) % 4 == 2, ny = q < 0 || q == 2;
  return make_float2((nx ? -x : x) * scale, (ny ? -y : y) * scale);
}

}  // namespace tfm
