// The angle of a rotated pair: cos and sin of position * frequency.
#pragma once

#include <hip/hip_runtime.h>

namespace spyre_hip {

// The product is formed and reduced to an eighth of a turn in 64 bits (far
// positions: 32 bits keep only 2^-24 of an angle of thousands of turns); what
// is left, |x| <= pi/4, goes through the Taylor series in 32, whose first
// omitted terms are below 2^-29.
__device__ __forceinline__ void cos_sin_of(double position, double frequency, float& c, float& s) {
  constexpr double kQuartersPerRadian = 0.63661977236758134308;  // 2 / pi
  const double quarters = position * frequency * kQuartersPerRadian;
  const double whole = rint(quarters);
  const float x = static_cast<float>(quarters - whole) * 1.57079632679489661923f;
  // whole modulo 4, for any size: the remainder by 4 is exact
  const int turn = static_cast<int>(whole - 4.0 * floor(whole * 0.25));
  const float y = x * x;
  float sn = __builtin_fmaf(y, -1.f / 39916800.f, 1.f / 362880.f);
  sn = __builtin_fmaf(y, sn, -1.f / 5040.f);
  sn = __builtin_fmaf(y, sn, 1.f / 120.f);
  sn = __builtin_fmaf(y, sn, -1.f / 6.f);
  sn = __builtin_fmaf(x * y, sn, x);
  float cn = __builtin_fmaf(y, -1.f / 3628800.f, 1.f / 40320.f);
  cn = __builtin_fmaf(y, cn, -1.f / 720.f);
  cn = __builtin_fmaf(y, cn, 1.f / 24.f);
  cn = __builtin_fmaf(y, cn, -0.5f);
  cn = __builtin_fmaf(y, cn, 1.f);
  const float a = (turn & 1) ? sn : cn, b = (turn & 1) ? cn : sn;
  c = (turn == 1 || turn == 2) ? -a : a;
  s = turn >= 2 ? -b : b;
}

// (x1, x2) turned.  Every kernel rounds alike: the fused operations are
// explicit, and the empty asm keeps a conversion that follows from being fused
// into them.
__device__ __forceinline__ void turn_pair(const float x1, const float x2, float c, float s, float& y1, float& y2) {
  y1 = __builtin_fmaf(x1, c, -(x2 * s));
  y2 = __builtin_fmaf(x2, c, x1 * s);
  asm("" : "+v"(y1), "+v"(y2));
}

}  // namespace spyre_hip
