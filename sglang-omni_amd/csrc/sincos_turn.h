// The sine and cosine of the rotary kernels whose angles are float64.
#pragma once

#include "common.h"

// sin and cos of 2 pi turn, |turn| <= 1/8 after the quarter turns are taken off: |angle| <= pi / 4,
// where the terms past the 9th (10th) power are below 2^-29.
OMNI_DEVICE void sincos_turn(double turn, float* s, float* c) {
  const double quarters = __builtin_rint(turn * 4.0);
  const float a = (float)((turn - quarters * 0.25) * 6.283185307179586);
  const float a2 = a * a;
  float ps = 1.f / 362880.f;
  ps = __builtin_fmaf(ps, a2, -1.f / 5040.f);
  ps = __builtin_fmaf(ps, a2, 1.f / 120.f);
  ps = __builtin_fmaf(ps, a2, -1.f / 6.f);
  const float sn = __builtin_fmaf(ps * a2, a, a);
  float pc = -1.f / 3628800.f;
  pc = __builtin_fmaf(pc, a2, 1.f / 40320.f);
  pc = __builtin_fmaf(pc, a2, -1.f / 720.f);
  pc = __builtin_fmaf(pc, a2, 1.f / 24.f);
  pc = __builtin_fmaf(pc, a2, -0.5f);
  const float cs = __builtin_fmaf(pc, a2, 1.f);
  const int quadrant = (int)((long long)quarters & 3);
  const float s1 = quadrant & 1 ? cs : sn, c1 = quadrant & 1 ? sn : cs;
  *s = quadrant & 2 ? -s1 : s1;
  *c = quadrant == 1 || quadrant == 2 ? -c1 : c1;
}
