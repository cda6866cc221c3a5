// Rotary angles shared by the rotary kernel and the 4-bit cache's append.
#pragma once

#include "pg_common.h"

namespace pg {

// cos and sin of position * 2 pi * turns, times ``amplitude``.  The angle is
// formed in revolutions and reduced in 64 bits: at position 2^31 it is still
// within 2^-22 of a revolution, where 32 bits would have lost it (2^24
// positions at one turn each already are whole numbers there).  The reduced
// angle, at most half a turn, is rounded to 32 bits once (2^-25).  The fused
// operation is spelled out here and below, so that a row's bits do not depend on the
// kernel or the vector width that turns it.
__device__ __forceinline__ float2 rotary_cos_sin(int64_t position, double turns, float amplitude) {
  const double at = static_cast<double>(position);
  const float reduced = static_cast<float>(fma(at, turns, -rint(at * turns)));
  float s, c;
  sincospif(2.0f * reduced, &s, &c);
  return make_float2(c * amplitude, s * amplitude);
}

// (a, b) turned, in float32: the results are pinned, or the compiler would let some
// kernels round them and their conversion to FP16 in one step.
__device__ __forceinline__ float2 rotate_pair(float a, float b, float2 cos_sin) {
  float x = fmaf(a, cos_sin.x, -(b * cos_sin.y)), y = fmaf(b, cos_sin.x, a * cos_sin.y);
  asm("" : "+v"(x), "+v"(y));
  return make_float2(x, y);
}

}  // namespace pg
