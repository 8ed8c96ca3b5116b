// The published affine 8-bit rule of a group of 64 elements (see kvquant.hip), shared by the kernels that write such rows.
// Float32, one operation per step: nothing here may be contracted.
#pragma once
#include "common.h"

// Scale and bias of a group from its smallest and largest element; the edge of larger magnitude is hit exactly.
__device__ __forceinline__ void affine_q8_scale(float mn, float mx, float& scale, float& bias) {
#pragma clang fp contract(off)
  scale = fmaxf((mx - mn) / 255.0f, 1e-7f);
  const bool side = fabsf(mn) > fabsf(mx);
  scale = side ? scale : -scale;
  const float edge = side ? mn : mx;
  const float q0 = rintf(edge / scale);
  const bool at_zero = q0 == 0.0f;
  scale = at_zero ? scale : edge / q0;
  bias = at_zero ? 0.0f : edge;
}

__device__ __forceinline__ uint32_t affine_q8_code(float v, float scale, float bias) {
#pragma clang fp contract(off)
  float c = rintf((v - bias) / scale);
  c = c < 255.0f ? c : 255.0f;
  c = c > 0.0f ? c : 0.0f;
  return (uint32_t)c;
}
