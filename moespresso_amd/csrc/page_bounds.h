// The 8-bit form of bounds and query codes: whole numbers of a power of two, so that scores are exact sums.
#pragma once
#include "common.h"

#include <initializer_list>
#include <type_traits>

constexpr int kBoundLimit = 50;  // exponents lie within +-50: a score, up to 2^24 times both powers, stays a float32

// The smallest e with top <= 127 * 2^e, within the limit (a largest magnitude of zero, or none: the lowest).
__device__ __forceinline__ int bound_exponent(float top) {
  if (!(top > 0.0f)) return -kBoundLimit;
  const float t = fminf(top, 3.4028234664e38f);
  const int e = __builtin_amdgcn_frexp_expf(t) - 7 + (__builtin_amdgcn_frexp_mantf(t) > 127.0f / 128.0f ? 1 : 0);
  return e < -kBoundLimit ? -kBoundLimit : e > kBoundLimit ? kBoundLimit : e;
}
__device__ __forceinline__ int bound_exponent(double top) {
  if (!(top > 0.0)) return -kBoundLimit;
  const double t = fmin(top, 1.7976931348623157e308);
  const int e = __builtin_amdgcn_frexp_exp(t) - 7 + (__builtin_amdgcn_frexp_mant(t) > 127.0 / 128.0 ? 1 : 0);
  return e < -kBoundLimit ? -kBoundLimit : e > kBoundLimit ? kBoundLimit : e;
}

// (the lowest value first: what a conversion makes of a NaN is held to the range too)
__device__ __forceinline__ int bound_code(float x) { return (int)fminf(fmaxf(x, -127.0f), 127.0f); }

constexpr int kBoundBytes = 512;  // of a page and KV head: 256 lower bounds, 256 upper ones
