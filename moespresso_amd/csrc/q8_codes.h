// 8-bit codes to float16 operands, shared by the kernels that attend quantised rows.
#pragma once
#include "common.h"

constexpr int kFmtQ8_0 = 0;
constexpr int kFmtAffine = 1;

typedef __attribute__((ext_vector_type(2))) _Float16 h2_t;

__device__ __forceinline__ uint32_t h2_bits(h2_t v) { return __builtin_bit_cast(uint32_t, v); }
__device__ __forceinline__ h2_t bits_h2(uint32_t v) { return __builtin_bit_cast(h2_t, v); }

// Four codes of one 32-bit word to four float16 values (two packed registers), exact integers:
// byte b becomes the float16 with bits 0x6400 | b = 1024 + b, then the offset is taken off.
template <int FMT>
__device__ __forceinline__ void codes4_to_h(uint32_t w, h2_t& lo, h2_t& hi) {
  if constexpr (FMT == kFmtQ8_0) {
    w ^= 0x80808080u;  // int8 -> offset binary
    lo = bits_h2(__builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) - h2_t{(_Float16)1152.0f, (_Float16)1152.0f};
    hi = bits_h2(__builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) - h2_t{(_Float16)1152.0f, (_Float16)1152.0f};
  } else {
    lo = bits_h2(__builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) - h2_t{(_Float16)1024.0f, (_Float16)1024.0f};
    hi = bits_h2(__builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) - h2_t{(_Float16)1024.0f, (_Float16)1024.0f};
  }
}
