// What the kernels that attend the rows of a paged cache share: rows of a page as buffer windows, operands of the matrix
// instructions, scales of 8-bit rows, the output.
#pragma once
#include "common.h"
#include "q8_codes.h"

#include <utility>

namespace {

constexpr int kD = 256;
constexpr int kTileKeys = 32;
constexpr int kVPitch = kD * 2 + 16;  // bytes per key row of the V tile
constexpr int kVTileBytes = kTileKeys * kVPitch;
constexpr int kNonTemporal = 2;    // cache policy of loads that are used once

constexpr int kAffine = 3;  // page format beside MSPR_F16 and MSPR_BF16

// Sums of `v` over this lane and those before it, by data-parallel moves (six steps; a lane permute each would go through LDS).
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // row_shr 1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast 15, 31
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
  return v;
}

__device__ __forceinline__ int length_of(const int32_t* lens, int batch, int b, int cap) {
  const int len = b < batch ? lens[b] : 0;
  return len < 0 ? 0 : len > cap ? cap : len;
}

// Rows of a page as a buffer: what lies behind the ones that count reads as zero, and costs no memory access.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_window(const void* base, int64_t row, int row_bytes, int rows) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(reinterpret_cast<const uint8_t*>(base) + row * row_bytes), 0,
                                           rows * row_bytes, 0x00027000);
}
__device__ __forceinline__ u32x4_t window_load16(__amdgpu_buffer_rsrc_t w, int lane_offset, int offset) {
  return __builtin_amdgcn_raw_buffer_load_b128(w, lane_offset + (offset & 4095), offset & ~4095, kNonTemporal);
}

template <int FMT>
__device__ __forceinline__ f32x4_t mfma(u32x4_t a, u32x4_t b, f32x4_t c) {
  if constexpr (FMT == MSPR_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}

// Eight float32 values as terms of eight 16-bit operands each: x ~ t[0] + t[1], the second the rounded rest.
template <int FMT, int TERMS>
__device__ __forceinline__ void split_terms(const float* x, u32x4_t* t) {
  float rest[8];
#pragma unroll
  for (int i = 0; i < 8; i++) rest[i] = x[i];
#pragma unroll
  for (int k = 0; k < TERMS; k++) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
      if constexpr (FMT == MSPR_BF16) {
        const bf16x2_t h = {(__bf16)rest[2 * j], (__bf16)rest[2 * j + 1]};
        t[k][j] = __builtin_bit_cast(uint32_t, h);
        rest[2 * j] -= (float)h.x;
        rest[2 * j + 1] -= (float)h.y;
      } else {
        const h2_t h = {(_Float16)rest[2 * j], (_Float16)rest[2 * j + 1]};
        t[k][j] = h2_bits(h);
        rest[2 * j] -= (float)h.x;
        rest[2 * j + 1] -= (float)h.y;
      }
    }
  }
}

template <int DT>
__device__ __forceinline__ void widen8(u32x4_t w, float* x) {
#pragma unroll
  for (int j = 0; j < 4; j++) {
    if constexpr (DT == MSPR_F16) {
      x[2 * j] = f16_bits_to_f32((uint16_t)(w[j] & 0xFFFFu));
      x[2 * j + 1] = f16_bits_to_f32((uint16_t)(w[j] >> 16));
    } else {
      x[2 * j] = __uint_as_float(w[j] << 16);
      x[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
    }
  }
}

// Four affine codes less 128 (signed bytes, were their upper bits turned) to float16, exactly.
__device__ __forceinline__ void centred_to_h(uint32_t w, h2_t& lo, h2_t& hi) { codes4_to_h<kFmtQ8_0>(w ^ 0x80808080u, lo, hi); }

// One scale or bias a lane, number i of a window. 16-bit ones are loaded with their neighbour, a word: what is done to them
// behind the load (a load of 16 bits is masked) is done, and waited for, a tile too early.
template <int SDT>
struct RowScales {
  static constexpr int kBytes = SDT == MSPR_F32 ? 4 : 2;
  uint32_t word;
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t w, int i) {
    word = __builtin_amdgcn_raw_buffer_load_b32(w, i * kBytes & ~3, 0, kNonTemporal);
  }
  __device__ __forceinline__ float value(int i) const {
    if constexpr (SDT == MSPR_F32) return __uint_as_float(word);
    else if constexpr (SDT == MSPR_F16) return f16_bits_to_f32((uint16_t)(word >> (i & 1) * 16));
    else return __uint_as_float(word << (~i & 1) * 16 & 0xFFFF0000u);
  }
};

// The value of lane L of a row of sixteen in all of them (a data-parallel operand of the instruction that takes it).
template <int L>
__device__ __forceinline__ float of_lane(float v) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x150 + L, 0xF, 0xF, true));  // row_newbcast
}

// f(0), ..., f(N - 1) with the counter a constant (lane numbers of data-parallel operands are)
template <typename F, int... I>
__device__ __forceinline__ void static_for(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void static_for(F&& f) {
  static_for(f, std::make_integer_sequence<int, N>{});
}

// Output of one head's four channels, divided by its sum of weights.
template <int ODT>
__device__ __forceinline__ void store_out(void* out, int64_t i, f32x4_t o, float l) {
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  if constexpr (ODT == MSPR_F32) {
    *reinterpret_cast<f32x4_t*>(reinterpret_cast<float*>(out) + i) = o * inv;
  } else {
    uint16_t h[4];
#pragma unroll
    for (int j = 0; j < 4; j++) h[j] = ODT == MSPR_BF16 ? f32_to_bf16_bits(o[j] * inv) : f32_to_f16_bits(o[j] * inv);
    *reinterpret_cast<u32x2_t*>(reinterpret_cast<uint16_t*>(out) + i) =
        u32x2_t{(uint32_t)h[0] | ((uint32_t)h[1] << 16), (uint32_t)h[2] | ((uint32_t)h[3] << 16)};
  }
}

}  // namespace
