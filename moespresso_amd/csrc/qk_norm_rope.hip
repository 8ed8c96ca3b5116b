// Norm of every query and key head with the rotary position in the same pass, and the append of keys and values to a paged cache.
//
//   y = x * rsqrt(mean(x^2) + eps) * weight          over the 256 channels of a head, in float32
//   (y_i, y_{i+r/2}) <- (y_i cos t - y_{i+r/2} sin t, y_{i+r/2} cos t + y_i sin t)   for i < r/2, t = position * inv_freq_i
//
// rounded once, to the type of what is written. With three position axes frequency i takes axis i % 3 while that axis has
// frequencies left (axis 1: 3 i' + 1 < 3 n_1, axis 2: 3 i' + 2 < 3 n_2), else axis 0. The angle is the exact product, reduced to
// a turn in 64 bits: a float32 product is off by 2^-24 of it, 0.007 radians at position 120000, which no later step makes good.
//
// Bound by HBM: every element is read and written once. Half a wave owns a head's row (a lane eight neighbouring channels,
// so that a 16-bit row is one 16-byte load a lane), the sum of squares is five lane exchanges, the partner of a channel
// eight more. The cosines and sines of a workgroup's tokens are made once, a thread each, and shared through LDS.
#include "affine_q8.h"
#include "common.h"

namespace {

constexpr int kD = 256;
constexpr int kThreads = 256;
constexpr int kRowLanes = 32;
constexpr int kRowsAtOnce = kThreads / kRowLanes;
constexpr int kMaxTokens = 8;  // tokens a workgroup
constexpr int kMaxHalf = kD / 2;

// what becomes of keys and values
constexpr int kDense = 0;  // keys to a dense tensor of their type, no values
constexpr int kPages = 1;  // both to pages of 16-bit rows
constexpr int kCodes = 2;  // both to pages of affine 8-bit rows

struct RopeArgs {
  const void *q, *k, *v;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head;  // strides in elements
  const void *q_weight, *k_weight;
  const int32_t* positions;  // [axes][n_tokens]
  const float* inv_freq;
  const int32_t* slots;
  int n_tokens, n_q, n_kv, half, axes, sec1, sec2;
  int tokens_per_wg, rows_per_wg;
  uint32_t rows_inverse;  // of the rows of a token that a workgroup takes
  float eps;
  int page_shift, n_pages;
  void *q_out, *k_out;      // dense [n_tokens][heads][256]; k_out: pages in the paged forms
  void* v_out;              // pages
  void *k_scales, *k_biases, *v_scales, *v_biases;
};

template <int DT>
__device__ __forceinline__ void load8(const void* p, int64_t i, float* x) {
  if constexpr (DT == MSPR_F32) {
    const f32x4_t* s = reinterpret_cast<const f32x4_t*>(reinterpret_cast<const float*>(p) + i);
    const f32x4_t a = s[0], b = s[1];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      x[j] = a[j];
      x[4 + j] = b[j];
    }
  } else {
    const u32x4_t w = *reinterpret_cast<const u32x4_t*>(reinterpret_cast<const uint16_t*>(p) + i);
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
}

template <int DT>
__device__ __forceinline__ uint16_t bits16(float v) {
  if constexpr (DT == MSPR_F16) return f32_to_f16_bits(v);
  else return f32_to_bf16_bits(v);
}

template <int DT>
__device__ __forceinline__ float rounded(float v) {
  if constexpr (DT == MSPR_F32) return v;
  else if constexpr (DT == MSPR_F16) return f16_bits_to_f32(f32_to_f16_bits(v));
  else return bf16_bits_to_f32(f32_to_bf16_bits(v));
}

template <int DT>
__device__ __forceinline__ void store8(void* p, int64_t i, const float* x) {
  if constexpr (DT == MSPR_F32) {
    f32x4_t* d = reinterpret_cast<f32x4_t*>(reinterpret_cast<float*>(p) + i);
    d[0] = f32x4_t{x[0], x[1], x[2], x[3]};
    d[1] = f32x4_t{x[4], x[5], x[6], x[7]};
  } else {
    u32x4_t w;
#pragma unroll
    for (int j = 0; j < 4; j++) w[j] = (uint32_t)bits16<DT>(x[2 * j]) | ((uint32_t)bits16<DT>(x[2 * j + 1]) << 16);
    *reinterpret_cast<u32x4_t*>(reinterpret_cast<uint16_t*>(p) + i) = w;
  }
}

template <int DT>
__device__ __forceinline__ void store1(void* p, int64_t i, float v) {
  if constexpr (DT == MSPR_F32) reinterpret_cast<float*>(p)[i] = v;
  else reinterpret_cast<uint16_t*>(p)[i] = bits16<DT>(v);
}

// A row to its page: 16-bit channels, or codes with a scale and bias of the row's type per 64 channels (eight lanes).
template <int DT, int KEEP, int PT>
__device__ __forceinline__ void keep_row(void* out, void* scales, void* biases, int64_t row, int lane, const float* y) {
  if constexpr (KEEP == kPages) {
    store8<PT>(out, row * kD + 8 * lane, y);
  } else {
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] = rounded<DT>(y[j]);  // (codes of the row as a dense tensor of its type would hold it)
    float mn = x[0], mx = x[0];
#pragma unroll
    for (int j = 1; j < 8; j++) {
      mn = fminf(mn, x[j]);
      mx = fmaxf(mx, x[j]);
    }
    mn = fminf(mn, lane_xor<1>(mn));
    mx = fmaxf(mx, lane_xor<1>(mx));
    mn = fminf(mn, lane_xor<2>(mn));
    mx = fmaxf(mx, lane_xor<2>(mx));
    mn = fminf(mn, lane_xor<4>(mn));
    mx = fmaxf(mx, lane_xor<4>(mx));
    float scale, bias;
    affine_q8_scale(mn, mx, scale, bias);
    u32x2_t w = {0u, 0u};
#pragma unroll
    for (int j = 0; j < 4; j++) {
      w.x |= affine_q8_code(x[j], scale, bias) << (8 * j);
      w.y |= affine_q8_code(x[4 + j], scale, bias) << (8 * j);
    }
    reinterpret_cast<u32x2_t*>(out)[row * (kD / 8) + lane] = w;
    if ((lane & 7) == 0) {
      store1<DT>(scales, row * (kD / 64) + (lane >> 3), scale);
      store1<DT>(biases, row * (kD / 64) + (lane >> 3), bias);
    }
  }
}

// grid: (tokens / tokens_per_wg, rows of a token / rows_per_wg); a token's rows are its query heads, its key heads and, where
// they are kept, its value heads
template <int DT, int KEEP, int PT>
__global__ __launch_bounds__(kThreads) void qk_norm_rope_kernel(RopeArgs a) {
  __shared__ f32x2_t turn[kMaxTokens * kMaxHalf];  // cosine and sine
  const int tid = threadIdx.x;
  const int lane = tid & (kRowLanes - 1);
  const int t0 = blockIdx.x * a.tokens_per_wg;
  const int tokens = min(a.tokens_per_wg, a.n_tokens - t0);
  const int row0 = blockIdx.y * a.rows_per_wg;
  const int all_rows = a.n_q + (KEEP == kDense ? 1 : 2) * a.n_kv;

  for (int i = tid; i < tokens * a.half; i += kThreads) {
    const int t = i / a.half;
    const int f = i - t * a.half;
    const int m = f % 3;
    const int axis = a.axes == 1 ? 0 : m == 1 && f < 3 * a.sec1 ? 1 : m == 2 && f < 3 * a.sec2 ? 2 : 0;
    const int pos = a.positions[(int64_t)axis * a.n_tokens + t0 + t];
    double turns = (double)pos * (double)a.inv_freq[f] * 0.15915494309189535;  // 1 / (2 pi)
    turns -= rint(turns);
    float s, c;
    sincospif(2.0f * (float)turns, &s, &c);
    turn[i] = f32x2_t{c, s};
  }
  __syncthreads();

  const int span = a.half / 8;  // lanes of half the rotary width
  const bool low = lane < span, rotary = lane < 2 * span;
  const int partner = low ? lane + span : lane - span;
  for (int item = tid / kRowLanes; item < tokens * a.rows_per_wg; item += kRowsAtOnce) {
    const int t = mspr_div(item, a.rows_per_wg, a.rows_inverse);
    const int row = row0 + item - t * a.rows_per_wg;
    if (row >= all_rows) continue;
    const int64_t token = t0 + t;
    const bool is_q = row < a.n_q;
    const bool is_v = KEEP != kDense && row >= a.n_q + a.n_kv;
    const int head = is_q ? row : is_v ? row - a.n_q - a.n_kv : row - a.n_q;
    int64_t at = 0;  // row in the pages
    if constexpr (KEEP != kDense) {
      if (!is_q) {
        const int slot = a.slots[token];
        const int page = slot >> a.page_shift;
        if (slot < 0 || page >= a.n_pages) continue;
        at = (((int64_t)page * a.n_kv + head) << a.page_shift) + (slot & ((1 << a.page_shift) - 1));
      }
    }
    float x[8];
    if (is_v) {
      load8<DT>(a.v, token * a.v_token + head * a.v_head + 8 * lane, x);
      if constexpr (KEEP != kDense) keep_row<DT, KEEP, PT>(a.v_out, a.v_scales, a.v_biases, at, lane, x);
      continue;
    }
    load8<DT>(is_q ? a.q : a.k, is_q ? token * a.q_token + head * a.q_head + 8 * lane : token * a.k_token + head * a.k_head + 8 * lane, x);
    float w[8];
    load8<DT>(is_q ? a.q_weight : a.k_weight, 8 * lane, w);
    float ss = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; j++) ss += x[j] * x[j];
    ss += lane_xor<1>(ss);
    ss += lane_xor<2>(ss);
    ss += lane_xor<4>(ss);
    ss += lane_xor<8>(ss);
    ss += lane_xor<16>(ss);
    const float r = 1.0f / sqrtf(ss * (1.0f / kD) + a.eps);
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] = x[j] * r * w[j];
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const float other = __shfl(x[j], partner, kRowLanes);
      if (rotary) {
        const f32x2_t cs = turn[t * a.half + 8 * (low ? lane : partner) + j];
        x[j] = x[j] * cs.x + (low ? -other : other) * cs.y;
      }
    }
    if (is_q) {
      store8<DT>(a.q_out, (token * a.n_q + head) * kD + 8 * lane, x);
    } else if constexpr (KEEP == kDense) {
      store8<DT>(a.k_out, (token * a.n_kv + head) * kD + 8 * lane, x);
    } else {
      keep_row<DT, KEEP, PT>(a.k_out, a.k_scales, a.k_biases, at, lane, x);
    }
  }
}

template <int DT, int KEEP, int PT>
int rope_launch(RopeArgs a, hipStream_t st) {
  const int rows = a.n_q + (KEEP == kDense ? 1 : 2) * a.n_kv;
  // eight tokens a workgroup share the angles' cost; few tokens are spread a pass of rows a workgroup, for latency
  a.tokens_per_wg = a.n_tokens >= 2048 ? kMaxTokens : 1;
  a.rows_per_wg = a.n_tokens >= 256 ? rows : kRowsAtOnce;
  a.rows_inverse = mspr_inverse(a.rows_per_wg);
  const dim3 grid((unsigned)((a.n_tokens + a.tokens_per_wg - 1) / a.tokens_per_wg),
                  (unsigned)((rows + a.rows_per_wg - 1) / a.rows_per_wg));
  qk_norm_rope_kernel<DT, KEEP, PT><<<grid, dim3(kThreads), 0, st>>>(a);
  MSPR_CHECK_LAUNCH("qk_norm_rope");
  return MSPR_OK;
}

int rope_checks(const char* what, const RopeArgs& a, int dtype, int head_dim) {
  MSPR_REQUIRE(a.q && a.k && a.q_weight && a.k_weight && a.positions && a.inv_freq && a.q_out && a.k_out, "%s: null pointer", what);
  MSPR_REQUIRE(dtype >= MSPR_F32 && dtype <= MSPR_BF16, "%s: dtype must be f32, f16 or bf16", what);
  MSPR_REQUIRE(head_dim == kD, "%s: head_dim must be 256", what);
  MSPR_REQUIRE(a.n_tokens >= 1 && a.n_tokens <= (1 << 24), "%s: 1 to 2^24 tokens", what);
  MSPR_REQUIRE(a.n_q >= 1 && a.n_kv >= 1 && a.n_q <= 1024 && a.n_kv <= 1024, "%s: 1 to 1024 heads of each kind", what);
  MSPR_REQUIRE(a.half >= 8 && a.half <= kMaxHalf && a.half % 8 == 0, "%s: the rotary width must be a multiple of 16 up to 256", what);
  MSPR_REQUIRE(a.axes == 1 || a.axes == 3, "%s: positions have one axis or three", what);
  MSPR_REQUIRE(a.axes == 1 || (a.sec1 >= 0 && a.sec2 >= 0 && 3 * a.sec1 <= a.half + 1 && 3 * a.sec2 <= a.half),
               "%s: the height and width axes have more frequencies than their turns", what);
  const int64_t unit = dtype == MSPR_F32 ? 4 : 8;
  MSPR_REQUIRE(a.q_token % unit == 0 && a.q_head % unit == 0 && a.k_token % unit == 0 && a.k_head % unit == 0 &&
                   a.v_token % unit == 0 && a.v_head % unit == 0 && mspr_aligned(a.q, 16) && mspr_aligned(a.k, 16) &&
                   mspr_aligned(a.v, 16) && mspr_aligned(a.q_weight, 16) && mspr_aligned(a.k_weight, 16) &&
                   mspr_aligned(a.q_out, 16) && mspr_aligned(a.k_out, 16) && mspr_aligned(a.v_out, 16),
               "%s: rows must be 16-byte aligned", what);
  return MSPR_OK;
}

RopeArgs rope_args(const void* q, const void* k, const void* q_weight, const void* k_weight, int n_tokens, int n_q_heads,
                   int n_kv_heads, const int64_t* strides, const int32_t* positions, int axes, int sec1, int sec2,
                   const float* inv_freq, int rotary_dim, float eps, void* q_out) {
  RopeArgs a{};
  a.q = q;
  a.k = k;
  a.q_token = strides[0];
  a.q_head = strides[1];
  a.k_token = strides[2];
  a.k_head = strides[3];
  a.q_weight = q_weight;
  a.k_weight = k_weight;
  a.positions = positions;
  a.inv_freq = inv_freq;
  a.n_tokens = n_tokens;
  a.n_q = n_q_heads;
  a.n_kv = n_kv_heads;
  a.half = rotary_dim / 2;
  a.axes = axes;
  a.sec1 = sec1;
  a.sec2 = sec2;
  a.eps = eps;
  a.q_out = q_out;
  return a;
}

int append_checks(const char* what, const RopeArgs& a, int page_size) {
  MSPR_REQUIRE(a.v && a.slots && a.v_out, "%s: null pointer", what);
  MSPR_REQUIRE(page_size >= 16 && (page_size & (page_size - 1)) == 0, "%s: page_size must be a power of two from 16 on", what);
  MSPR_REQUIRE(a.n_pages >= 1 && (int64_t)a.n_pages * page_size <= 0x7FFFFFFF, "%s: the pool must hold fewer than 2^31 tokens", what);
  return MSPR_OK;
}

}  // namespace

extern "C" int mspr_qk_norm_rope(const void* q, const void* k, const void* q_weight, const void* k_weight, int dtype, int n_tokens,
                                 int n_q_heads, int n_kv_heads, int head_dim, int64_t q_token_stride, int64_t q_head_stride,
                                 int64_t k_token_stride, int64_t k_head_stride, const int32_t* positions, int axes,
                                 int height_freqs, int width_freqs, const float* inv_freq, int rotary_dim, float eps,
                                 void* q_out, void* k_out, void* stream) {
  const int64_t strides[4] = {q_token_stride, q_head_stride, k_token_stride, k_head_stride};
  RopeArgs a = rope_args(q, k, q_weight, k_weight, n_tokens, n_q_heads, n_kv_heads, strides, positions, axes, height_freqs,
                         width_freqs, inv_freq, rotary_dim, eps, q_out);
  a.k_out = k_out;
  MSPR_REQUIRE(rotary_dim % 2 == 0, "qk_norm_rope: the rotary width must be a multiple of 16 up to 256");
  if (int rc = rope_checks("qk_norm_rope", a, dtype, head_dim)) return rc;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == MSPR_F32) return rope_launch<MSPR_F32, kDense, MSPR_F32>(a, st);
  if (dtype == MSPR_F16) return rope_launch<MSPR_F16, kDense, MSPR_F16>(a, st);
  return rope_launch<MSPR_BF16, kDense, MSPR_BF16>(a, st);
}

extern "C" int mspr_qk_norm_rope_append(const void* q, const void* k, const void* v, const void* q_weight, const void* k_weight,
                                        int dtype, int n_tokens, int n_q_heads, int n_kv_heads, int head_dim,
                                        const int64_t* strides, const int32_t* positions, int axes, int height_freqs,
                                        int width_freqs, const float* inv_freq, int rotary_dim, float eps, const int32_t* slots,
                                        int n_pages, int page_size, int page_dtype, void* k_pages, void* v_pages, void* q_out,
                                        void* stream) {
  MSPR_REQUIRE(strides, "qk_norm_rope_append: null pointer");
  RopeArgs a = rope_args(q, k, q_weight, k_weight, n_tokens, n_q_heads, n_kv_heads, strides, positions, axes, height_freqs,
                         width_freqs, inv_freq, rotary_dim, eps, q_out);
  a.v = v;
  a.v_token = strides[4];
  a.v_head = strides[5];
  a.k_out = k_pages;
  a.v_out = v_pages;
  a.slots = slots;
  a.n_pages = n_pages;
  MSPR_REQUIRE(rotary_dim % 2 == 0, "qk_norm_rope_append: the rotary width must be a multiple of 16 up to 256");
  if (int rc = rope_checks("qk_norm_rope_append", a, dtype, head_dim)) return rc;
  if (int rc = append_checks("qk_norm_rope_append", a, page_size)) return rc;
  MSPR_REQUIRE((page_dtype == MSPR_F16 || page_dtype == MSPR_BF16) && (dtype == MSPR_F32 || page_dtype == dtype),
               "qk_norm_rope_append: pages must be of the rows' 16-bit type, or of either for float32 rows");
  a.page_shift = __builtin_ctz(page_size);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == MSPR_F16) return rope_launch<MSPR_F16, kPages, MSPR_F16>(a, st);
  if (dtype == MSPR_BF16) return rope_launch<MSPR_BF16, kPages, MSPR_BF16>(a, st);
  if (page_dtype == MSPR_F16) return rope_launch<MSPR_F32, kPages, MSPR_F16>(a, st);
  return rope_launch<MSPR_F32, kPages, MSPR_BF16>(a, st);
}

extern "C" int mspr_qk_norm_rope_append_q8(const void* q, const void* k, const void* v, const void* q_weight,
                                           const void* k_weight, int dtype, int n_tokens, int n_q_heads, int n_kv_heads,
                                           int head_dim, const int64_t* strides, const int32_t* positions, int axes,
                                           int height_freqs, int width_freqs, const float* inv_freq, int rotary_dim, float eps,
                                           const int32_t* slots, int n_pages, int page_size, void* k_wq, void* k_scales,
                                           void* k_biases, void* v_wq, void* v_scales, void* v_biases, void* q_out,
                                           void* stream) {
  MSPR_REQUIRE(strides && k_scales && k_biases && v_scales && v_biases, "qk_norm_rope_append_q8: null pointer");
  RopeArgs a = rope_args(q, k, q_weight, k_weight, n_tokens, n_q_heads, n_kv_heads, strides, positions, axes, height_freqs,
                         width_freqs, inv_freq, rotary_dim, eps, q_out);
  a.v = v;
  a.v_token = strides[4];
  a.v_head = strides[5];
  a.k_out = k_wq;
  a.v_out = v_wq;
  a.k_scales = k_scales;
  a.k_biases = k_biases;
  a.v_scales = v_scales;
  a.v_biases = v_biases;
  a.slots = slots;
  a.n_pages = n_pages;
  MSPR_REQUIRE(rotary_dim % 2 == 0, "qk_norm_rope_append_q8: the rotary width must be a multiple of 16 up to 256");
  if (int rc = rope_checks("qk_norm_rope_append_q8", a, dtype, head_dim)) return rc;
  if (int rc = append_checks("qk_norm_rope_append_q8", a, page_size)) return rc;
  a.page_shift = __builtin_ctz(page_size);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == MSPR_F32) return rope_launch<MSPR_F32, kCodes, MSPR_F32>(a, st);
  if (dtype == MSPR_F16) return rope_launch<MSPR_F16, kCodes, MSPR_F16>(a, st);
  return rope_launch<MSPR_BF16, kCodes, MSPR_BF16>(a, st);
}
