// Norm of every query and key head with the rotary position in the same pass, and the append of keys and values to a paged cache.
//
//   y = x * rsqrt(mean(x^2) + eps) * weight          over the 256 channels of a head, in float32
//   (y_i, y_{i+r/2}) <- (y_i cos t - y_{i+r/2} sin t, y_{i+r/2} cos t + y_i sin t)   for i < r/2, t = position * inv_freq_i
//
// rounded once, to the type of what is written. With three position axes frequency i takes axis i % 3 while that axis has
// frequencies left (axis 1: 3 i' + 1 < 3 n_1, axis 2: 3 i' + 2 < 3 n_2), else axis 0. The angle is the product in 64 bits, reduced
// to a turn there: a float32 product is off by 2^-24 of it, 0.007 radians at position 120000, which no later step makes good.
//
// Bound by HBM: every element is read and written once. A lane owns 16 bytes of a head's row, so that a load or store of a wave
// is whole rows (with 32 bytes of a float32 row a lane, every line was asked for twice), the sum of squares is five or six lane
// exchanges, the partner of a channel one more. A wave takes neighbouring heads of one kind, so that whose row it is and where
// it lies is scalar arithmetic, and asks for its next rows before it works on these. Loads are non-temporal, as nothing reads
// the projections' output again (16384 tokens of bfloat16 rows, appended: the kernel alone 56 us, 6.0 TB/s, instead of 67; calls
// behind each other, of which each finds the last one's writes still under way, 71 us, 4.7 TB/s). The cosines and sines of a
// workgroup's tokens are made once, a thread each, under the first rows' loads, and shared through LDS.
#include "affine_q8.h"
#include "common.h"

namespace {

constexpr int kD = 256;
constexpr int kThreads = 256;
// a lane's channels of a row, the lanes of a row, the rows of a wave
template <int DT>
constexpr int kChannels = DT == MSPR_F32 ? 4 : 8;
template <int DT>
constexpr int kRowLanes = kD / kChannels<DT>;
template <int DT>
constexpr int kRows = MSPR_WAVE / kRowLanes<DT>;
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
  int tokens_per_wg, groups_per_wg;
  float eps;
  int page_shift, n_pages;
  void *q_out, *k_out;      // dense [n_tokens][heads][256]; k_out: pages in the paged forms
  void* v_out;              // pages
  void *k_scales, *k_biases, *v_scales, *v_biases;
};

// A lane's channels as they lie in memory.
template <int DT>
struct Raw {
  u32x4_t w;
  __device__ __forceinline__ void load(const void* p, int64_t i) {
    w = __builtin_nontemporal_load(
        reinterpret_cast<const u32x4_t*>(reinterpret_cast<const uint8_t*>(p) + i * (DT == MSPR_F32 ? 4 : 2)));
  }
  __device__ __forceinline__ void widen(float* x) const {
#pragma unroll
    for (int j = 0; j < 4; j++) {
      if constexpr (DT == MSPR_F32) {
        x[j] = __uint_as_float(w[j]);
      } else if constexpr (DT == MSPR_F16) {
        x[2 * j] = f16_bits_to_f32((uint16_t)(w[j] & 0xFFFFu));
        x[2 * j + 1] = f16_bits_to_f32((uint16_t)(w[j] >> 16));
      } else {
        x[2 * j] = __uint_as_float(w[j] << 16);
        x[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
      }
    }
  }
};

template <int DT>
__device__ __forceinline__ uint16_t bits16(float v) {
  if constexpr (DT == MSPR_F16) return f32_to_f16_bits(v);
  else return __builtin_bit_cast(uint16_t, (__bf16)v);
}

template <int DT>
__device__ __forceinline__ uint32_t pair16(float a, float b) {
  if constexpr (DT == MSPR_BF16) return __builtin_bit_cast(uint32_t, bf16x2_t{(__bf16)a, (__bf16)b});  // one instruction
  else return (uint32_t)bits16<DT>(a) | ((uint32_t)bits16<DT>(b) << 16);
}

template <int DT>
__device__ __forceinline__ float rounded(float v) {
  if constexpr (DT == MSPR_F32) return v;
  else if constexpr (DT == MSPR_F16) return f16_bits_to_f32(f32_to_f16_bits(v));
  else return (float)(__bf16)v;
}

// 1 / sqrt(v), off by little more than half a unit of its last place: the instruction's value, a unit off at most, and one step
// of Newton's method with the rounding of v * y in it. The instruction takes numbers below 2^-126 for zero: they are scaled.
__device__ __forceinline__ float rsqrt_near(float v) {
  const bool tiny = v < 0x1p-96f;
  const float u = tiny ? v * 0x1p64f : v;
  const float y = __builtin_amdgcn_rsqf(u);
  const float h = u * y;
  const float e = fmaf(-y, fmaf(u, y, -h), fmaf(-h, y, 1.0f));  // 1 - u y^2
  const float z = u > 0.0f && u < __builtin_inff() ? fmaf(0.5f * y, e, y) : y;
  return tiny ? z * 0x1p32f : z;
}

// N channels of type DT.
template <int DT, int N>
__device__ __forceinline__ void store_row(void* p, int64_t i, const float* x) {
  if constexpr (DT == MSPR_F32) {
    static_assert(N == 4, "16 bytes");
    *reinterpret_cast<f32x4_t*>(reinterpret_cast<float*>(p) + i) = f32x4_t{x[0], x[1], x[2], x[3]};
  } else if constexpr (N == 4) {
    *reinterpret_cast<u32x2_t*>(reinterpret_cast<uint16_t*>(p) + i) = u32x2_t{pair16<DT>(x[0], x[1]), pair16<DT>(x[2], x[3])};
  } else {
    u32x4_t w;
#pragma unroll
    for (int j = 0; j < 4; j++) w[j] = pair16<DT>(x[2 * j], x[2 * j + 1]);
    *reinterpret_cast<u32x4_t*>(reinterpret_cast<uint16_t*>(p) + i) = w;
  }
}

template <int DT>
__device__ __forceinline__ void store1(void* p, int64_t i, float v) {
  if constexpr (DT == MSPR_F32) reinterpret_cast<float*>(p)[i] = v;
  else reinterpret_cast<uint16_t*>(p)[i] = bits16<DT>(v);
}

// A row to its page: 16-bit channels, or codes with a scale and bias of the row's type per 64 channels.
template <int DT, int KEEP, int PT>
__device__ __forceinline__ void keep_row(void* out, void* scales, void* biases, int64_t row, int lane, const float* y) {
  constexpr int N = kChannels<DT>;
  if constexpr (KEEP == kPages) {
    store_row<PT, N>(out, row * kD + N * lane, y);
  } else {
    float x[N];
#pragma unroll
    for (int j = 0; j < N; j++) x[j] = rounded<DT>(y[j]);  // (codes of the row as a dense tensor of its type would hold it)
    float mn = x[0], mx = x[0];
#pragma unroll
    for (int j = 1; j < N; j++) {
      mn = fminf(mn, x[j]);
      mx = fmaxf(mx, x[j]);
    }
    mn = fminf(mn, lane_xor<1>(mn));
    mx = fmaxf(mx, lane_xor<1>(mx));
    mn = fminf(mn, lane_xor<2>(mn));
    mx = fmaxf(mx, lane_xor<2>(mx));
    mn = fminf(mn, lane_xor<4>(mn));
    mx = fmaxf(mx, lane_xor<4>(mx));
    if constexpr (N == 4) {
      mn = fminf(mn, lane_xor<8>(mn));
      mx = fmaxf(mx, lane_xor<8>(mx));
    }
    float scale, bias;
    affine_q8_scale(mn, mx, scale, bias);
    uint32_t w[N / 4];
#pragma unroll
    for (int k = 0; k < N / 4; k++) {
      w[k] = 0;
#pragma unroll
      for (int j = 0; j < 4; j++) w[k] |= affine_q8_code(x[4 * k + j], scale, bias) << (8 * j);
    }
    uint32_t* codes = reinterpret_cast<uint32_t*>(out) + row * (kD / 4) + lane * (N / 4);
    if constexpr (N == 8) *reinterpret_cast<u32x2_t*>(codes) = u32x2_t{w[0], w[1]};
    else *codes = w[0];
    if (lane % (64 / N) == 0) {
      store1<DT>(scales, row * (kD / 64) + lane / (64 / N), scale);
      store1<DT>(biases, row * (kD / 64) + lane / (64 / N), bias);
    }
  }
}

// grid: (tokens / tokens_per_wg, groups of a token / groups_per_wg); a token's groups are a wave's rows each of its query heads,
// its key heads and, where they are kept, its value heads (a kind whose heads are not a multiple of them ends with part of one)
template <int DT, int KEEP, int PT>
__global__ __launch_bounds__(kThreads) void qk_norm_rope_kernel(RopeArgs a) {
  constexpr int N = kChannels<DT>, R = kRows<DT>;
  __shared__ __attribute__((aligned(16))) f32x2_t turn[kMaxTokens * 2 * kMaxHalf];  // [token][lower, upper half][cosine, sine]
  const int tid = threadIdx.x;
  const int lane = tid % kRowLanes<DT>;
  const int mine = tid % MSPR_WAVE / kRowLanes<DT>;  // row of the group
  const int wave = __builtin_amdgcn_readfirstlane(tid / MSPR_WAVE);
  const int t0 = blockIdx.x * a.tokens_per_wg;
  const int tokens = min(a.tokens_per_wg, a.n_tokens - t0);
  const int q_groups = (a.n_q + R - 1) / R, kv_groups = (a.n_kv + R - 1) / R;
  const int group0 = blockIdx.y * a.groups_per_wg;
  const int groups = min(a.groups_per_wg, q_groups + (KEEP == kDense ? 1 : 2) * kv_groups - group0);

  const int64_t q_lane = mine * a.q_head + N * lane, k_lane = mine * a.k_head + N * lane, v_lane = mine * a.v_head + N * lane;
  // A wave's items are those of number wave, wave + 4, ... in the order token by token.
  struct Item {
    int t, group;
  };
  auto next = [&](Item& i, int by) {
    i.group += by;
    while (i.group >= groups) {
      i.group -= groups;
      i.t++;
    }
  };
  auto load = [&](const Item& i, Raw<DT>& raw) {
    const int64_t token = t0 + i.t;
    const int group = group0 + i.group;
    if (group < q_groups) {
      if (R * group + mine < a.n_q) raw.load(a.q, token * a.q_token + R * group * a.q_head + q_lane);
    } else if (group < q_groups + kv_groups) {
      const int head = R * (group - q_groups);
      if (head + mine < a.n_kv) raw.load(a.k, token * a.k_token + head * a.k_head + k_lane);
    } else if constexpr (KEEP != kDense) {
      const int head = R * (group - q_groups - kv_groups);
      if (head + mine < a.n_kv) raw.load(a.v, token * a.v_token + head * a.v_head + v_lane);
    }
  };
  Item item = {0, 0};
  next(item, wave);
  Raw<DT> raw, qw, kw;
  if (item.t < tokens) load(item, raw);
  qw.load(a.q_weight, N * lane);
  kw.load(a.k_weight, N * lane);

  for (int i = tid; i < tokens * a.half; i += kThreads) {
    const int t = i / a.half;
    const int f = i - t * a.half;
    const int m = f % 3;
    const int axis = a.axes == 1 ? 0 : m == 1 && f < 3 * a.sec1 ? 1 : m == 2 && f < 3 * a.sec2 ? 2 : 0;
    const int pos = a.positions[(int64_t)axis * a.n_tokens + t0 + t];
    double turns = (double)pos * (double)a.inv_freq[f] * 0.15915494309189535;  // 1 / (2 pi)
    turns -= rint(turns);
    const float near = (float)turns;  // (2 pi of what that rounds off, up to 9e-8, is added to the angle to first order)
    const float rest = (float)(turns - (double)near) * 6.2831853f;
    float s, c;
    sincospif(2.0f * near, &s, &c);
    const float c0 = c;
    c = fmaf(-s, rest, c);
    s = fmaf(c0, rest, s);
    turn[2 * t * a.half + f] = f32x2_t{c, -s};
    turn[(2 * t + 1) * a.half + f] = f32x2_t{c, s};
  }
  __syncthreads();

  const int span = a.half / N;  // lanes of half the rotary width
  const bool low = lane < span, rotary = lane < 2 * span;
  const int partner = low ? lane + span : lane - span;
  auto process = [&](const Item& here, const Raw<DT>& raw) {
    const int64_t token = t0 + here.t;
    const int group = group0 + here.group;
    const bool is_q = group < q_groups;
    const bool is_v = KEEP != kDense && group >= q_groups + kv_groups;
    const int head = R * (is_q ? group : is_v ? group - q_groups - kv_groups : group - q_groups) + mine;
    int64_t at = 0;  // row in the pages
    if constexpr (KEEP != kDense) {
      if (!is_q) {
        const int slot = a.slots[token];
        const int page = slot >> a.page_shift;
        if (slot < 0 || page >= a.n_pages) return;
        at = (((int64_t)page * a.n_kv + head) << a.page_shift) + (slot & ((1 << a.page_shift) - 1));
      }
    }
    if (head >= (is_q ? a.n_q : a.n_kv)) return;
    float x[N];
    raw.widen(x);
    if (!is_v) {
      float w[N];
      if (is_q) qw.widen(w);
      else kw.widen(w);
      float ss = 0.0f;
#pragma unroll
      for (int j = 0; j < N; j++) ss += x[j] * x[j];
      ss += lane_xor<1>(ss);
      ss += lane_xor<2>(ss);
      ss += lane_xor<4>(ss);
      ss += lane_xor<8>(ss);
      ss += lane_xor<16>(ss);
      if constexpr (N == 4) ss = half_wave_sum(ss);
      const float r = rsqrt_near(fmaf(ss, 1.0f / kD, a.eps));
#pragma unroll
      for (int j = 0; j < N; j++) x[j] = x[j] * r * w[j];
      if (rotary) {
        const f32x2_t* of_token = turn + (2 * here.t + (low ? 0 : 1)) * a.half;
        const f32x4_t* cs = reinterpret_cast<const f32x4_t*>(of_token + N * (low ? lane : partner));
#pragma unroll
        for (int j = 0; j < N; j += 2) {
          const f32x4_t c = cs[j / 2];
          const float o0 = __shfl(x[j], partner, kRowLanes<DT>), o1 = __shfl(x[j + 1], partner, kRowLanes<DT>);
          x[j] = x[j] * c.x + o0 * c.y;
          x[j + 1] = x[j + 1] * c.z + o1 * c.w;
        }
      }
    }
    if (is_q) {
      store_row<DT, N>(a.q_out, (token * a.n_q + head) * kD + N * lane, x);
    } else if constexpr (KEEP == kDense) {
      store_row<DT, N>(a.k_out, (token * a.n_kv + head) * kD + N * lane, x);
    } else {
      keep_row<DT, KEEP, PT>(is_v ? a.v_out : a.k_out, is_v ? a.v_scales : a.k_scales, is_v ? a.v_biases : a.k_biases, at, lane,
                             x);
    }
  };
  // (two sets of registers in turn: a copy from one to the other would wait for its load)
  while (item.t < tokens) {
    Item here = item;
    Raw<DT> other;
    next(item, kThreads / MSPR_WAVE);
    if (item.t < tokens) load(item, other);
    process(here, raw);
    if (item.t >= tokens) break;
    here = item;
    next(item, kThreads / MSPR_WAVE);
    if (item.t < tokens) load(item, raw);
    process(here, other);
  }
}

template <int DT, int KEEP, int PT>
int rope_launch(RopeArgs a, hipStream_t st) {
  constexpr int R = kRows<DT>;
  const int groups = (a.n_q + R - 1) / R + (KEEP == kDense ? 1 : 2) * ((a.n_kv + R - 1) / R);
  // Few rows: a group a wave, for latency, while the chip holds all of them at once. Many: a token's groups together, and up to
  // eight tokens, which share the angles' cost, where eight workgroups a compute unit are left (3844 tokens of float32 rows, in
  // workgroups of seven tokens each: 50 us, of one: 27; 16384 tokens of bfloat16 rows: 56 either way).
  const bool few = (int64_t)a.n_tokens * groups <= 8192;
  const int share = a.n_tokens / 2048;
  a.tokens_per_wg = few || share < 1 ? 1 : share > kMaxTokens ? kMaxTokens : share;
  a.groups_per_wg = few ? kThreads / MSPR_WAVE : groups;
  const dim3 grid((unsigned)((a.n_tokens + a.tokens_per_wg - 1) / a.tokens_per_wg),
                  (unsigned)((groups + a.groups_per_wg - 1) / a.groups_per_wg));
  qk_norm_rope_kernel<DT, KEEP, PT><<<grid, dim3(kThreads), 0, st>>>(a);
  MSPR_CHECK_LAUNCH("qk_norm_rope");
  return MSPR_OK;
}

int rope_checks(const char* what, const RopeArgs& a, int dtype, int head_dim) {
  MSPR_REQUIRE(a.q && a.k && a.q_weight && a.k_weight && a.positions && a.inv_freq && a.q_out && a.k_out, "%s: null pointer",
               what);
  MSPR_REQUIRE(dtype >= MSPR_F32 && dtype <= MSPR_BF16, "%s: dtype must be f32, f16 or bf16", what);
  MSPR_REQUIRE(head_dim == kD, "%s: head_dim must be 256", what);
  MSPR_REQUIRE(a.n_tokens >= 1 && a.n_tokens <= (1 << 24), "%s: 1 to 2^24 tokens", what);
  MSPR_REQUIRE(a.n_q >= 1 && a.n_kv >= 1 && a.n_q <= 1024 && a.n_kv <= 1024, "%s: 1 to 1024 heads of each kind", what);
  MSPR_REQUIRE(a.half >= 8 && a.half <= kMaxHalf && a.half % 8 == 0, "%s: the rotary width must be a multiple of 16 up to 256",
               what);
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
  MSPR_REQUIRE(a.n_pages >= 1 && (int64_t)a.n_pages * page_size <= 0x7FFFFFFF, "%s: the pool must hold fewer than 2^31 tokens",
               what);
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
