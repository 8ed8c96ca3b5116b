// Bounds of the keys of every page that a step wrote to, in 8 bits.
//
//   e = smallest with max |k| <= 127 * 2^e,   lo[d] = floor(min k[d] * 2^-e),   hi[d] = ceil(max k[d] * 2^-e)
//
// over the rows of a page and KV head. Steps are powers of two because floor(floor(x / 2^a) / 2^b) = floor(x / 2^(a + b)): bounds made
// of the old codes and the new rows equal those of all rows, so that an append reads its own rows only.
//
// Bound by latency (slots, rows, codes one after the other; 16 tokens 3.6 us, 16088 rows of 8 bits, 4.2 MB, 6.7 us): a key row is read once. A
// workgroup takes the runs of rows (consecutive slots of one page) that end among `span` rows of the step, of one KV head; its
// four waves take a run's rows in turn, two 16-bit rows or one 8-bit row a load, and meet in LDS. 8-bit rows are code * scale +
// bias in 64 bits, rounded down for the lower bounds and up for the upper ones: a value next to a whole number of steps must not be
// rounded to it.
#include "page_bounds.h"

namespace {

constexpr int kWaves = 4;
constexpr int kAffineRows = 3;  // page format beside MSPR_F16 and MSPR_BF16

template <typename T>
__device__ __forceinline__ T min_of(T a, T b);
template <>
__device__ __forceinline__ float min_of(float a, float b) { return fminf(a, b); }
template <>
__device__ __forceinline__ double min_of(double a, double b) { return fmin(a, b); }
template <typename T>
__device__ __forceinline__ T max_of(T a, T b) { return -min_of(-a, -b); }
template <>
__device__ __forceinline__ float max_of(float a, float b) { return fmaxf(a, b); }
template <>
__device__ __forceinline__ double max_of(double a, double b) { return fmax(a, b); }

// Whether code * scale + bias is a float64 number for every code: of the scale's exponent E and the bias's F (multiples of 2^(E - 23) and
// 2^(F - 23), sums below 2^(max(E + 9, F + 1) + 1)) 53 bits are enough where F - E is within -20 and 28. (Of zeros, infinities and NaN
// either answer will do.)
__device__ __forceinline__ bool affine_is_exact(float scale, float bias) {
  return (unsigned)(__builtin_amdgcn_frexp_expf(bias) - __builtin_amdgcn_frexp_expf(scale) + 20) <= 48u;
}
// code * scale + bias between the two float64 numbers nearest to it (the same number twice where it is one). The product, of 32 bits, is
// exact, and so is the rest of the sum. Whole numbers of a step are float64 numbers themselves, so that rounding down and up leaves
// floor, ceiling and exponent as they are of the number that is meant. (The sum rounded to nearest put 127 + 10^-20 within 127 steps of 1.)
// In us a call of a captured graph, 16088 rows of two KV heads: 9.1 where all sums are exact anyway (8.9 without the question whether
// they are), 21.6 with this for every row.
__device__ __forceinline__ void affine_within(double code, double scale, double bias, double* below, double* above) {
  const double product = code * scale, sum = product + bias;
  const double of_bias = sum - product;
  const double rest = (product - (sum - of_bias)) + (bias - of_bias);
  const int64_t bits = __builtin_bit_cast(int64_t, sum);  // (a sum of zero has no rest)
  *below = rest < 0.0 ? __builtin_bit_cast(double, bits + (sum < 0.0 ? 1 : -1)) : sum;
  *above = rest > 0.0 ? __builtin_bit_cast(double, bits + (sum < 0.0 ? -1 : 1)) : sum;
}

// FMT: type of 16-bit rows, or 8-bit ones with scales of SDT. grid: (spans, KV heads)
template <int FMT, int SDT>
__global__ __launch_bounds__(64 * kWaves) void page_bounds_kernel(const int32_t* slots, const void* keys, const void* key_scales,
                                                                  const void* key_biases, int8_t* codes, float* scales, int n_rows,
                                                                  int span, int page_shift, int n_pages) {
  constexpr bool kCodes = FMT == kAffineRows;
  using T = std::conditional_t<kCodes, double, float>;
  constexpr int kElements = kCodes ? 4 : 8;     // channels a lane has of a row
  constexpr int kLanes = 256 / kElements;       // lanes of a row
  constexpr int kRows = 64 / kLanes;            // rows a load
  constexpr int kAhead = kCodes ? 16 : 8;       // loads in flight: sixteen rows a wave
  const T inf = (T)__builtin_inff();
  __shared__ T edge[2][kWaves * kRows][256];
  __shared__ float tops[kWaves];
  const int t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int n_kv = gridDim.y, kvh = blockIdx.y;
  const int page_mask = (1 << page_shift) - 1;
  const int r0 = blockIdx.x * span;
  const int mine = lane / kLanes, channel = kElements * (lane % kLanes);
  auto slot_at = [&](int r) { return r >= 0 && r < n_rows ? slots[r] : -1; };
  // which of the span's rows are the last of their run, all at once
  const int here = lane < span ? slot_at(r0 + lane) : -1, behind = slot_at(r0 + lane + 1);
  uint64_t ends = __ballot(here >= 0 && here >> page_shift < n_pages && (behind != here + 1 || (here & page_mask) == page_mask));
  for (; ends; ends &= ends - 1) {
    const int i_end = __builtin_ctzll(ends), r = r0 + i_end;
    const int slot = __builtin_amdgcn_readlane(here, i_end);
    const int page = slot >> page_shift, row = slot & page_mask;
    int count = 0;  // rows of the run
    for (int back = 0; back <= row; back += 64) {
      const uint64_t broken = __ballot(back + lane > row || slot_at(r - back - lane) != slot - back - lane);
      const int more = broken ? __builtin_ctzll(broken) : 64;
      count += more;
      if (more < 64) break;
    }
    const int64_t page_head = (int64_t)page * n_kv + kvh;
    const bool fresh = count > row;
    // (asked for ahead of the rows)
    int8_t old_lo = 0, old_hi = 0;
    float old_scale = 0.0f;
    int8_t* at = codes + page_head * kBoundBytes;
    if (!fresh) {
      old_lo = at[t];
      old_hi = at[256 + t];
      old_scale = scales[page_head];
    }
    const int64_t first = (page_head << page_shift) + (row + 1 - count);
    T lo[kElements], hi[kElements];
#pragma unroll
    for (int j = 0; j < kElements; j++) {
      lo[j] = inf;
      hi[j] = -inf;
    }
    using Word = std::conditional_t<kCodes, uint32_t, u32x4_t>;
    auto row_at = [&](int i) { return first + min(i, count - 1); };  // (behind the last, the last again)
    auto word_at = [&](int64_t from) {
      return reinterpret_cast<const Word*>(reinterpret_cast<const uint8_t*>(keys) + from * (kCodes ? 256 : 512))[lane % kLanes];
    };
    auto scale_at = [&](const void* of, int64_t from) { return load_as_f32<SDT>(of, from * 4 + channel / 64); };
    bool exact = true;
    for (int i0 = kRows * wave; i0 < count; i0 += kRows * kWaves * kAhead) {
      Word raw[kAhead];
      float scale[kAhead], bias[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; k++) {
        const int64_t from = row_at(i0 + kRows * kWaves * k + mine);
        raw[k] = word_at(from);
        if constexpr (kCodes) {
          scale[k] = scale_at(key_scales, from);
          bias[k] = scale_at(key_biases, from);
        }
      }
      if constexpr (kCodes) {  // (the sixteen lanes of a group look at its scales of the sixteen rows)
        static_assert(kAhead == 64 / kElements, "a lane of a group for every row");
        int tl = lane;
        asm volatile("" : "+v"(tl));  // (made here: registers for a workgroup more a compute unit, 9.8 -> 9.1 us for 16088 rows)
        const int64_t from = row_at(i0 + kWaves * (tl % kAhead));
        exact &= affine_is_exact(scale_at(key_scales, from), scale_at(key_biases, from));
      }
#pragma unroll
      for (int k = 0; k < kAhead; k++) {
#pragma unroll
        for (int j = 0; j < kElements; j++) {
          T x;
          if constexpr (kCodes) x = fma((double)(raw[k] >> 8 * j & 0xFFu), (double)scale[k], (double)bias[k]);
          else if constexpr (FMT == MSPR_F16) x = f16_bits_to_f32((uint16_t)(raw[k][j / 2] >> 16 * (j % 2)));
          else x = bf16_bits_to_f32((uint16_t)(raw[k][j / 2] >> 16 * (j % 2)));
          lo[j] = min_of(lo[j], x);
          hi[j] = max_of(hi[j], x);
        }
      }
    }
    if constexpr (kCodes) {
      // (a sum rounded to nearest is one of the two numbers beside it: the outer ones replace it)
      if (!__all(exact)) {
        asm volatile("" ::: "memory");  // (addresses are made anew, not kept through the loop above)
#pragma unroll 1
        for (int i = wave; i < count; i += kWaves) {
          const int64_t from = row_at(i);
          const Word word = word_at(from);
          const double s = scale_at(key_scales, from), z = scale_at(key_biases, from);
#pragma unroll
          for (int j = 0; j < kElements; j++) {
            double below, above;
            affine_within((double)(word >> 8 * j & 0xFFu), s, z, &below, &above);
            lo[j] = min_of(lo[j], below);
            hi[j] = max_of(hi[j], above);
          }
        }
      }
    }
    __syncthreads();  // (of the run before, all is read)
#pragma unroll
    for (int j = 0; j < kElements; j++) {
      edge[0][wave * kRows + mine][channel + j] = lo[j];
      edge[1][wave * kRows + mine][channel + j] = hi[j];
    }
    __syncthreads();
    // a channel a thread
    T low = inf, high = -inf;
#pragma unroll
    for (int w = 0; w < kWaves * kRows; w++) {
      low = min_of(low, edge[0][w][t]);
      high = max_of(high, edge[1][w][t]);
    }
    const bool some = low <= high;  // (a channel of NaN only has neither)
    // (the exponent of the largest magnitude is the largest exponent)
    const T top = some ? max_of(max_of(-low, high), (T)0) : (T)0;
    int e = bound_exponent(top);
    for (int m = 32; m > 0; m >>= 1) e = max(e, __shfl_xor(e, m, MSPR_WAVE));
    if (lane == 0) tops[wave] = (float)e;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; w++) e = max(e, (int)tops[w]);
    int shift = 0;  // of the old codes, to the new step
    if (!fresh) {
      const int old = old_scale > 0.0f ? min(max(__builtin_amdgcn_frexp_expf(old_scale) - 1, -kBoundLimit), kBoundLimit) : -kBoundLimit;
      e = max(e, old);
      shift = min(e - old, 31);
    }
    int code_lo = 0, code_hi = 0;
    if (some) {
      if constexpr (kCodes) {
        code_lo = (int)fmin(fmax(floor(ldexp(low, -e)), -127.0), 127.0);
        code_hi = (int)fmin(fmax(ceil(ldexp(high, -e)), -127.0), 127.0);
      } else {
        // (a bfloat16 number 2^-150 of the step becomes zero, but stays on its side of it)
        code_lo = min(bound_code(floorf(__builtin_amdgcn_ldexpf(low, -e))), low < 0.0f ? -1 : 127);
        code_hi = max(bound_code(ceilf(__builtin_amdgcn_ldexpf(high, -e))), high > 0.0f ? 1 : -127);
      }
    }
    if (!fresh) {
      const int before_lo = (int)old_lo >> shift, before_hi = -(-(int)old_hi >> shift);  // floor and ceiling of the old ones
      code_lo = some ? min(code_lo, before_lo) : before_lo;
      code_hi = some ? max(code_hi, before_hi) : before_hi;
    }
    at[t] = (int8_t)code_lo;
    at[256 + t] = (int8_t)code_hi;
    if (t == 0) scales[page_head] = __builtin_amdgcn_ldexpf(1.0f, e);
  }
}

// Rows of a step from which on a workgroup looks after sixteen of them (fewer: each after one, which may end a run). In us with the
// copies of a captured call, sixteen and one: 16 requests of one row 29.7 and 8.8, 1024 such 34.0 and 16.3, 8 of 400 8-bit rows 10.4 and 12.7
// (16-bit ones 11.8 and 12.6), 8 of 2011 12.1 and 24.4 (64 rows a workgroup 14.1).
constexpr int kManyRows = 2048;

template <int FMT, int SDT>
int bounds_launch(const int32_t* slots, const void* keys, const void* scales_of_keys, const void* biases, int8_t* codes, float* scales,
                  int n_rows, int n_kv, int n_pages, int page_size, hipStream_t st) {
  const int span = n_rows < kManyRows ? 1 : 16;
  page_bounds_kernel<FMT, SDT><<<dim3((unsigned)((n_rows + span - 1) / span), (unsigned)n_kv), dim3(64 * kWaves), 0, st>>>(
      slots, keys, scales_of_keys, biases, codes, scales, n_rows, span, __builtin_ctz(page_size), n_pages);
  MSPR_CHECK_LAUNCH("page_bounds");
  return MSPR_OK;
}

int bounds_check(const void* slots, const void* keys, const void* codes, const void* scales, int n_rows, int n_kv, int head_dim,
                 int n_pages, int page_size) {
  MSPR_REQUIRE(slots && keys && codes && scales, "page_bounds: null pointer");
  MSPR_REQUIRE(head_dim == 256, "page_bounds: head_dim must be 256");
  MSPR_REQUIRE(n_rows >= 1 && n_kv >= 1 && n_kv <= 1024, "page_bounds: 1 row or more, 1 to 1024 KV heads");
  MSPR_REQUIRE(page_size >= 16 && (page_size & (page_size - 1)) == 0, "page_bounds: page_size must be a power of two from 16 on");
  MSPR_REQUIRE(n_pages >= 1 && (int64_t)n_pages * page_size <= 0x7FFFFFFF, "page_bounds: the pool must hold fewer than 2^31 tokens");
  MSPR_REQUIRE(mspr_aligned(keys, 16) && mspr_aligned(codes, 16) && mspr_aligned(scales, 4), "page_bounds: pointers must be 16-byte aligned");
  return MSPR_OK;
}

}  // namespace

extern "C" int mspr_page_bounds(const int32_t* slots, const void* k_pages, int dtype, int n_rows, int n_kv_heads, int head_dim,
                                int n_pages, int page_size, int8_t* codes, float* scales, void* stream) {
  MSPR_REQUIRE(dtype == MSPR_F16 || dtype == MSPR_BF16, "page_bounds: pages must be f16 or bf16");
  if (int rc = bounds_check(slots, k_pages, codes, scales, n_rows, n_kv_heads, head_dim, n_pages, page_size)) return rc;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == MSPR_F16)
    return bounds_launch<MSPR_F16, MSPR_F16>(slots, k_pages, nullptr, nullptr, codes, scales, n_rows, n_kv_heads, n_pages, page_size, st);
  return bounds_launch<MSPR_BF16, MSPR_BF16>(slots, k_pages, nullptr, nullptr, codes, scales, n_rows, n_kv_heads, n_pages, page_size, st);
}

extern "C" int mspr_page_bounds_q8(const int32_t* slots, const void* k_wq, const void* k_scales, const void* k_biases, int sb_dtype,
                                   int n_rows, int n_kv_heads, int head_dim, int n_pages, int page_size, int8_t* codes,
                                   float* scales, void* stream) {
  MSPR_REQUIRE(sb_dtype >= MSPR_F32 && sb_dtype <= MSPR_BF16, "page_bounds: scales must be f32, f16 or bf16");
  MSPR_REQUIRE(k_scales && k_biases, "page_bounds: null pointer");
  if (int rc = bounds_check(slots, k_wq, codes, scales, n_rows, n_kv_heads, head_dim, n_pages, page_size)) return rc;
  hipStream_t st = (hipStream_t)stream;
#define MSPR_BOUNDS(sdt) \
  bounds_launch<kAffineRows, sdt>(slots, k_wq, k_scales, k_biases, codes, scales, n_rows, n_kv_heads, n_pages, page_size, st)
  if (sb_dtype == MSPR_F32) return MSPR_BOUNDS(MSPR_F32);
  if (sb_dtype == MSPR_F16) return MSPR_BOUNDS(MSPR_F16);
  return MSPR_BOUNDS(MSPR_BF16);
#undef MSPR_BOUNDS
}
