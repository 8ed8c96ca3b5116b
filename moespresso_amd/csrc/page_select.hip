// The pages that a query may weigh most, per KV head, and attention over them.
//
//   bound[h, p] = sum_d max(c[h, d] lo[p, d], c[h, d] hi[p, d]) * 2^(e_h + e_p)       c, e_h: the head's query in 8 bits
//   worth[p]    = max_h (bound[h, p] - max_p' bound[h, p'])
//
// over the pages p of the query's request: how far the largest product that a page may hold with a head lies below that head's
// best, at its best head (softmax weights fall with the exponential of that distance). The first pages and the last ones are taken
// whatever they are worth, of the others the best, ties to the lower page.
//
// A bound is a product of 512: the negative codes with lo, the positive ones with hi, by 16x16x64 integer matrix instructions.
// Sums are whole numbers below 2^24 and scales powers of two, so that a bound is exact in float32, and the selection does not
// depend on the order of anything.
//
// Two launches: bounds of 16 pages a wave (516 bytes a page and KV head), and the choice, a workgroup a query and KV head. Bound by
// latency: requests and lengths, table, bounds one after the other (4.7 us for one request of 256 or of 2048 pages), then the choice's
// barriers (4.3 us for 256 pages, 7.5 for 2048); 48 ragged requests read 49 MB of bounds in 14.3 us, 3.4 TB/s. The pages of a KV head are then
// pages of a pool of its own (page * n_kv + head, one head a page), over which paged_decode.hip attends.
#include "page_bounds.h"

namespace {

typedef __attribute__((ext_vector_type(4))) int i32x4_t;

constexpr int kTile = 16;          // pages of a matrix instruction
constexpr int kScoreWaves = 4;
// Tiles of all tables, as wide as they are, from which on a wave takes two (fewer: one, on as many more compute units). In us, with one
// and with two: a request of 256 pages 8.5 and 9.6, 16 of up to 2048 18.3 and 17.1, 64 such 36.6 and 33.1.
constexpr int kManyTiles = 1024;
constexpr int kMaxTablePages = 32768;  // a workgroup of 1024 threads has 32 a thread
constexpr int kMaxSelected = 4096;

struct SelectArgs {
  const void* q;            // [R, n_kv * rep, 256]
  const int32_t* requests;  // [R] or null
  const int32_t* lens;      // [R]
  const int32_t* tables;    // [n_tables, width]
  const int8_t* codes;      // [n_pages, n_kv, 2, 256]
  const float* scales;      // [n_pages, n_kv]
  int rows, n_kv, rep, width, n_tables, n_pages, page_shift, selected, first, recent;
  float* bounds;            // [R * n_kv][rep][padded]
  int padded;               // width, up to a multiple of 16
  int32_t* out;             // [R * n_kv][selected]
  int32_t* out_lens;        // [R * n_kv]
};

// Rows that query r sees, and its request's table (none: no rows).
struct Seen {
  int len, request;
};
__device__ __forceinline__ Seen seen_by(const SelectArgs& a, int r) {
  const int request = a.requests ? a.requests[r] : r;
  const int cap = a.width << a.page_shift;
  const int len = a.lens[r];
  const bool known = request >= 0 && request < a.n_tables;
  return Seen{!known || len < 0 ? 0 : len > cap ? cap : len, known ? request : 0};
}

// grid: (groups of pages, queries x KV heads)
template <int QDT, int TILES>
__global__ __launch_bounds__(64 * kScoreWaves) void page_score_kernel(SelectArgs a) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = blockIdx.y, r = row / a.n_kv, kvh = row - r * a.n_kv;
  const Seen seen = seen_by(a, r);
  const int n = (seen.len + (1 << a.page_shift) - 1) >> a.page_shift;
  if (n <= a.selected) return;  // (all of them are taken)
  const int tile0 = ((int)blockIdx.x * kScoreWaves + wave) * TILES;
  if (tile0 * kTile >= n) return;
  const int head = lane & 15, g = lane >> 4;
  // ---- page numbers, then the bounds of two tiles; the query in the meantime
  const int32_t* table = a.tables + (int64_t)seen.request * a.width;
  int page[TILES];
  bool good[TILES];
#pragma unroll
  for (int i = 0; i < TILES; i++) {
    const int p = (tile0 + i) * kTile + head;
    page[i] = p < n ? table[p] : -1;
  }
  const bool mine = head < a.rep;
  float x[64];  // channels 64 s + 16 g + j
  {
    const int64_t q0 = ((int64_t)row * a.rep + (mine ? head : 0)) * 256;
    constexpr int kBytes = QDT == MSPR_F32 ? 4 : 2;
#pragma unroll
    for (int s = 0; s < 4; s++) {
      const u32x4_t* from = reinterpret_cast<const u32x4_t*>(reinterpret_cast<const uint8_t*>(a.q) + (q0 + 64 * s + 16 * g) * kBytes);
      u32x4_t w[kBytes];
#pragma unroll
      for (int j = 0; j < kBytes; j++) w[j] = from[j];
#pragma unroll
      for (int j = 0; j < 16; j++) {
        if constexpr (QDT == MSPR_F32) x[16 * s + j] = __uint_as_float(w[j / 4][j % 4]);
        else if constexpr (QDT == MSPR_F16) x[16 * s + j] = f16_bits_to_f32((uint16_t)(w[j / 8][j / 2 % 4] >> 16 * (j % 2)));
        else x[16 * s + j] = bf16_bits_to_f32((uint16_t)(w[j / 8][j / 2 % 4] >> 16 * (j % 2)));
      }
    }
  }
  i32x4_t tile[TILES][8];
  float scale[TILES];
#pragma unroll
  for (int i = 0; i < TILES; i++) {
    good[i] = page[i] >= 0 && page[i] < a.n_pages;
    const int64_t at = (int64_t)(good[i] ? page[i] : 0) * a.n_kv + kvh;
    const i32x4_t* from = reinterpret_cast<const i32x4_t*>(a.codes + at * kBoundBytes + 16 * g);
#pragma unroll
    for (int s = 0; s < 8; s++) tile[i][s] = from[4 * s];
    scale[i] = a.scales[at];
  }
  // ---- the query's codes: operand s < 4 has the negative ones of 64 channels, 4 + s the positive ones
  float top = 0.0f;
#pragma unroll
  for (int j = 0; j < 64; j++) top = fmaxf(top, mine ? fabsf(x[j]) : 0.0f);
  top = half_wave_max(row_pair_max(top));
  const int e = bound_exponent(top);
  i32x4_t neg[4], pos[4];
#pragma unroll
  for (int s = 0; s < 4; s++)
#pragma unroll
    for (int w = 0; w < 4; w++) {
      uint32_t m = 0, p = 0;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int c = mine ? bound_code(rintf(__builtin_amdgcn_ldexpf(x[16 * s + 4 * w + j], -e))) : 0;
        m |= (uint32_t)((c < 0 ? c : 0) & 0xFF) << 8 * j;
        p |= (uint32_t)(c > 0 ? c : 0) << 8 * j;
      }
      neg[s][w] = (int)m;
      pos[s][w] = (int)p;
    }
  const float unit = __builtin_amdgcn_ldexpf(1.0f, e);
#pragma unroll
  for (int i = 0; i < TILES; i++) {
    const int p0 = (tile0 + i) * kTile;
    if (p0 >= n) break;
    i32x4_t acc = {0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < 4; s++) {
      acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(tile[i][s], neg[s], acc, 0, 0, 0);
      acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(tile[i][4 + s], pos[s], acc, 0, 0, 0);
    }
    // page 4 g + j of the tile, head `head`
    f32x4_t b;
    const float of_page = good[i] ? scale[i] : 0.0f;  // (bounds of a page that is not in the pool: none)
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const float s = __shfl(of_page, 4 * g + j, MSPR_WAVE);
      const bool there = __shfl((int)good[i], 4 * g + j, MSPR_WAVE) != 0;
      b[j] = there ? (float)acc[j] * unit * s : -__builtin_inff();
    }
    if (mine) *reinterpret_cast<f32x4_t*>(a.bounds + ((int64_t)row * a.rep + head) * a.padded + p0 + 4 * g) = b;
  }
}

constexpr int kBins = 1024;
constexpr int kRanked = 512;  // keys of a bin that are ranked one by one

// Largest value over the wave, in all lanes.
__device__ __forceinline__ float wave_max(float v) {
  v = fmaxf(v, lane_xor<1>(v));
  v = fmaxf(v, lane_xor<2>(v));
  v = fmaxf(v, lane_xor<4>(v));
  v = fmaxf(v, lane_xor<8>(v));
  return half_wave_max(row_pair_max(v));
}
// One step of the largest values of 2 HALF numbers a lane: lanes that differ in bit X exchange, and keep half of the numbers each.
template <int HALF, int X>
__device__ __forceinline__ void fold_max(float* v, int lane) {
  const bool up = (lane & X) != 0;
#pragma unroll
  for (int j = 0; j < HALF; j++) {
    const float keep = up ? v[HALF + j] : v[j], give = up ? v[j] : v[HALF + j];
    v[j] = fmaxf(keep, lane_xor<X>(give));
  }
}
__device__ __forceinline__ int wave_sum_upto(int v) {  // sums over this lane and those before it, by data-parallel moves
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
  return v;
}

// A workgroup a query and KV head, PER pages a thread, one behind the other, whose worths stay in registers. The worth of rank
// `selected` lies in one of 1024 bins over the range that worths have (a monotone map); the keys of that bin are ranked one by one, or,
// where they are too many (worths that are alike), the bin is found again among their 32-bit keys, ten bits at a time.
// HEADS: rows of bounds that are read, the query heads or, of fewer, the first again (without branches between them, their loads and
// reductions go on at once).
template <int THREADS, int PER, int HEADS>
__global__ __launch_bounds__(THREADS) void page_choose_kernel(SelectArgs a) {
  constexpr int kWaves = THREADS / 64;
  constexpr bool kHold = PER <= 8 && THREADS <= 512;  // all heads' bounds stay in registers between the best one and the worths
  static_assert(kWaves <= 16, "the waves' best bounds are sixteen a head");
  __shared__ int bins[kBins];
  __shared__ float tops[kWaves][16], lows[kWaves];
  __shared__ int sums[2][kWaves];
  __shared__ int found[2], listed;
  __shared__ uint32_t list_key[kRanked];
  __shared__ int list_page[kRanked];
  const int t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int row = blockIdx.x, r = row / a.n_kv, kvh = row - r * a.n_kv;
  const int p0 = t * PER;
  const float* bounds = a.bounds + (int64_t)row * a.rep * a.padded;
  // Bounds of head h, asked for ahead of the lengths and masked behind them (what lies behind the last page was not written; rows are
  // `padded`, a multiple of four, long).
  auto load_bounds = [&](int h, float* b) {
#pragma unroll
    for (int q = 0; q < PER / 4; q++) {
      const f32x4_t v = *reinterpret_cast<const f32x4_t*>(bounds + (int64_t)(h < a.rep ? h : 0) * a.padded + min(p0 + 4 * q, a.padded - 4));
#pragma unroll
      for (int i = 0; i < 4; i++) b[4 * q + i] = v[i];
    }
  };
  float held[kHold ? HEADS : 1][PER];
  if constexpr (kHold) {
#pragma unroll
    for (int h = 0; h < HEADS; h++) load_bounds(h, held[h]);
    __builtin_amdgcn_sched_barrier(0);
  }
  const Seen seen = seen_by(a, r);
  const int page_size = 1 << a.page_shift;
  const int n = __builtin_amdgcn_readfirstlane((seen.len + page_size - 1) >> a.page_shift);
  const int32_t* table = a.tables + (int64_t)seen.request * a.width;
  int32_t* out = a.out + (int64_t)row * a.selected;
  auto id_of = [&](int page) { return page >= 0 && page < a.n_pages ? page * a.n_kv + kvh : -1; };
  if (t == 0) a.out_lens[row] = n > a.selected ? seen.len - ((n - a.selected) << a.page_shift) : seen.len;
  if (n <= a.selected) {
    for (int i = t; i < a.selected; i += THREADS) out[i] = i < n ? id_of(table[i]) : -1;
    return;
  }
  // (asked for now: behind the choice each would be one more access to wait for)
  int page[kHold ? PER : 1];
  if constexpr (kHold) {
#pragma unroll
    for (int i = 0; i < PER; i++) page[i] = table[min(p0 + i, n - 1)];
  }
  auto mask_bounds = [&](float* b) {
#pragma unroll
    for (int i = 0; i < PER; i++) b[i] = p0 + i < n ? b[i] : -__builtin_inff();
  };
  // ---- every head's best bound
  auto best_of = [&](const float* b) {
    float best = b[0];
#pragma unroll
    for (int i = 1; i < PER; i++) best = fmaxf(best, b[i]);
    return best;
  };
  if constexpr (kHold) {
    float best[HEADS];
#pragma unroll
    for (int h = 0; h < HEADS; h++) {
      if (64 * PER * (wave + 1) > n) mask_bounds(held[h]);  // (wave-uniform: of the others all are there)
      best[h] = best_of(held[h]);
    }
    // (all heads together: a third of the instructions of one reduction a head)
    fold_max<HEADS / 2, 1>(best, lane);
    fold_max<HEADS / 4, 2>(best, lane);
    fold_max<HEADS / 8, 4>(best, lane);
    if constexpr (HEADS == 16) fold_max<1, 8>(best, lane);
    else best[0] = fmaxf(best[0], lane_xor<8>(best[0]));
    best[0] = half_wave_max(row_pair_max(best[0]));
    const int head = HEADS == 16 ? 8 * (lane & 1) + 4 * (lane >> 1 & 1) + 2 * (lane >> 2 & 1) + (lane >> 3 & 1)
                                 : 4 * (lane & 1) + 2 * (lane >> 1 & 1) + (lane >> 2 & 1);
    if (lane < HEADS) tops[wave][head] = best[0];
  } else {
#pragma unroll 1
    for (int h = 0; h < HEADS; h++) {
      load_bounds(h, held[0]);
      mask_bounds(held[0]);
      const float best = wave_max(best_of(held[0]));
      if (lane == 0) tops[wave][h] = best;
    }
  }
  for (int i = t; i < kBins; i += THREADS) bins[i] = 0;
  if (t == 0) listed = 0;
  __syncthreads();
  // ---- worths
  float worth[PER];
#pragma unroll
  for (int i = 0; i < PER; i++) worth[i] = -__builtin_inff();
  float of_head = -__builtin_inff();  // lane h: of head h
#pragma unroll
  for (int w = 0; w < kWaves; w++) of_head = fmaxf(of_head, tops[w][lane % HEADS]);
  of_head = of_head == -__builtin_inff() ? 0.0f : of_head;
  auto take = [&](int h, const float* b) {
    const float top = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(of_head), h));
#pragma unroll
    for (int i = 0; i < PER; i++) worth[i] = fmaxf(worth[i], b[i] - top);
  };
  if constexpr (kHold) {
#pragma unroll
    for (int h = 0; h < HEADS; h++) take(h, held[h]);
  } else {
#pragma unroll 1
    for (int h = 0; h < HEADS; h++) {
      load_bounds(h, held[0]);
      mask_bounds(held[0]);
      take(h, held[0]);
    }
  }
  auto always = [&](int p) { return p < a.first || p >= n - a.recent; };
  float low = 0.0f;  // (the best page of a head is worth nothing less)
#pragma unroll
  for (int i = 0; i < PER; i++)  // (a last page of few rows may lie far below the others)
    low = fminf(low, worth[i] == -__builtin_inff() || always(p0 + i) ? 0.0f : worth[i]);
  low = -wave_max(-low);
  if (lane == 0) lows[wave] = low;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; w++) low = fminf(low, lows[w]);
  // ---- the bin of the page of rank `selected`: from the last one down, in which the pages are that are taken whatever they are worth
  const float by = low < 0.0f ? (float)(kBins - 2) / -low : 0.0f;
  int bin[PER];
#pragma unroll
  for (int i = 0; i < PER; i++) {
    const int p = p0 + i;
    const float place = (worth[i] - low) * by;
    bin[i] = p >= n ? -1 : always(p) ? kBins - 1 : worth[i] == -__builtin_inff() ? 0 : min((int)place, kBins - 2);
    if (bin[i] >= 0) atomicAdd(&bins[bin[i]], 1);
  }
  // Which bin has the key of rank `want`, and its rank in it: thread t of 256 has four bins, from the highest down.
  auto find_bin = [&](int want) {
    __syncthreads();
    int own[4] = {}, mine = 0;
    if (t < kBins / 4)
#pragma unroll
      for (int i = 0; i < 4; i++) mine += own[i] = bins[kBins - 1 - 4 * t - i];
    const int upto = wave_sum_upto(mine);
    if (lane == 63) sums[0][wave] = upto;
    __syncthreads();
    int before = upto - mine;
    for (int w = 0; w < min(wave, 4); w++) before += sums[0][w];
    if (t < kBins / 4 && before < want && want <= before + mine)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        if (before < want && want <= before + own[i]) {
          found[0] = kBins - 1 - 4 * t - i;
          found[1] = want - before;
        }
        before += own[i];
      }
    __syncthreads();
  };
  find_bin(a.selected);
  const int last = found[0];
  int want = found[1];  // of that bin's pages
  const int in_bin = bins[last];
  static_assert(PER <= 32, "a bit a page");
  uint32_t taken = 0;
#pragma unroll
  for (int i = 0; i < PER; i++) taken |= (uint32_t)(bin[i] > last) << i;
  if (in_bin == want) {
#pragma unroll
    for (int i = 0; i < PER; i++) taken |= (uint32_t)(bin[i] == last) << i;
  } else if (in_bin <= kRanked) {
#pragma unroll
    for (int i = 0; i < PER; i++)
      if (bin[i] == last) {
        const int at = atomicAdd(&listed, 1);
        list_key[at] = score_key(worth[i]);
        list_page[at] = p0 + i;
      }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; i++)
      if (bin[i] == last) {
        const uint32_t key = score_key(worth[i]);
        int ahead = 0;  // pages of the bin that are worth more, or as much and lower
        for (int k = 0; k < in_bin; k++) ahead += list_key[k] > key || (list_key[k] == key && list_page[k] < p0 + i);
        taken |= (uint32_t)(ahead < want) << i;
      }
  } else {
    uint32_t prefix = 0, known = 0;
#pragma unroll 1
    for (int shift = 22; shift >= 0; shift = shift == 2 ? 0 : shift - 10) {  // bits 22 to 31, 12 to 21, 2 to 11, 0 and 1
      const uint32_t mask = shift == 0 ? 3u : 1023u;
      __syncthreads();
      for (int i = t; i < kBins; i += THREADS) bins[i] = 0;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < PER; i++) {
        const uint32_t key = score_key(worth[i]);
        if (bin[i] == last && (key & known) == prefix) atomicAdd(&bins[key >> shift & mask], 1);
      }
      find_bin(want);
      prefix |= (uint32_t)found[0] << shift;
      known |= mask << shift;
      want = found[1];
      if (shift == 0) break;
    }
    // the first `want` pages with that key
    int ties = 0;
#pragma unroll
    for (int i = 0; i < PER; i++) ties += bin[i] == last && score_key(worth[i]) == prefix;
    const int upto = wave_sum_upto(ties);
    if (lane == 63) sums[1][wave] = upto;
    __syncthreads();
    int before = upto - ties;
    for (int w = 0; w < wave; w++) before += sums[1][w];
#pragma unroll
    for (int i = 0; i < PER; i++)
      if (bin[i] == last) {
        const uint32_t key = score_key(worth[i]);
        taken |= (uint32_t)(key > prefix || (key == prefix && before++ < want)) << i;
      }
  }
  // ---- in the order of their positions
  const int mine = __builtin_popcount(taken);
  const int upto = wave_sum_upto(mine);
  __syncthreads();
  if (lane == 63) sums[0][wave] = upto;
  __syncthreads();
  int at = upto - mine;
  for (int w = 0; w < wave; w++) at += sums[0][w];
#pragma unroll
  for (int i = 0; i < PER; i++)
    if (taken >> i & 1) {
      if (at < a.selected) out[at] = id_of(kHold ? page[i] : table[p0 + i]);
      at++;
    }
}

struct SelectScratch {
  int padded;
  size_t bytes;
};
SelectScratch select_scratch(int64_t rows, int rep, int width) {
  SelectScratch s;
  s.padded = (width + kTile - 1) / kTile * kTile;
  s.bytes = (size_t)rows * rep * s.padded * sizeof(float);
  return s;
}

int select_fill(const char* what, SelectArgs& a, const void* q, int q_dtype, const int8_t* codes, const float* scales,
                const int32_t* tables, const int32_t* lens, const int32_t* requests, int rows, int n_q_heads, int n_kv_heads,
                int head_dim, int n_pages, int page_size, int n_tables, int table_width, int selected, int first, int recent,
                void* workspace, size_t workspace_bytes) {
  MSPR_REQUIRE(q && codes && scales && tables && lens, "%s: null pointer", what);
  MSPR_REQUIRE(q_dtype >= MSPR_F32 && q_dtype <= MSPR_BF16, "%s: queries must be f32, f16 or bf16", what);
  MSPR_REQUIRE(head_dim == 256, "%s: head_dim must be 256", what);
  MSPR_REQUIRE(n_kv_heads >= 1 && n_kv_heads <= 1024 && n_q_heads >= n_kv_heads && n_q_heads % n_kv_heads == 0,
               "%s: bad head counts", what);
  MSPR_REQUIRE(n_q_heads / n_kv_heads <= 16, "%s: at most 16 query heads per KV head", what);
  MSPR_REQUIRE(rows >= 1 && (int64_t)rows * n_kv_heads <= 65535, "%s: 1 to 65535 queries times KV heads", what);
  MSPR_REQUIRE(n_tables >= 1 && (requests || n_tables == rows), "%s: a table for every query, or the requests they belong to", what);
  MSPR_REQUIRE(page_size >= 16 && (page_size & (page_size - 1)) == 0, "%s: page_size must be a power of two from 16 on", what);
  MSPR_REQUIRE(n_pages >= 1 && (int64_t)n_pages * n_kv_heads * page_size <= 0x7FFFFFFF,
               "%s: the pool must hold fewer than 2^31 tokens times KV heads", what);
  MSPR_REQUIRE(table_width >= 1 && table_width <= kMaxTablePages && (int64_t)table_width * page_size <= 0x40000000,
               "%s: a request's table must hold 1 to %d pages and at most 2^30 tokens", what, kMaxTablePages);
  MSPR_REQUIRE(first >= 0 && recent >= 1 && selected >= 1 && selected <= kMaxSelected && (int64_t)first + recent <= selected,
               "%s: first >= 0, recent >= 1, and both together within 1 to %d selected pages", what, kMaxSelected);
  MSPR_REQUIRE(mspr_aligned(q, 16) && mspr_aligned(codes, 16) && mspr_aligned(scales, 4), "%s: pointers must be 16-byte aligned", what);
  const int rep = n_q_heads / n_kv_heads;
  const SelectScratch s = select_scratch((int64_t)rows * n_kv_heads, rep, table_width);
  MSPR_REQUIRE(workspace && workspace_bytes >= s.bytes && mspr_aligned(workspace, 16),
               "%s: workspace of %zu bytes (16-byte aligned) needed, %zu given", what, s.bytes, workspace_bytes);
  a = SelectArgs{};
  a.q = q;
  a.requests = requests;
  a.lens = lens;
  a.tables = tables;
  a.codes = codes;
  a.scales = scales;
  a.rows = rows;
  a.n_kv = n_kv_heads;
  a.rep = rep;
  a.width = table_width;
  a.n_tables = n_tables;
  a.n_pages = n_pages;
  a.page_shift = __builtin_ctz(page_size);
  a.selected = selected;
  a.first = first;
  a.recent = recent;
  a.padded = s.padded;
  a.bounds = reinterpret_cast<float*>(workspace);
  return MSPR_OK;
}

int select_launch(const char* what, const SelectArgs& a, int q_dtype, hipStream_t st) {
  const unsigned rows = (unsigned)(a.rows * a.n_kv);
  if (a.width > a.selected) {
    auto score = [&](auto tiles) {
      constexpr int kTiles = decltype(tiles)::value, kPages = kTile * kScoreWaves * kTiles;
      const dim3 grid((unsigned)((a.width + kPages - 1) / kPages), rows);
      if (q_dtype == MSPR_F32) page_score_kernel<MSPR_F32, kTiles><<<grid, dim3(64 * kScoreWaves), 0, st>>>(a);
      else if (q_dtype == MSPR_F16) page_score_kernel<MSPR_F16, kTiles><<<grid, dim3(64 * kScoreWaves), 0, st>>>(a);
      else page_score_kernel<MSPR_BF16, kTiles><<<grid, dim3(64 * kScoreWaves), 0, st>>>(a);
    };
    if ((int64_t)rows * ((a.width + kTile - 1) / kTile) < kManyTiles) score(std::integral_constant<int, 1>{});
    else score(std::integral_constant<int, 2>{});
    MSPR_CHECK_LAUNCH(what);
  }
  // (In us: 256 pages by 256 threads 8.5, by 512 10.1, by 1024 14.8; 16 requests of up to 2048 pages by 512 17.0, by 1024 22.2. Rows of bounds
  // for 16 heads where there are 8: 256 pages 8.8, 2048 13.3 instead of 11.6.)
  auto choose = [&](auto heads) {
    constexpr int kHeads = decltype(heads)::value;
    if (a.width <= 1024) page_choose_kernel<256, 4, kHeads><<<dim3(rows), dim3(256), 0, st>>>(a);
    else if (a.width <= 4096) page_choose_kernel<512, 8, kHeads><<<dim3(rows), dim3(512), 0, st>>>(a);
    else if (a.width <= 8192) page_choose_kernel<1024, 8, kHeads><<<dim3(rows), dim3(1024), 0, st>>>(a);
    else page_choose_kernel<1024, 32, kHeads><<<dim3(rows), dim3(1024), 0, st>>>(a);
  };
  if (a.rep <= 8) choose(std::integral_constant<int, 8>{});
  else choose(std::integral_constant<int, 16>{});
  MSPR_CHECK_LAUNCH(what);
  return MSPR_OK;
}

// Scratch of a sparse call: the selection's, then its tables and lengths, then the decode's.
struct SparseScratch {
  size_t select, tables, lens, decode;
  size_t total() const { return select + tables + lens + decode; }
};
SparseScratch sparse_scratch(int rows, int n_q_heads, int n_kv_heads, int page_size, int table_width, int selected) {
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  SparseScratch s;
  s.select = up(select_scratch((int64_t)rows * n_kv_heads, n_q_heads / n_kv_heads, table_width).bytes);
  s.tables = up((size_t)rows * n_kv_heads * selected * sizeof(int32_t));
  s.lens = up((size_t)rows * n_kv_heads * sizeof(int32_t));
  s.decode = mspr_sdpa_decode_paged_workspace_bytes(rows * n_kv_heads, n_q_heads / n_kv_heads, 1, page_size, selected);
  return s;
}

bool sparse_sizes_ok(int rows, int n_q_heads, int n_kv_heads, int page_size, int table_width, int selected) {
  return rows >= 1 && n_kv_heads >= 1 && n_q_heads >= n_kv_heads && page_size >= 1 && table_width >= 1 && selected >= 1 &&
         (int64_t)rows * n_kv_heads <= 65535 && n_q_heads / n_kv_heads <= 16 && table_width <= kMaxTablePages &&
         selected <= kMaxSelected;
}

// The selection of a sparse call into its workspace; then the decode's operands.
struct Sparse {
  int32_t *tables, *lens;
  void* workspace;
  size_t bytes;
};
int sparse_select(const char* what, const void* q, int q_dtype, const int8_t* codes, const float* scales, const int32_t* tables,
                  const int32_t* lens, const int32_t* requests, int rows, int n_q_heads, int n_kv_heads, int head_dim, int n_pages,
                  int page_size, int n_tables, int table_width, int selected, int first, int recent, float scale, void* workspace,
                  size_t workspace_bytes, Sparse* s, hipStream_t st) {
  MSPR_REQUIRE(selected >= 1 && (int64_t)selected * page_size <= 0x40000000 &&
                   (int64_t)rows * n_kv_heads * (((int64_t)selected * page_size + 31) / 32 + 1) <= 0x3FFFFFFF,
               "%s: the selected pages hold too many tokens together", what);
  // (a negative scale would turn the order of the bounds round)
  MSPR_REQUIRE(scale >= 0.0f, "%s: the softmax scale must not be negative", what);
  SelectArgs a;
  if (int rc = select_fill(what, a, q, q_dtype, codes, scales, tables, lens, requests, rows, n_q_heads, n_kv_heads, head_dim, n_pages,
                           page_size, n_tables, table_width, selected, first, recent, workspace, workspace_bytes))
    return rc;
  const SparseScratch z = sparse_scratch(rows, n_q_heads, n_kv_heads, page_size, table_width, selected);
  MSPR_REQUIRE(workspace_bytes >= z.total(), "%s: workspace of %zu bytes needed, %zu given", what, z.total(), workspace_bytes);
  uint8_t* at = reinterpret_cast<uint8_t*>(workspace) + z.select;
  s->tables = a.out = reinterpret_cast<int32_t*>(at);
  s->lens = a.out_lens = reinterpret_cast<int32_t*>(at += z.tables);
  s->workspace = at + z.lens;
  s->bytes = z.decode;
  return select_launch(what, a, q_dtype, st);
}

}  // namespace

extern "C" size_t mspr_select_pages_workspace_bytes(int batch, int n_q_heads, int n_kv_heads, int table_width) {
  if (!sparse_sizes_ok(batch, n_q_heads, n_kv_heads, 16, table_width, 1)) return 0;
  return select_scratch((int64_t)batch * n_kv_heads, n_q_heads / n_kv_heads, table_width).bytes;
}

extern "C" int mspr_select_pages(const void* queries, int q_dtype, const int8_t* codes, const float* scales, const int32_t* tables,
                                 const int32_t* lens, const int32_t* requests, int batch, int n_q_heads, int n_kv_heads,
                                 int head_dim, int n_pages, int page_size, int n_tables, int table_width, int selected, int first,
                                 int recent, int32_t* out_tables, int32_t* out_lens, void* workspace, size_t workspace_bytes,
                                 void* stream) {
  MSPR_REQUIRE(out_tables && out_lens, "select_pages: null pointer");
  SelectArgs a;
  if (int rc = select_fill("select_pages", a, queries, q_dtype, codes, scales, tables, lens, requests, batch, n_q_heads, n_kv_heads,
                           head_dim, n_pages, page_size, n_tables, table_width, selected, first, recent, workspace, workspace_bytes))
    return rc;
  a.out = out_tables;
  a.out_lens = out_lens;
  return select_launch("select_pages", a, q_dtype, (hipStream_t)stream);
}

extern "C" size_t mspr_sdpa_decode_paged_sparse_workspace_bytes(int batch, int n_q_heads, int n_kv_heads, int page_size,
                                                                int table_width, int selected) {
  if (!sparse_sizes_ok(batch, n_q_heads, n_kv_heads, page_size, table_width, selected)) return 0;
  return sparse_scratch(batch, n_q_heads, n_kv_heads, page_size, table_width, selected).total();
}

extern "C" int mspr_sdpa_decode_paged_sparse(const void* queries, const void* k_pages, const void* v_pages, int dtype,
                                             const int8_t* codes, const float* scales, const int32_t* tables, const int32_t* lens,
                                             const int32_t* requests, int batch, int n_q_heads, int n_kv_heads, int head_dim,
                                             int n_pages, int page_size, int n_tables, int table_width, int selected, int first,
                                             int recent, float scale, void* out, void* workspace, size_t workspace_bytes,
                                             void* stream) {
  const char* what = "sdpa_decode_paged_sparse";
  MSPR_REQUIRE(dtype == MSPR_F16 || dtype == MSPR_BF16, "%s: dtype must be f16 or bf16", what);
  MSPR_REQUIRE(k_pages && v_pages && out, "%s: null pointer", what);
  MSPR_REQUIRE(mspr_aligned(k_pages, 16) && mspr_aligned(v_pages, 16) && mspr_aligned(out, 16), "%s: pointers must be 16-byte aligned", what);
  Sparse s;
  if (int rc = sparse_select(what, queries, dtype, codes, scales, tables, lens, requests, batch, n_q_heads, n_kv_heads, head_dim,
                             n_pages, page_size, n_tables, table_width, selected, first, recent, scale, workspace, workspace_bytes, &s,
                             (hipStream_t)stream))
    return rc;
  return mspr_sdpa_decode_paged(queries, k_pages, v_pages, dtype, s.tables, s.lens, nullptr, batch * n_kv_heads,
                                n_q_heads / n_kv_heads, 1, head_dim, n_pages * n_kv_heads, page_size, batch * n_kv_heads, selected,
                                scale, out, s.workspace, s.bytes, stream);
}

extern "C" int mspr_sdpa_decode_paged_sparse_q8(const void* queries, int q_dtype, const void* k_wq, const void* k_scales,
                                                const void* k_biases, const void* v_wq, const void* v_scales,
                                                const void* v_biases, int sb_dtype, const int8_t* codes, const float* scales,
                                                const int32_t* tables, const int32_t* lens, const int32_t* requests, int batch,
                                                int n_q_heads, int n_kv_heads, int head_dim, int n_pages, int page_size,
                                                int n_tables, int table_width, int selected, int first, int recent, float scale,
                                                int group_size, int bits, void* out, void* workspace, size_t workspace_bytes,
                                                void* stream) {
  const char* what = "sdpa_decode_paged_sparse_q8";
  MSPR_REQUIRE(group_size == 64 && bits == 8, "%s: only group_size=64, bits=8 is supported", what);
  MSPR_REQUIRE(sb_dtype >= MSPR_F32 && sb_dtype <= MSPR_BF16, "%s: scales must be f32, f16 or bf16", what);
  for (const void* p : {k_wq, k_scales, k_biases, v_wq, v_scales, v_biases, (const void*)out}) {
    MSPR_REQUIRE(p, "%s: null pointer", what);
    MSPR_REQUIRE(mspr_aligned(p, 16), "%s: pointers must be 16-byte aligned", what);
  }
  Sparse s;
  if (int rc = sparse_select(what, queries, q_dtype, codes, scales, tables, lens, requests, batch, n_q_heads, n_kv_heads, head_dim,
                             n_pages, page_size, n_tables, table_width, selected, first, recent, scale, workspace, workspace_bytes, &s,
                             (hipStream_t)stream))
    return rc;
  return mspr_sdpa_decode_paged_q8(queries, q_dtype, k_wq, k_scales, k_biases, v_wq, v_scales, v_biases, sb_dtype, s.tables, s.lens,
                                   nullptr, batch * n_kv_heads, n_q_heads / n_kv_heads, 1, head_dim, n_pages * n_kv_heads, page_size,
                                   batch * n_kv_heads, selected, scale, group_size, bits, out, s.workspace, s.bytes, stream);
}
