// Attention of one new token per request over a paged KV cache.
//
//   out[b, h] = sum_k softmax_k(q[b, h] . K[k] * scale) V[k]   over the lens[b] rows that the query's table names, 0 where
//                                                              there are none
//
// Pages [n_pages][KV heads][page_size][256] of 16-bit rows, or affine 8-bit rows in groups of 64 (value = code * scale + bias).
// Head dim 256, up to 16 query heads per KV head.
//
// Bound by HBM: every key and value row is read once (1024 bytes of 16-bit rows a key and KV head, 544 of 8-bit ones with
// 16-bit scales) and met by 16 FLOP a byte. A wave walks 32-key tiles of a request and KV head (a row of tiles) with an online
// softmax of its own.
//
// What is attended where follows from the lengths, which only the device knows: the rows of tiles lie in one line, of which
// every workgroup takes an equal share (with ranges cut request by request, the last workgroups of ragged batches ran alone:
// 212 us where 64 requests of up to 16384 rows took 167 in shares). A share holds parts of one row or of several; a part
// that is not its whole row leaves partials, and only rows that were cut go through the second kernel.
//
// With few rows the four waves of a workgroup take a share's tiles in turn and meet in LDS. With many, whose parts have few
// tiles, every wave takes a share of its own: nothing is exchanged, and no wave waits for another.
//
// Rows are read as buffer windows: rows that do not count, in the last tile, behind it or in a page that is not in the pool,
// read as zeros and cost no access, so that a wave always asks for a next tile and what is outstanding does not depend on
// it. Loads are non-temporal (8 requests of 37000 rows 107 -> 97 us).
//
// Per tile and wave: K rows come from HBM into registers as the A operand of S^T = K.Q^T (keys x heads, so that a head's
// statistics lie in one lane column); V rows pass through LDS, whose transpose read yields the A operand of O^T = V^T.P^T.
// Products are exact: 16-bit rows are multiplied as they are and the scale is applied to the sums; 8-bit codes are multiplied
// as the whole numbers they are. A group's sum over K then takes its scale in float32; a group's scale of V goes into the
// weights first; biases are products of their own, of float32 matrix instructions (K: biases x sums of the query over a
// group, V: weights x biases). Codes count from 128 on, and 128 scales go into the biases: of rows around zero, the sums over
// codes and over biases would be many times the result, and what is lost in them (float32 results over 37000 keys are 0.5e-6
// off, 0.9e-6 with K's codes from 0 on, 1.8e-6 with V's). Weights, and queries whose type has more digits than an operand, go
// in as two terms of it, the rounded value and the rounded rest. Weights of 8-bit rows do so for a bfloat16 result too, though
// it has fewer digits than one float16 term: the sums over codes and over biases, which take the weights apart, may be many
// times the result (a key whose scale is 10^4 of the others' left results 1.8e-2 of the values' sum off; one term took 186 us
// for 16 ragged requests where two take 193).
#include "paged_parts.h"

namespace {

constexpr int kWaves = 4;
constexpr int kMaxGroups = 256;    // workgroups: one a compute unit

// Tiles of a share, and what a row counts for, at least. (Four, a tile a wave: a request of 8191 rows 10.2 us
// where two took 8.2, with no cost of rows.)
constexpr int kMinTiles = 2;

// What a part of a row costs beside its tiles (query, page numbers, first loads, output: 10000 cycles, a tile 6000), in tiles of a
// share of four waves, and of one. A row counts for so many more, so that a share with several parts has fewer tiles: without
// that, those ended last (1712 rows of 0 to 612 8-bit keys 91 us, 78 with it; 528 of 1 to 1985 with float32 queries 74 and 63;
// 2 of 37000 with float32 queries 23.8 and 20.8; 16 of 0 to 2000 keys 14.8 and 11.3). No more than a share, which costs and
// tiles then fill about evenly (with half a share, 512 rows of 1 to 300 keys 30 us instead of 27.5).
constexpr int kGroupCost = 8, kWaveCost = 2;

// Rows of tiles from which on waves take shares of their own. Shares of workgroups and of waves, in us: 2 rows of 8191 keys
// 12.2 and 16.1; of 8-bit rows, 80 of 0 to 300 keys 12.1 and 14.2, of 0 to 4000 27.2 and 32.8; 126 of these 16.9 and 14.9, 36.4
// and 38.0; 240 of them 19.3 and 16.3, 59.9 and 59.2; 500 of them 30.6 and 22.4, 107.3 and 106.7.
constexpr int kManyRows = 128;

// What the first loads take comes as plain arguments, which are in registers when a wave starts; the rest is loaded under them.
struct PagedRest {
  const void* q;            // [B, Hq, D]
  const int32_t* requests;  // [B], the table of a query; null: its own place
  const void *k_scales, *k_biases, *v_scales, *v_biases;
  int n_tables;
  float scale_log2;
  float* ws_o;    // partial outputs [2 shares][rep][256]: of the row that a share ends (2 w) and that it begins (2 w + 1)
  float* ws_ml;   // their statistics [2 shares][16][2]
  int32_t* cut;   // {row, its first share, its last share} of a row that was cut, row -1 of none: by row where there are no
                  // more of them than shares, else by the share that begins the row
  void* out;      // [B, Hq, D]; or, where other keys of the same queries are joined with these,
  float* own;     // [B * n_kv * rep][256] sums, relative to their reference maximum, of rows that are not cut (else null)
  float* own_ml;  // [B * n_kv * rep][2]
};

struct PagedArgs {
  const int32_t* lens;    // [B]
  const int32_t* tables;  // [n_tables, width]
  const void *k, *v;
  int batch, n_kv, rep, width, n_pages, page_shift;
  PagedRest rest;
};

// Tiles that a row of `len` keys counts for.
__device__ __forceinline__ int tiles_of(int len) {
  const int t = (len + kTileKeys - 1) / kTileKeys;
  return t < kMinTiles ? kMinTiles : t;
}

struct Place {
  int b, kvh, tile, len;  // request, KV head, tile of its row, keys
};

constexpr int kNearInts = kWaves * 2 * MSPR_WAVE;  // what every wave knows of the first chunks' lengths

// LDS of a workgroup: the waves' V tiles (or what they exchange at the end) and the query operands, of all or of each.
__host__ __device__ constexpr int loop_lds(int qdt, int fmt, bool alone) {
  const int tiles = kWaves * kVTileBytes;
  const int query = 8 * 64 * 16 * (fmt == kAffine && qdt == MSPR_F32 ? 2 : 1) * (alone ? kWaves : 1);
  return tiles + query;
}
static_assert(kWaves * kVTileBytes >= (kWaves * 16 * 64 * 4 + kWaves * 16 * 2) * 4, "the exchange fits into the V tiles");

// QDT: type of queries and output; FMT: page format; SDT: type of scales and biases (8-bit pages); ALONE: a share a wave
// One workgroup a CU: with two, and half the share each, 16-bit rows took 100 us instead of 95 (8 requests of 37000 rows) and
// 168 instead of 157 (64 ragged ones). The forms that fit 256 registers are held to them: beyond, values move to and from
// accumulation registers (16 ragged requests of 8-bit rows 204 us instead of 193); the others would spill (104 instead of 95).
template <int QDT, int FMT, int SDT, bool ALONE>
__global__ __launch_bounds__(64 * kWaves, FMT == kAffine && QDT != MSPR_F32 ? 2 : 1) void paged_decode_kernel(
    const int32_t* lens, const int32_t* tables, const void* k, const void* v, int batch, int n_kv, int width, int page_shift,
    int n_pages, int rep, PagedRest a) {
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  constexpr bool kCodes = FMT == kAffine;
  // Operands of the second product: of 8-bit rows float16, in which the codes cost fewest instructions and a term of a weight
  // has eleven digits (three terms of bfloat16 are as exact; 66 requests of 1 to 1985 keys with float32 queries took 79 us with
  // them, 73 with these).
  constexpr int kVType = kCodes ? MSPR_F16 : FMT;
  constexpr int kPTerms = 2;                                   // terms of a weight
  constexpr int kQTerms = kCodes && QDT == MSPR_F32 ? 2 : 1;  // terms of a query element
  // float16 weights are taken 2^11 times as large: up to 2^15, as the reference maximum lags by 2^4 at most, and the smallest
  // that is not lost is 2^-35 of the largest (at 2^-24, the many small weights of a long context would all be rounded one way)
  constexpr float kLag = 4.0f;
  constexpr float kUp = kVType == MSPR_F16 ? 11.0f : 0.0f;
  constexpr int kRowBytes = kCodes ? kD : kD * 2;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  static_assert(kWaves == 4, "with a share a workgroup, a wave makes the query operands of a quarter of the channels");
  constexpr int kShares = ALONE ? kMaxGroups * kWaves : kMaxGroups;
  constexpr int kStride = ALONE ? 1 : kWaves;                  // tiles from one of a wave's to its next
  constexpr int kSteps = ALONE ? 8 : 8 / kWaves;               // of the query operand, made by a wave
  const int step0 = ALONE ? 0 : kSteps * wave;
  const int first_tile = ALONE ? 0 : wave;                     // of a share
  const int n = lane & 15;  // MFMA column: query head of the group; row (key) of the K operand
  const int g = lane >> 4;
  unsigned char* vt = lds + wave * kVTileBytes;

  const int cap = width << page_shift;
  const int page_mask = (1 << page_shift) - 1;

  // ---- the share: every wave adds up all tiles for itself, of more than 64 queries the four together, a chunk of 64 at a time
  const int chunks = (batch + MSPR_WAVE - 1) / MSPR_WAVE;
  int* near = reinterpret_cast<int*>(lds + loop_lds(QDT, FMT, ALONE));  // lengths and sums of the first four: [4][2][64]
  int* chunk_sums = near + kNearInts;                                   // [chunks]
  auto tiles_at = [&](int i, int& len) {
    len = length_of(lens, batch, i, cap);
    return i < batch ? tiles_of(len) : 0;
  };
  Place at = {0, 0, 0, 0};
  int chunk = chunks == 1 ? 0 : wave, all = 0, before = 0, len0, tiles0 = tiles_at(chunk * MSPR_WAVE + lane, len0);
  int sums0 = wave_scan(tiles0);
  int chunk_sum = 0, in_lanes = 0, per_lane = 1;  // (of more chunks than one: lane i has the sum of `per_lane`, and those before)
  if (chunks == 1) {
    all = __builtin_amdgcn_readlane(sums0, 63);
  } else {
    near[2 * MSPR_WAVE * wave + lane] = len0;
    near[2 * MSPR_WAVE * wave + MSPR_WAVE + lane] = sums0;
    if (lane == 63 && wave < chunks) chunk_sums[wave] = sums0;
    for (int c = wave + kWaves; c < chunks; c += kWaves) {
      int len;
      const int sum = wave_scan(tiles_at(c * MSPR_WAVE + lane, len));
      if (lane == 63) chunk_sums[c] = sum;
    }
    __syncthreads();
    per_lane = (chunks + MSPR_WAVE - 1) / MSPR_WAVE;
    for (int c = lane * per_lane; c < min((lane + 1) * per_lane, chunks); c++) chunk_sum += chunk_sums[c];
    in_lanes = wave_scan(chunk_sum);
    all = __builtin_amdgcn_readlane(in_lanes, 63);
  }
  all *= n_kv;
  // (none where no row is longer than the smallest share: none is cut then, and the second kernel is not launched)
  const int cost = cap <= kMinTiles * kTileKeys ? 0 : min(ALONE ? kWaveCost : kGroupCost, (all + kShares - 1) / kShares);
  all += cost * n_kv * batch;
  int share = (all + kShares - 1) / kShares;
  share = share < kMinTiles ? kMinTiles : share;
  // Number of the share. Up to two a workgroup, waves' shares go round the workgroups, to be on as many compute units as can be
  // (64 requests of 1 to 300 keys 17.1 -> 14.3 us); more go to a workgroup one behind the other (64 ragged ones of up to 16384
  // keys 161.7 -> 159.7).
  const int number = !ALONE                                          ? (int)blockIdx.x
                     : all <= kMinTiles * kMaxGroups * (kWaves / 2) ? (int)(blockIdx.x + gridDim.x * wave)
                                                                     : (int)blockIdx.x * kWaves + wave;
  int pos = number * share;
  const int end = min(pos + share, all);
  const bool by_row = !ALONE || batch * n_kv <= kShares;
  static_assert(kManyRows <= kMaxGroups, "with a share a workgroup there are fewer rows than shares");
  if (!by_row && lane == 0) a.cut[3 * number] = -1;
  if (pos >= end) return;
  // (Whose tile `pos` is: it is below the total, so that there is one. Lengths that another stream changes meanwhile may say
  // otherwise: every loop ends and every index stays in its range all the same.)
  auto first_beyond = [&](int sum) {
    const uint64_t beyond = __ballot(sum * n_kv > pos);
    return beyond ? __builtin_ctzll(beyond) : MSPR_WAVE - 1;
  };
  if (chunks > 1) {
    const int i = first_beyond(in_lanes + cost * min((lane + 1) * per_lane * MSPR_WAVE, batch));
    before = __builtin_amdgcn_readlane(in_lanes, i) - __builtin_amdgcn_readlane(chunk_sum, i);
    chunk = min(i * per_lane, chunks - 1);
    before += cost * chunk * MSPR_WAVE;
    for (; chunk < chunks - 1; chunk++) {
      const int sum = __builtin_amdgcn_readfirstlane(chunk_sums[chunk]) + cost * MSPR_WAVE;
      if ((before + sum) * n_kv > pos) break;
      before += sum;
    }
    if (chunk < kWaves) {
      len0 = near[2 * MSPR_WAVE * chunk + lane];
      sums0 = near[2 * MSPR_WAVE * chunk + MSPR_WAVE + lane];
      tiles0 = tiles_of(len0);
    } else {
      tiles0 = tiles_at(chunk * MSPR_WAVE + lane, len0);
      sums0 = wave_scan(tiles0);
    }
  }
  {
    sums0 += cost * min(lane + 1, batch - chunk * MSPR_WAVE);
    const int i = first_beyond(before + sums0);
    const int t = __builtin_amdgcn_readlane(tiles0, i) + cost;
    at.b = chunk * MSPR_WAVE + i;
    at.len = __builtin_amdgcn_readlane(len0, i);
    at.tile = pos - (before + __builtin_amdgcn_readlane(sums0, i) - t) * n_kv;
    while (at.tile >= t && at.kvh < n_kv - 1) {
      at.tile -= t;
      at.kvh++;
    }
    if (at.b >= batch) return;
  }

  auto go_on = [&](int by) {  // to the next row, if the share reaches it
    pos += by;
    if (pos >= end) return false;
    at.tile = 0;
    if (++at.kvh < n_kv) return true;
    at.kvh = 0;
    if (++at.b >= batch) return false;
    at.len = __builtin_amdgcn_readfirstlane(length_of(lens, batch, at.b, cap));
    return true;
  };
  for (;;) {
    const int row_tiles = tiles_of(at.len);
    const int tile0 = at.tile;
    if (tile0 >= row_tiles) {  // (a share may begin in a row's cost, which lies behind its tiles)
      if (!go_on(row_tiles + cost - tile0)) return;
      continue;
    }
    const int tile1 = min(tile0 + (end - pos), row_tiles);

    // ---- the query is asked for first: loads come back in order, and the pages' addresses wait for the table anyway
    const bool mine = n < rep;
    constexpr int kQWords = QDT == MSPR_F32 ? 2 : 1;  // of sixteen bytes a step
    u32x4_t qraw[kSteps * kQWords];
    {
      const int64_t q0 = (((int64_t)at.b * n_kv + at.kvh) * rep + (mine ? n : 0)) * kD;
#pragma unroll
      for (int i = 0; i < kSteps; i++) {
        // step s: channels 32 s + 8 g on, of 8-bit rows 64 (s / 2) + 16 g + 8 (s % 2) on
        const int channel = kCodes ? 32 * (step0 + i & ~1) + 16 * g + 8 * (i & 1) : 32 * (step0 + i) + 8 * g;
        constexpr int kQBytes = QDT == MSPR_F32 ? 4 : 2;
        const u32x4_t* p = reinterpret_cast<const u32x4_t*>(reinterpret_cast<const uint8_t*>(a.q) + (q0 + channel) * kQBytes);
#pragma unroll
        for (int j = 0; j < kQWords; j++) qraw[i * kQWords + j] = p[j];
      }
    }
    __builtin_amdgcn_sched_barrier(0);

    const int request = a.requests ? __builtin_amdgcn_readfirstlane(a.requests[at.b]) : at.b;
    const bool known = request >= 0 && (!a.requests || request < a.n_tables);
    const int len = known ? at.len : 0;
    const int32_t* table = tables + (int64_t)(known ? request : 0) * width;
    const int last_tile = min(tile1, (len + kTileKeys - 1) / kTileKeys);

    f32x4_t oacc[16];
#pragma unroll
    for (int mt = 0; mt < 16; mt++) oacc[mt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    auto rescale = [&](float by) {
#pragma unroll
      for (int mt = 0; mt < 16; mt++) oacc[mt] = oacc[mt] * by;
    };
    float m_run = -__builtin_inff(), l_run = 0.0f;
    f32x4_t bacc = {0.f, 0.f, 0.f, 0.f};  // weighted biases: lane n (g = 0) has those of head n and the four groups
    // what V's scales of group n % 4 are multiples of: a power of two from their largest magnitude on. (A group's own: weights
    // end at 2^-36 of it, and one for all four cost a group whose scales are 10^-6 of another's all but 2^-12 of its results.)
    float v_unit = 0x1p-126f;

    // Pages of this wave's tiles, two half tiles of 16 keys each (a page holds 16 rows or more): lane i of `ids` has the page
    // of half tile i of 31 tiles and the one behind them, the next tiles' are on their way while these are used.
    const int n_mine = last_tile - tile0 > first_tile ? (last_tile - tile0 - first_tile + kStride - 1) / kStride : 0;
    auto load_ids = [&](int it0) {
      const int it = it0 + (lane >> 1);
      const int key = (tile0 + first_tile + kStride * it) * kTileKeys + 16 * (lane & 1);
      const int e = it < n_mine && key < len ? key >> page_shift : -1;
      return e >= 0 ? table[e] : -1;
    };

    // A half tile: its page's rows, and how many of them count (none of a page that is not in the pool).
    struct Half {
      int64_t row;  // first row in the pages
      int rows;
    };
    auto half_at = [&](int ids, int it0, int it, int u) {
      const int key = (tile0 + first_tile + kStride * it) * kTileKeys + 16 * u;
      const int p = __builtin_amdgcn_readlane(ids, 2 * (it - it0) + u);
      const bool good = p >= 0 && p < n_pages;
      Half h;
      h.row = ((((int64_t)(good ? p : 0) * n_kv + at.kvh) << page_shift) + (key & page_mask));
      // (a scalar by hand: the compiler clamps with a vector instruction, and then takes the window for one of each lane's)
      h.rows = __builtin_amdgcn_readfirstlane(!good || it >= n_mine ? 0 : len - key >= 16 ? 16 : len - key < 0 ? 0 : len - key);
      return h;
    };

    constexpr int kKLoads = kCodes ? 4 : 8;   // 16-byte pieces a lane and half tile
    constexpr int kVLoads = kCodes ? 4 : 8;
    u32x4_t kr[2][kKLoads], vr[2][kVLoads];
    RowScales<SDT> ks[2], kb[2], vs[2], vb[2];
    auto load_k = [&](const Half* h) {
#pragma unroll
      for (int u = 0; u < 2; u++) {
        const auto w = rows_window(k, h[u].row, kRowBytes, h[u].rows);
#pragma unroll
        for (int j = 0; j < kKLoads; j++) kr[u][j] = window_load16(w, n * kRowBytes + 16 * g, 64 * j);
        if constexpr (kCodes) {
          // (scales: row 4 g + n / 4, group n % 4, to be spread over a row's sixteen lanes; biases: row n, group g, an operand)
          ks[u].load(rows_window(a.k_scales, h[u].row, 4 * RowScales<SDT>::kBytes, h[u].rows), 16 * g + n);
          kb[u].load(rows_window(a.k_biases, h[u].row, 4 * RowScales<SDT>::kBytes, h[u].rows), 4 * n + g);
        }
      }
    };
    auto load_v = [&](const Half* h) {
#pragma unroll
      for (int u = 0; u < 2; u++) {
        const auto w = rows_window(v, h[u].row, kRowBytes, h[u].rows);
#pragma unroll
        for (int j = 0; j < kVLoads; j++) vr[u][j] = window_load16(w, 16 * lane, 1024 * j);
      }
    };
    auto load_v_scales = [&](const Half* h) {
#pragma unroll
      for (int u = 0; u < 2; u++) {
        vs[u].load(rows_window(a.v_scales, h[u].row, 4 * RowScales<SDT>::kBytes, h[u].rows), 16 * g + n);
        vb[u].load(rows_window(a.v_biases, h[u].row, 4 * RowScales<SDT>::kBytes, h[u].rows), 16 * g + n);
      }
    };

    int ids = load_ids(0);
    Half cur[2] = {half_at(ids, 0, 0, 0), half_at(ids, 0, 0, 1)}, nxt[2];
    load_k(cur);
    load_v(cur);
    if constexpr (kCodes) load_v_scales(cur);
    int ids_next = load_ids(31);
    __builtin_amdgcn_sched_barrier(0);  // the first tile is on its way before the query is fetched

    // ---- Q^T operand, in LDS (for all waves, or the one): lane (n = head, g) has the eight channels that the K operand has
    //      in its place
    u32x4_t* qt = reinterpret_cast<u32x4_t*>(lds + kWaves * kVTileBytes) + lane;  // [8 steps][terms][64 lanes]
    if constexpr (ALONE) qt += wave * (8 * kQTerms * 64);
    float q_unit = a.scale_log2;           // what a product's unit stands for, in powers of two
    float qsum = 0.0f;                     // sum of the query's head n over group g
    if constexpr (!kCodes) {
#pragma unroll
      for (int i = 0; i < kSteps; i++) qt[64 * (step0 + i)] = mine ? qraw[i] : u32x4_t{0u, 0u, 0u, 0u};
    } else {
      auto element = [&](int i, float* x) {
        if constexpr (QDT == MSPR_F32) {
#pragma unroll
          for (int j = 0; j < 8; j++) x[j] = __uint_as_float(qraw[2 * i + j / 4][j % 4]);
        } else {
          widen8<QDT>(qraw[i], x);
        }
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = mine ? x[j] : 0.0f;
      };
      // The operand is float16: a power of two brings the head's largest element to [2^14, 2^15), so that what falls below
      // float16's range is 2^-39 of it; float16 queries go in as they are.
      float* shared = reinterpret_cast<float*>(lds);  // [2][waves][16 heads], where the V tiles will be
      int e = 0;
      if constexpr (QDT != MSPR_F16) {
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < kSteps; i++) {
          float x[8];
          element(i, x);
#pragma unroll
          for (int j = 0; j < 8; j++) top = fmaxf(top, fabsf(x[j]));
        }
        top = half_wave_max(row_pair_max(top));
        if constexpr (!ALONE) {
          if (g == 0) shared[16 * wave + n] = top;
          __syncthreads();
#pragma unroll
          for (int w = 0; w < kWaves; w++) top = fmaxf(top, shared[16 * w + n]);
        }
        if (top > 0.0f && top < __builtin_inff()) e = __builtin_amdgcn_frexp_expf(top) - 15;
      }
      float sums[kSteps / 2] = {};  // by group
#pragma unroll
      for (int i = 0; i < kSteps; i++) {
        float x[8];
        element(i, x);
#pragma unroll
        for (int j = 0; j < 8; j++) {
          x[j] = __builtin_amdgcn_ldexpf(x[j], -e);
        }
        u32x4_t terms[kQTerms];
        split_terms<MSPR_F16, kQTerms>(x, terms);
        // (of the terms, as the products are: what the two have too little is then multiplied with a value, not with its code)
#pragma unroll
        for (int t = 0; t < kQTerms; t++) {
          float y[8];
          widen8<MSPR_F16>(terms[t], y);
#pragma unroll
          for (int j = 0; j < 8; j++) sums[i / 2] += y[j];
        }
#pragma unroll
        for (int t = 0; t < kQTerms; t++) qt[64 * ((step0 + i) * kQTerms + t)] = terms[t];
      }
      q_unit = __builtin_amdgcn_ldexpf(q_unit, e);
#pragma unroll
      for (int j = 0; j < kSteps / 2; j++) {
        sums[j] += __shfl_xor(sums[j], 16, MSPR_WAVE);
        sums[j] += __shfl_xor(sums[j], 32, MSPR_WAVE);
      }
      if constexpr (ALONE) {
        qsum = g == 0 ? sums[0] : g == 1 ? sums[kSteps / 2 - 3] : g == 2 ? sums[kSteps / 2 - 2] : sums[kSteps / 2 - 1];
      } else {
        if (g == 0) shared[64 + 16 * wave + n] = sums[0];
        __syncthreads();
        qsum = shared[64 + 16 * g + n];
      }
    }
    if constexpr (ALONE) __builtin_amdgcn_wave_barrier();
    else __syncthreads();

    const int tr_off = (4 * g + ((lane & 15) >> 2)) * kVPitch + 4 * (lane & 3) * 2;
    for (int it0 = 0; it0 < n_mine; it0 += 31) {  // (a loop of its own, so that only its head waits for pages)
      const int it_end = min(it0 + 31, n_mine);
      for (int it = it0; it < it_end; it++) {
        // the next tile (behind the last, one that has no rows: what is outstanding does not depend on the tile)
        nxt[0] = half_at(ids, it0, it + 1, 0);
        nxt[1] = half_at(ids, it0, it + 1, 1);

        // ---- S^T = K . Q^T
        float s[8];  // key 16 u + 4 g + i at 4 u + i
#pragma unroll
        for (int u = 0; u < 2; u++) {
          if constexpr (!kCodes) {
            f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < 8; j++) acc = mfma<FMT>(kr[u][j], qt[64 * j], acc);
#pragma unroll
            for (int i = 0; i < 4; i++) s[4 * u + i] = acc[i] * q_unit;
          } else {
            const f32x4_t zero = {0.f, 0.f, 0.f, 0.f};
            const float ksf = ks[u].value(n);
            const float of_bias = __int_as_float(__builtin_amdgcn_ds_bpermute(4 * (4 * n + g), __float_as_int(ksf)));
            f32x4_t sum = __builtin_amdgcn_mfma_f32_16x16x4f32(fmaf(128.0f, of_bias, kb[u].value(g)), qsum, zero, 0, 0, 0);
            static_for<4>([&](auto jc) {
              constexpr int j = decltype(jc)::value;
              f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int h = 0; h < 2; h++) {
                u32x4_t c;
#pragma unroll
                for (int w = 0; w < 2; w++) {
                  h2_t lo, hi;
                  centred_to_h(kr[u][j][2 * h + w], lo, hi);
                  c[2 * w] = h2_bits(lo);
                  c[2 * w + 1] = h2_bits(hi);
                }
#pragma unroll
                for (int t = 0; t < kQTerms; t++) acc = mfma<MSPR_F16>(c, qt[64 * ((2 * j + h) * kQTerms + t)], acc);
              }
              static_for<4>([&](auto ic) {
                constexpr int i = decltype(ic)::value;
                sum[i] = fmaf(of_lane<4 * i + j>(ksf), acc[i], sum[i]);
              });
            });
#pragma unroll
            for (int i = 0; i < 4; i++) s[4 * u + i] = sum[i] * q_unit;
          }
        }
        load_k(nxt);
        __builtin_amdgcn_sched_barrier(0);

        // ---- online softmax (powers of two), the reference maximum moves only past 2^4
        float tmax = -__builtin_inff();
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            if (4 * g + i >= cur[u].rows) s[4 * u + i] = -__builtin_inff();
            tmax = fmaxf(tmax, s[4 * u + i]);
          }
        tmax = half_wave_max(row_pair_max(tmax));
        const bool grow = tmax > m_run + kLag;
        if (__any(grow)) {
          const float m_new = grow ? tmax : m_run;
          if (it > 0) {  // (sums of nothing need no new scale)
            const float alpha = grow ? __builtin_amdgcn_exp2f(m_run - m_new) : 1.0f;
            l_run *= alpha;
            rescale(alpha);
            bacc = bacc * alpha;
          }
          m_run = m_new;
        }
        const float m_safe = (m_run == -__builtin_inff() ? 0.0f : m_run) - kUp;
#pragma unroll
        for (int i = 0; i < 8; i++) {
          s[i] = __builtin_amdgcn_exp2f(s[i] - m_safe);
          l_run += s[i];
        }

        // ---- V rows to LDS (zeros in the place of rows that do not count, so that what lies there meets no weight of zero)
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
          for (int j = 0; j < kVLoads; j++) {
            if constexpr (!kCodes) {
              *reinterpret_cast<u32x4_t*>(vt + (16 * u + 2 * j + (lane >> 5)) * kVPitch + 16 * (lane & 31)) = vr[u][j];
            } else {
              u32x4_t lo, hi;
#pragma unroll
              for (int w = 0; w < 4; w++) {
                h2_t c01, c23;
                centred_to_h(vr[u][j][w], c01, c23);
                (w < 2 ? lo : hi)[2 * (w & 1)] = h2_bits(c01);
                (w < 2 ? lo : hi)[2 * (w & 1) + 1] = h2_bits(c23);
              }
              unsigned char* d = vt + (16 * u + 4 * j + (lane >> 4)) * kVPitch + 32 * (lane & 15);
              *reinterpret_cast<u32x4_t*>(d) = lo;
              *reinterpret_cast<u32x4_t*>(d + 16) = hi;
            }
          }
        load_v(nxt);
        cur[0] = nxt[0];
        cur[1] = nxt[1];
        __builtin_amdgcn_sched_barrier(0);

        // ---- O^T += V^T . P^T (the tile was written by this wave only: LDS operations of one wave complete in order, the wave
        //      barrier keeps the compiler from moving the reads up)
        __builtin_amdgcn_wave_barrier();
        // (operands of four tiles of channels are read while the four before are multiplied)
        u32x4_t vf[2][4];
        auto read_v = [&](int q4) {
#pragma unroll
          for (int m = 0; m < 4; m++) {
            const unsigned char* base = vt + tr_off + (4 * q4 + m) * 32;
            const u32x2_t lo = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(MSPR_LDS_PTR(s16x4_t, base)));
            const u32x2_t hi =
                __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(MSPR_LDS_PTR(s16x4_t, base + 16 * kVPitch)));
            vf[q4 & 1][m] = u32x4_t{lo.x, lo.y, hi.x, hi.y};
          }
        };
        auto accumulate = [&](int q4, const u32x4_t* pf) {
          if (q4 < 3) read_v(q4 + 1);
#pragma unroll
          for (int t = 0; t < kPTerms; t++)
#pragma unroll
            for (int m = 0; m < 4; m++) oacc[4 * q4 + m] = mfma<kVType>(vf[q4 & 1][m], pf[t], oacc[4 * q4 + m]);
        };
        read_v(0);
        u32x4_t pf[kPTerms];
        if constexpr (!kCodes) {
          split_terms<kVType, kPTerms>(s, pf);
#pragma unroll
          for (int q4 = 0; q4 < 4; q4++) accumulate(q4, pf);
        } else {
          // The operand is float16: scales are taken as multiples of a power of two that is as large as any of their group.
          float vsf[2] = {vs[0].value(n), vs[1].value(n)};
          const float largest = fmaxf(fabsf(vsf[0]), fabsf(vsf[1]));
          if (__any(largest > v_unit)) {
            float top = largest;
            top = fmaxf(top, lane_xor<4>(top));
            top = fmaxf(top, lane_xor<8>(top));
            top = half_wave_max(row_pair_max(top));
            const int e = top < 0x1p126f ? __builtin_amdgcn_frexp_expf(top) : 126;
            const float unit = top > v_unit ? __builtin_amdgcn_ldexpf(1.0f, e) : v_unit;
            if (it > 0) {
              const float by = v_unit / unit;
              static_for<16>([&](auto mt) { oacc[mt] = oacc[mt] * of_lane<decltype(mt)::value / 4>(by); });
            }
            v_unit = unit;
          }
          const float per_unit = 1.0f / v_unit;
          vsf[0] *= per_unit;
          vsf[1] *= per_unit;
          // biases: operand row m has group m of key 16 u + 4 g + i (rows from 4 on are not used)
          const float vbf[2] = {fmaf(128.0f, vs[0].value(n), vb[0].value(n)), fmaf(128.0f, vs[1].value(n), vb[1].value(n))};
          static_for<8>([&](auto ic) {
            constexpr int i = decltype(ic)::value;
            float b = vbf[i >> 2];
            if constexpr ((i & 3) != 0)
              b = __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(b), 0x100 + 4 * (i & 3), 0xF, 0xF, true));  // row_shl
            bacc = __builtin_amdgcn_mfma_f32_16x16x4f32(b, s[i], bacc, 0, 0, 0);
          });
          static_for<4>([&](auto jc) {  // the weights of group j, which has channels 64 j on
            constexpr int j = decltype(jc)::value;
            float w[8];
            static_for<8>([&](auto ic) {
              constexpr int i = decltype(ic)::value;
              w[i] = of_lane<4 * (i & 3) + j>(vsf[i >> 2]) * s[i];
              // (a rounded product: else the compiler makes a term's operand from that and what it takes off for the rest from
              // the exact product, and where the two round apart the weight is off by a step of the first term)
              asm("" : "+v"(w[i]));
            });
            split_terms<kVType, kPTerms>(w, pf);
            accumulate(j, pf);
          });
        }
        if constexpr (kCodes) load_v_scales(nxt);
        __builtin_amdgcn_wave_barrier();
      }
      ids = ids_next;
      ids_next = load_ids(it_end + 31);
    }

    // ---- the end of a part: the wave's own, or the four waves' through LDS (the V tiles are free now)
    l_run += __shfl_xor(l_run, 16, MSPR_WAVE);
    l_run += __shfl_xor(l_run, 32, MSPR_WAVE);
    if constexpr (kCodes) {
      float bias[4];
#pragma unroll
      for (int j = 0; j < 4; j++) bias[j] = __shfl(bacc[j], n, MSPR_WAVE);
      static_for<16>([&](auto mt) { oacc[mt] = oacc[mt] * of_lane<decltype(mt)::value / 4>(v_unit) + bias[mt >> 2]; });
    }
    const bool whole = tile0 == 0 && tile1 == row_tiles;
    const int row = at.b * n_kv + at.kvh;
    const int64_t part = 2 * (int64_t)number + (tile0 == 0 ? 1 : 0);
    const auto po = store_window(a.ws_o + part * rep * kD, rep * kD * (int)sizeof(float));
    float m_all = m_run, l_all = l_run;
    auto write = [&](int mt, f32x4_t acc) {
      if (n >= rep) return;
      const int64_t at = ((int64_t)row * rep + n) * kD + 16 * mt + 4 * g;
      if (whole && a.own) *reinterpret_cast<f32x4_t*>(a.own + at) = acc;
      else if (whole) store_out<QDT>(a.out, at, acc, l_all);
      else window_store<kStoreThrough>(po, (n * kD + 16 * mt + 4 * g) * 4, __builtin_bit_cast(u32x4_t, acc));
    };
    if constexpr (ALONE) {
#pragma unroll
      for (int mt = 0; mt < 16; mt++) write(mt, oacc[mt]);
    } else {
      __syncthreads();
      float* xo = reinterpret_cast<float*>(lds);   // [waves][16 mt][64 lanes][4]
      float* xml = xo + kWaves * 16 * 64 * 4;      // [waves][16 heads][2]
#pragma unroll
      for (int mt = 0; mt < 16; mt++) *reinterpret_cast<f32x4_t*>(xo + ((wave * 16 + mt) * 64 + lane) * 4) = oacc[mt];
      if (g == 0) {
        xml[(wave * 16 + n) * 2] = m_run;
        xml[(wave * 16 + n) * 2 + 1] = l_run;
      }
      __syncthreads();
      float mw[kWaves];
#pragma unroll
      for (int w = 0; w < kWaves; w++) {
        mw[w] = xml[(w * 16 + n) * 2];
        m_all = fmaxf(m_all, mw[w]);
      }
      const float m_safe = m_all == -__builtin_inff() ? 0.0f : m_all;
      l_all = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; w++) {
        mw[w] = __builtin_amdgcn_exp2f(mw[w] - m_safe);
        l_all += xml[(w * 16 + n) * 2 + 1] * mw[w];
      }
#pragma unroll
      for (int q4 = 0; q4 < 16 / kWaves; q4++) {
        const int mt = wave * (16 / kWaves) + q4;
        f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kWaves; w++) acc += *reinterpret_cast<const f32x4_t*>(xo + ((w * 16 + mt) * 64 + lane) * 4) * mw[w];
        write(mt, acc);
      }
    }
    if (first_tile == 0 && g == 0) {
      if (!whole) *reinterpret_cast<f32x2_t*>(a.ws_ml + (part * 16 + n) * 2) = f32x2_t{m_all, l_all};
      else if (a.own && n < rep) *reinterpret_cast<f32x2_t*>(a.own_ml + ((int64_t)row * rep + n) * 2) = f32x2_t{m_all, l_all};
      if (n == 0 && tile0 == 0 && (by_row || !whole)) {
        int32_t* c = a.cut + 3 * (int64_t)(by_row ? row : number);
        c[0] = whole ? -1 : row;
        c[1] = number;
        c[2] = min(number + (row_tiles - tile1 + share - 1) / share, (int)gridDim.x * (ALONE ? kWaves : 1) - 1);
      }
    }
    if (!go_on(row_tiles + cost - tile0)) return;
    if constexpr (ALONE) __builtin_amdgcn_wave_barrier();
    else __syncthreads();
  }
}

constexpr int kAtOnce = 16;  // parts that a wave joins at a time

// A running join of parts: reference maximum, sum of weights, weighted sum of four channels a lane.
struct Join {
  float m = -__builtin_inff(), l = 0.0f;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};

  // Parts p0, p0 + step, ... (at most sixteen, below `count`) of the row whose first part is share `first`'s: all are fetched
  // at once, the statistics of the j-th by lane j, in one load.
  __device__ __forceinline__ void add(const float* ws_o, const float* ws_ml, int first, int p0, int step, int count, int rep,
                                      int hn) {
    const int lane = threadIdx.x & 63;
    const int mine = p0 + step * (lane % kAtOnce);
    f32x2_t stat = {-__builtin_inff(), 0.0f};
    if (mine < count) stat = *reinterpret_cast<const f32x2_t*>(ws_ml + (part_of(first, mine) * 16 + hn) * 2);
    f32x4_t ov[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; j++)  // (wave-uniform: parts past the end cost no load)
      if (p0 + step * j < count)
        ov[j] = *reinterpret_cast<const f32x4_t*>(ws_o + (part_of(first, p0 + step * j) * rep + hn) * kD + 4 * lane);
    float m_new = stat.x;
    m_new = fmaxf(m_new, lane_xor<1>(m_new));
    m_new = fmaxf(m_new, lane_xor<2>(m_new));
    m_new = fmaxf(m_new, lane_xor<4>(m_new));
    m_new = fmaxf(m, fmaxf(m_new, lane_xor<8>(m_new)));
    const float m_safe = m_new == -__builtin_inff() ? 0.0f : m_new;
    const float alpha = __builtin_amdgcn_exp2f(m - m_safe);
    const float w = __builtin_amdgcn_exp2f(stat.x - m_safe);
    float lw = stat.y * w;
    lw += lane_xor<1>(lw);
    lw += lane_xor<2>(lw);
    lw += lane_xor<4>(lw);
    l = l * alpha + (lw + lane_xor<8>(lw));
    o = o * alpha;
#pragma unroll
    for (int j = 0; j < kAtOnce; j++)
      if (p0 + step * j < count) o += ov[j] * __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), j));
    m = m_new;
  }
};

// A head's four channels: the result, or (with own_ml) what is joined with other keys.
template <int ODT>
__device__ __forceinline__ void store_joined(void* out, int64_t at, f32x4_t o, float m, float l, float* own_ml) {
  const int lane = threadIdx.x & 63;
  if (!own_ml) {
    store_out<ODT>(out, at + 4 * lane, o, l);
  } else {
    *reinterpret_cast<f32x4_t*>(reinterpret_cast<float*>(out) + at + 4 * lane) = o;
    if (lane == 0) *reinterpret_cast<f32x2_t*>(own_ml + at / kD * 2) = f32x2_t{m, l};
  }
}

// Parts of a row that a workgroup's waves took every WAVES-th of, joined in LDS and written by the first wave.
template <int ODT, int WAVES>
__device__ __forceinline__ void join_waves(const Join& part, float (*xo)[kD + 2], void* out, int64_t at, float* own_ml) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (lane == 0) {
    xo[wave][kD] = part.m;
    xo[wave][kD + 1] = part.l;
  }
#pragma unroll
  for (int i = 0; i < 4; i++) xo[wave][4 * lane + i] = part.o[i];
  __syncthreads();
  if (wave != 0) return;
  float m_all = -__builtin_inff();
#pragma unroll
  for (int w = 0; w < WAVES; w++) m_all = fmaxf(m_all, xo[w][kD]);
  const float m_safe = m_all == -__builtin_inff() ? 0.0f : m_all;
  float l_all = 0.0f;
  f32x4_t o_all = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int w = 0; w < WAVES; w++) {
    const float wt = __builtin_amdgcn_exp2f(xo[w][kD] - m_safe);
    l_all += xo[w][kD + 1] * wt;
#pragma unroll
    for (int i = 0; i < 4; i++) o_all[i] += xo[w][4 * lane + i] * wt;
  }
  store_joined<ODT>(out, at, o_all, m_all, l_all, own_ml);
}

// Joins the parts of one row that was cut, for one query head: eight waves take every eighth part.
// grid: (rows, query heads of a KV head)
constexpr int kMergeWaves = 8;
template <int ODT>
__global__ __launch_bounds__(64 * kMergeWaves) void paged_merge_kernel(const int32_t* cut, const float* ws_o, const float* ws_ml,
                                                                       int rep, int rows, int shares, void* out) {
  __shared__ __attribute__((aligned(16))) float xo[kMergeWaves][kD + 2];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hn = blockIdx.y;
  Cut c;
  c.load(cut, blockIdx.x, rows, shares);
  if (c.count == 0) return;
  Join join;
  for (int p0 = wave; p0 < c.count; p0 += kAtOnce * kMergeWaves)
    join.add(ws_o, ws_ml, c.first, p0, kMergeWaves, c.count, rep, hn);
  join_waves<ODT, kMergeWaves>(join, xo, out, ((int64_t)c.row * rep + hn) * kD, nullptr);
}

// The same for many rows, of which most have few parts: a wave takes an entry, and the four of a workgroup together those of
// theirs that have more than sixteen parts. (An entry and head a workgroup of eight waves, most of which found nothing to do,
// took 20 us for 1712 rows of 0 to 612 keys, 6.6 in this form.) grid: (entries / 4, query heads of a KV head)
template <int ODT>
__global__ __launch_bounds__(64 * kWaves) void paged_merge_many_kernel(const int32_t* cut, const float* ws_o, const float* ws_ml,
                                                                       int rep, int rows, int shares, unsigned entries,
                                                                       void* out, float* own_ml) {
  __shared__ __attribute__((aligned(16))) float xo[kWaves][kD + 2];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hn = blockIdx.y;
  __shared__ Cut entry[kWaves];
  Cut c = {0, 0, 0};
  const unsigned e = blockIdx.x + gridDim.x * wave;
  if (e < entries) c.load(cut, e, rows, shares);
  if ((threadIdx.x & 63) == 0) entry[wave] = c;
  if (c.count > 0 && c.count <= kAtOnce) {
    Join join;
    join.add(ws_o, ws_ml, c.first, 0, 1, c.count, rep, hn);
    store_joined<ODT>(out, ((int64_t)c.row * rep + hn) * kD, join.o, join.m, join.l, own_ml);
  }
  __syncthreads();
#pragma unroll 1
  for (int w = 0; w < kWaves; w++) {
    const int count = __builtin_amdgcn_readfirstlane(entry[w].count);
    if (count <= kAtOnce) continue;
    const int first = __builtin_amdgcn_readfirstlane(entry[w].first);
    Join join;
    for (int p0 = wave; p0 < count; p0 += kAtOnce * kWaves) join.add(ws_o, ws_ml, first, p0, kWaves, count, rep, hn);
    join_waves<ODT, kWaves>(join, xo, out, ((int64_t)__builtin_amdgcn_readfirstlane(entry[w].row) * rep + hn) * kD, own_ml);
    __syncthreads();
  }
}

int64_t row_tiles_most(int64_t cap) {
  const int64_t t = (cap + kTileKeys - 1) / kTileKeys;
  return t < kMinTiles ? kMinTiles : t;
}

bool paged_alone(int batch, int n_kv) { return (int64_t)batch * n_kv >= kManyRows; }

// Shares: no more than the tiles of full tables give, with their rows' costs (at most kMinTiles where there are too few tiles
// for all shares, as a cost is at most a share).
int paged_shares(int batch, int n_kv, int64_t cap) {
  const int most = kMaxGroups * (paged_alone(batch, n_kv) ? kWaves : 1);
  const int64_t n = (batch * n_kv * (row_tiles_most(cap) + kMinTiles) + kMinTiles - 1) / kMinTiles;
  return (int)(n < most ? n : most);
}

// Scratch: partial outputs and statistics of two rows a share, which rows were cut.
size_t paged_scratch(int batch, int n_kv, int rep, int64_t cap) {
  return (size_t)paged_shares(batch, n_kv, cap) * 2 * ((size_t)rep * kD + 32) * sizeof(float) +
         kMaxGroups * kWaves * 3 * sizeof(int32_t);
}

template <int QDT, int FMT, int SDT, bool ALONE>
int paged_launch_form(const PagedArgs& a, hipStream_t st) {
  const int64_t cap = (int64_t)a.width << a.page_shift;
  const int chunks = (a.batch + MSPR_WAVE - 1) / MSPR_WAVE;
  constexpr int kLds = loop_lds(QDT, FMT, ALONE), kMostLds = kLds + (kNearInts + 65536 / MSPR_WAVE) * (int)sizeof(int);
  const int lds = kLds + (chunks > 1 ? (kNearInts + chunks) * (int)sizeof(int) : 0);
  static bool attr_set[64] = {};  // by device
  int device = 0;
  if (hipGetDevice(&device) != hipSuccess || device < 0 || device >= 64 || !attr_set[device]) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&paged_decode_kernel<QDT, FMT, SDT, ALONE>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, kMostLds);
    if (e != hipSuccess) {
      mspr_set_error("sdpa_decode_paged: cannot reserve %d bytes of LDS: %s", kMostLds, hipGetErrorString(e));
      return MSPR_ERR_LAUNCH;
    }
    if (device >= 0 && device < 64) attr_set[device] = true;
  }
  const int shares = paged_shares(a.batch, a.n_kv, cap);
  const PagedRest& r = a.rest;
  const unsigned groups = (unsigned)(shares < kMaxGroups ? shares : kMaxGroups);
  paged_decode_kernel<QDT, FMT, SDT, ALONE><<<dim3(groups), dim3(64 * kWaves), lds, st>>>(
      a.lens, a.tables, a.k, a.v, a.batch, a.n_kv, a.width, a.page_shift, a.n_pages, a.rep, r);
  MSPR_CHECK_LAUNCH("sdpa_decode_paged");
  // (rows of kMinTiles tiles are cut only where there are more of them than shares)
  const int rows = a.batch * a.n_kv;
  const bool more = ALONE && rows > kMaxGroups * kWaves;
  if (r.own && !more) return MSPR_OK;  // (the caller joins the parts, which it finds row by row)
  if (row_tiles_most(cap) > kMinTiles || more) {
    if constexpr (ALONE) {
      const unsigned entries = (unsigned)(more ? shares : rows);
      paged_merge_many_kernel<QDT><<<dim3((entries + kWaves - 1) / kWaves, (unsigned)a.rep), dim3(64 * kWaves), 0, st>>>(
          r.cut, r.ws_o, r.ws_ml, a.rep, rows, shares, entries, r.own ? r.own : r.out, r.own_ml);
    } else {
      paged_merge_kernel<QDT><<<dim3((unsigned)rows, (unsigned)a.rep), dim3(64 * kMergeWaves), 0, st>>>(r.cut, r.ws_o, r.ws_ml, a.rep,
                                                                                                        rows, shares, r.out);
    }
    MSPR_CHECK_LAUNCH("sdpa_decode_paged (merge)");
  }
  return MSPR_OK;
}

template <int QDT, int FMT, int SDT>
int paged_launch(const PagedArgs& a, hipStream_t st) {
  if (paged_alone(a.batch, a.n_kv)) return paged_launch_form<QDT, FMT, SDT, true>(a, st);
  return paged_launch_form<QDT, FMT, SDT, false>(a, st);
}

int paged_fill(const char* what, PagedArgs& a, const void* q, const void* k, const void* v, const int32_t* tables,
               const int32_t* lens, const int32_t* requests, int batch, int n_q_heads, int n_kv_heads, int head_dim, int n_pages,
               int page_size, int n_tables, int table_width, float scale, void* out, void* workspace, size_t workspace_bytes) {
  MSPR_REQUIRE(q && k && v && tables && lens && out, "%s: null pointer", what);
  MSPR_REQUIRE(head_dim == kD, "%s: head_dim must be 256", what);
  MSPR_REQUIRE(batch >= 1 && batch <= 65535, "%s: 1 to 65535 queries", what);
  MSPR_REQUIRE(n_tables >= 1 && (requests || n_tables == batch), "%s: a table for every query, or the requests they belong to",
               what);
  MSPR_REQUIRE(n_kv_heads >= 1 && n_kv_heads <= 1024 && n_q_heads >= n_kv_heads && n_q_heads % n_kv_heads == 0,
               "%s: bad head counts", what);
  MSPR_REQUIRE(n_q_heads / n_kv_heads <= 16, "%s: at most 16 query heads per KV head", what);
  MSPR_REQUIRE(page_size >= 16 && (page_size & (page_size - 1)) == 0, "%s: page_size must be a power of two from 16 on", what);
  MSPR_REQUIRE(n_pages >= 1 && (int64_t)n_pages * page_size <= 0x7FFFFFFF, "%s: the pool must hold fewer than 2^31 tokens", what);
  MSPR_REQUIRE(table_width >= 1 && (int64_t)table_width * page_size <= 0x40000000,
               "%s: a request's table must hold 1 page or more and at most 2^30 tokens", what);
  MSPR_REQUIRE((int64_t)batch * n_kv_heads * row_tiles_most((int64_t)table_width * page_size) <= 0x3FFFFFFF,
               "%s: the tables hold too many tokens together", what);
  MSPR_REQUIRE(mspr_aligned(q, 16) && mspr_aligned(k, 16) && mspr_aligned(v, 16) && mspr_aligned(out, 16),
               "%s: pointers must be 16-byte aligned", what);
  const int rep = n_q_heads / n_kv_heads;
  const int64_t cap = (int64_t)table_width * page_size;
  const size_t need = paged_scratch(batch, n_kv_heads, rep, cap);
  MSPR_REQUIRE(workspace && workspace_bytes >= need && mspr_aligned(workspace, 16),
               "%s: workspace of %zu bytes (16-byte aligned) needed, %zu given", what, need, workspace_bytes);
  const int64_t parts = 2 * (int64_t)paged_shares(batch, n_kv_heads, cap);
  a = PagedArgs{};
  a.rest.q = q;
  a.k = k;
  a.v = v;
  a.tables = tables;
  a.lens = lens;
  a.rest.requests = requests;
  a.rest.n_tables = n_tables;
  a.batch = batch;
  a.n_kv = n_kv_heads;
  a.rep = rep;
  a.width = table_width;
  a.n_pages = n_pages;
  a.page_shift = __builtin_ctz(page_size);
  a.rest.scale_log2 = (float)((double)scale * 1.4426950408889634);
  a.rest.ws_o = reinterpret_cast<float*>(workspace);
  a.rest.ws_ml = a.rest.ws_o + parts * rep * kD;
  a.rest.cut = reinterpret_cast<int32_t*>(a.rest.ws_ml + parts * 32);
  a.rest.out = out;
  return MSPR_OK;
}

template <int QDT>
int paged_q8_launch(const PagedArgs& a, int sb_dtype, hipStream_t st) {
  if (sb_dtype == MSPR_F32) return paged_launch<QDT, kAffine, MSPR_F32>(a, st);
  if (sb_dtype == MSPR_F16) return paged_launch<QDT, kAffine, MSPR_F16>(a, st);
  return paged_launch<QDT, kAffine, MSPR_BF16>(a, st);
}

// The entry points' launches, of 16-bit rows and of 8-bit ones.
int rows_launch(const PagedArgs& a, int dtype, hipStream_t st) {
  if (dtype == MSPR_F16) return paged_launch<MSPR_F16, MSPR_F16, MSPR_F16>(a, st);
  return paged_launch<MSPR_BF16, MSPR_BF16, MSPR_BF16>(a, st);
}
int codes_launch(const PagedArgs& a, int q_dtype, int sb_dtype, hipStream_t st) {
  if (q_dtype == MSPR_F32) return paged_q8_launch<MSPR_F32>(a, sb_dtype, st);
  if (q_dtype == MSPR_F16) return paged_q8_launch<MSPR_F16>(a, sb_dtype, st);
  return paged_q8_launch<MSPR_BF16>(a, sb_dtype, st);
}

}  // namespace

int mspr_paged_decode_parts(const char* what, const PagedPartsCall& c, PagedParts* parts, hipStream_t st) {
  PagedArgs a;
  if (int rc = paged_fill(what, a, c.q, c.k, c.v, c.tables, c.lens, c.requests, c.batch, c.rep * c.n_kv, c.n_kv, kD, c.n_pages,
                          1 << c.page_shift, c.n_tables, c.width, 1.0f, c.own, c.workspace, c.workspace_bytes))
    return rc;
  a.rest.scale_log2 = c.scale_log2;
  a.rest.k_scales = c.k_scales;
  a.rest.k_biases = c.k_biases;
  a.rest.v_scales = c.v_scales;
  a.rest.v_biases = c.v_biases;
  a.rest.own = c.own;
  a.rest.own_ml = c.own_ml;
  const int rows = c.batch * c.n_kv;
  const int64_t cap = (int64_t)c.width << c.page_shift;
  // (of more rows than shares parts are not found row by row, and have been joined; of rows that are never cut there are none)
  const bool joined = paged_alone(c.batch, c.n_kv) ? rows > kMaxGroups * kWaves : false;
  parts->cut = joined || row_tiles_most(cap) <= kMinTiles ? nullptr : a.rest.cut;
  parts->o = a.rest.ws_o;
  parts->ml = a.rest.ws_ml;
  parts->shares = paged_shares(c.batch, c.n_kv, cap);
  if (c.k_scales) return codes_launch(a, c.q_dtype, c.sb_dtype, st);
  return rows_launch(a, c.q_dtype, st);
}

extern "C" size_t mspr_sdpa_decode_paged_workspace_bytes(int batch, int n_q_heads, int n_kv_heads, int page_size,
                                                         int table_width) {
  if (batch < 1 || n_kv_heads < 1 || n_q_heads < n_kv_heads || page_size < 1 || table_width < 1) return 0;
  return paged_scratch(batch, n_kv_heads, n_q_heads / n_kv_heads, (int64_t)page_size * table_width);
}

extern "C" int mspr_sdpa_decode_paged(const void* queries, const void* k_pages, const void* v_pages, int dtype,
                                      const int32_t* tables, const int32_t* lens, const int32_t* requests, int batch,
                                      int n_q_heads, int n_kv_heads, int head_dim, int n_pages, int page_size, int n_tables,
                                      int table_width, float scale, void* out, void* workspace, size_t workspace_bytes,
                                      void* stream) {
  MSPR_REQUIRE(dtype == MSPR_F16 || dtype == MSPR_BF16, "sdpa_decode_paged: dtype must be f16 or bf16");
  PagedArgs a;
  if (int rc = paged_fill("sdpa_decode_paged", a, queries, k_pages, v_pages, tables, lens, requests, batch, n_q_heads, n_kv_heads,
                          head_dim, n_pages, page_size, n_tables, table_width, scale, out, workspace, workspace_bytes))
    return rc;
  return rows_launch(a, dtype, (hipStream_t)stream);
}

extern "C" int mspr_sdpa_decode_paged_q8(const void* queries, int q_dtype, const void* k_wq, const void* k_scales,
                                         const void* k_biases, const void* v_wq, const void* v_scales, const void* v_biases,
                                         int sb_dtype, const int32_t* tables, const int32_t* lens, const int32_t* requests,
                                         int batch, int n_q_heads, int n_kv_heads, int head_dim, int n_pages, int page_size,
                                         int n_tables, int table_width, float scale, int group_size, int bits, void* out,
                                         void* workspace, size_t workspace_bytes, void* stream) {
  MSPR_REQUIRE(group_size == 64 && bits == 8, "sdpa_decode_paged_q8: only group_size=64, bits=8 is supported");
  MSPR_REQUIRE(q_dtype >= MSPR_F32 && q_dtype <= MSPR_BF16, "sdpa_decode_paged_q8: queries must be f32, f16 or bf16");
  MSPR_REQUIRE(sb_dtype >= MSPR_F32 && sb_dtype <= MSPR_BF16, "sdpa_decode_paged_q8: scales must be f32, f16 or bf16");
  MSPR_REQUIRE(k_scales && k_biases && v_scales && v_biases, "sdpa_decode_paged_q8: null pointer");
  MSPR_REQUIRE(mspr_aligned(k_scales, 16) && mspr_aligned(k_biases, 16) && mspr_aligned(v_scales, 16) &&
                   mspr_aligned(v_biases, 16),
               "sdpa_decode_paged_q8: pointers must be 16-byte aligned");
  PagedArgs a;
  if (int rc = paged_fill("sdpa_decode_paged_q8", a, queries, k_wq, v_wq, tables, lens, requests, batch, n_q_heads, n_kv_heads,
                          head_dim, n_pages, page_size, n_tables, table_width, scale, out, workspace, workspace_bytes))
    return rc;
  a.rest.k_scales = k_scales;
  a.rest.k_biases = k_biases;
  a.rest.v_scales = v_scales;
  a.rest.v_biases = v_biases;
  return codes_launch(a, q_dtype, sb_dtype, (hipStream_t)stream);
}
