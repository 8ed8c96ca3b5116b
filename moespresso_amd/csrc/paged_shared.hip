// Attention of new tokens over a paged KV cache in which groups of requests share a prefix.
//
//   out[r, h] = sum_k softmax_k(q[r, h] . K[k] * scale) V[k]   over the rows of the prefix that the query's request continues,
//                                                              then the first lens[r] rows of the request's own table
//
// Pages, head dim and arithmetic are those of paged_decode.hip (16-bit rows, or affine 8-bit rows in groups of 64; S^T = K.Q^T
// and O^T = V^T.P^T by 16x16x32 matrix instructions, an online softmax a wave, weights in two terms). What differs: a wave
// multiplies a tile of 32 keys, once it is in registers, with up to 32 columns, the query heads of several members of a group.
//
// Work is cut into pieces: a block of a prefix's members, or a query's own rows, of one KV head, over a range of tiles. Every
// workgroup plans for itself (lengths and groups are known on the device only): a range's length follows from all tiles there are,
// so that a piece falls to every compute unit; the number of a piece says what it is. Blocks of one range lie eight workgroups
// apart, on one XCD, whose L2 then has the rows for the second block. A last kernel joins a query's pieces.
//
// Two forms. Of few query heads or short prefixes one launch (paged_shared_kernel) has prefixes, in blocks of 32 columns, and own
// rows: a tile is a wave's own, in registers, and the four waves of a workgroup, which take the tiles of a piece in turn, meet in
// LDS. Else prefixes are a kernel's own, with up to 128 columns a block, and own rows paged_decode.hip's: tiles of 32 keys come by
// asynchronous copies into a ring of LDS, read from HBM once a block and from LDS by every wave. Of 16-bit rows (paged_prefix_kernel) a
// wave has 32 columns of every second tile, of 8-bit ones (paged_prefix_codes_kernel) sixteen of every tile.
//
// What bounds it: few queries the chain of accesses (requests, groups, lengths, table, rows) and two launches; long prefixes of few
// queries HBM (16 queries over 32768 rows: the tiles' loop reads 6.4 TB/s, 10 of the kernel's 27 us; the others are the plan, the first
// tiles, and 34 MB of partials); many columns the matrix units (256 queries over 8192 rows: 45 us at the rate of a library's product
// with two terms a weight, 55 to 65 taken); 8-bit rows a wave's own chain of scales, terms and cross-lane moves (60 us for 33 queries over
// 20001 rows).
#include "paged_parts.h"

namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kGroups = 256;    // workgroups that run at once: one a compute unit
constexpr int kColumns = 32;    // of a piece, in blocks of 16
constexpr int kWideWaves = 8;   // of the kernels for prefixes alone
constexpr int kWideThreads = 64 * kWideWaves;
constexpr int kAtATime = 2;     // tiles that the waves of a kernel for 16-bit rows take at a time
constexpr int kWideColumns = 128;  // of a block: 32 a wave and tile, of 8-bit rows 16 a wave
constexpr int kBlocks = kColumns / 16;
constexpr int kMinShare = 4;    // tiles of a range, at least: one a wave
constexpr int kMaxRows = 2048;  // queries, and prefixes, of a call

struct SharedRest {
  const void* q;                  // [B, Hq, D]
  const int32_t* prefix_tables;   // [n_prefixes, prefix_width]
  const int32_t* tables;          // [n_tables, width]
  const void *k, *v, *k_scales, *k_biases, *v_scales, *v_biases;
  int n_pages, page_shift, prefix_width, width, prefix_slots, own_slots;
  int block;          // columns of a block of a prefix's members, at most
  float scale_log2;
  float* ws_pre;      // partial outputs of prefix pieces [prefix_slots][block columns][256]
  float* ws_pre_ml;   // their statistics [prefix_slots][block][4]: maximum, sum of weights, two that nothing uses
  float* ws_own;      // of own pieces [own_slots][rep][256]
  float* ws_own_ml;   // [own_slots][16][2]
  int32_t* parts;     // [B * n_kv][8]: of own pieces the first and how many; of prefix pieces the first, ranges, blocks, first column
  void* out;          // [B, Hq, D]
};

struct SharedArgs {
  const int32_t *requests, *groups, *lens, *prefix_lens;
  int batch, n_prefixes, n_tables, n_kv, rep;
  int pieces;  // workgroups: no less than the pieces there can be
  void* decode;
  size_t decode_bytes;
  bool wide;
  SharedRest rest;
};

__device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }

// Pieces of a prefix: ranges of all KV heads ("bundles" of blocks) by eights, block by block, so that the blocks of a bundle are
// multiples of eight apart.
__device__ __forceinline__ int bundle_piece(int bundle, int block, int bundles, int blocks) {
  const int q = bundle / 8;
  return 8 * blocks * q + block * min(8, bundles - 8 * q) + bundle % 8;
}

constexpr int kPlanInts = 5 * kMaxRows;  // groups and requests of queries; lengths of prefixes and queries; members of prefixes

__host__ __device__ constexpr int shared_query_bytes(int qdt, int fmt) {
  return kBlocks * 8 * 64 * 16 * (fmt == kAffine && qdt == MSPR_F32 ? 2 : 1);
}
__host__ __device__ constexpr int shared_lds(int qdt, int fmt) { return kWaves * kVTileBytes + shared_query_bytes(qdt, fmt); }
static_assert(kWaves * kVTileBytes >= kPlanInts * 4, "the plan fits into the V tiles");
static_assert(kWaves * kVTileBytes >= (kWaves * 16 * 64 * 4 + kWaves * 16 * 2) * 4, "the exchange fits into the V tiles");

// What a workgroup works on.
struct Piece {
  int prefix;          // number of the prefix, -1: a query's own rows
  int row;             // the query (own rows), its first column's (a prefix)
  int block, blocks;   // of a prefix's members
  int kvh, range, ranges;
  int first;           // the first piece of the prefix, or the query's first piece of this KV head among own pieces
  int slot;            // where partials go
};

// The tiles of one piece for NB blocks of 16 columns.
template <int QDT, int FMT, int SDT, int NB>
__device__ __forceinline__ void attend_piece(const SharedRest& a, const Piece& p, const int32_t* table, int len, int tile0, int tile1,
                                             int n_kv, int rep, int columns, bool whole, const int* members, unsigned char* lds) {
  constexpr bool kCodes = FMT == kAffine;
  constexpr int kVType = kCodes ? MSPR_F16 : FMT;
  constexpr int kPTerms = 2;                                   // terms of a weight
  constexpr int kQTerms = kCodes && QDT == MSPR_F32 ? 2 : 1;  // terms of a query element
  // (float16 weights are taken 2^11 times as large, see paged_decode.hip; the reference maximum lags by 2^4 at most)
  constexpr float kLag = 4.0f;
  constexpr float kUp = kVType == MSPR_F16 ? 11.0f : 0.0f;
  constexpr int kRowBytes = kCodes ? kD : kD * 2;
  constexpr int kSteps = 8 / kWaves;  // of the query operand, made by a wave
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15;  // MFMA column within its block; row (key) of the K operand
  const int g = lane >> 4;
  unsigned char* vt = lds + wave * kVTileBytes;
  const int page_mask = (1 << a.page_shift) - 1;
  const int last_tile = min(tile1, ceil_div(len, kTileKeys));

  // ---- the queries are asked for first: loads come back in order, and the pages' addresses wait for the table anyway
  constexpr int kQWords = QDT == MSPR_F32 ? 2 : 1;  // of sixteen bytes a step
  bool mine[NB];
  u32x4_t qraw[NB][kSteps * kQWords];
#pragma unroll
  for (int b = 0; b < NB; b++) {
    const int column = 16 * b + n;
    mine[b] = column < columns;
    const int member = mine[b] ? column / rep : 0;
    const int64_t q0 = (((int64_t)members[member] * n_kv + p.kvh) * rep + (mine[b] ? column - member * rep : 0)) * kD;
#pragma unroll
    for (int i = 0; i < kSteps; i++) {
      const int step = kSteps * wave + i;
      const int channel = kCodes ? 32 * (step & ~1) + 16 * g + 8 * (i & 1) : 32 * step + 8 * g;
      constexpr int kQBytes = QDT == MSPR_F32 ? 4 : 2;
      const u32x4_t* from = reinterpret_cast<const u32x4_t*>(reinterpret_cast<const uint8_t*>(a.q) + (q0 + channel) * kQBytes);
#pragma unroll
      for (int j = 0; j < kQWords; j++) qraw[b][i * kQWords + j] = from[j];
    }
  }
  __builtin_amdgcn_sched_barrier(0);

  f32x4_t oacc[NB][16];
#pragma unroll
  for (int b = 0; b < NB; b++)
#pragma unroll
    for (int mt = 0; mt < 16; mt++) oacc[b][mt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  float m_run[NB], l_run[NB];
  f32x4_t bacc[NB];  // weighted biases: lane n (g = 0) has those of column n and the four groups
#pragma unroll
  for (int b = 0; b < NB; b++) {
    m_run[b] = -__builtin_inff();
    l_run[b] = 0.0f;
    bacc[b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  float v_unit = 0x1p-126f;  // what V's scales of group n % 4 are multiples of

  // Pages of this wave's tiles, two half tiles of 16 keys each: lane i of `ids` has the page of half tile i of 31 tiles and the
  // one behind them.
  const int n_mine = last_tile - tile0 > wave ? (last_tile - tile0 - wave + kWaves - 1) / kWaves : 0;
  auto load_ids = [&](int it0) {
    const int it = it0 + (lane >> 1);
    const int key = (tile0 + wave + kWaves * it) * kTileKeys + 16 * (lane & 1);
    const int e = it < n_mine && key < len ? key >> a.page_shift : -1;
    return e >= 0 ? table[e] : -1;
  };
  struct Half {
    int64_t row;  // first row in the pages
    int rows;     // how many count
  };
  auto half_at = [&](int ids, int it0, int it, int u) {
    const int key = (tile0 + wave + kWaves * it) * kTileKeys + 16 * u;
    const int page = __builtin_amdgcn_readlane(ids, 2 * (it - it0) + u);
    const bool good = page >= 0 && page < a.n_pages;
    Half h;
    h.row = ((((int64_t)(good ? page : 0) * n_kv + p.kvh) << a.page_shift) + (key & page_mask));
    h.rows = __builtin_amdgcn_readfirstlane(!good || it >= n_mine ? 0 : len - key >= 16 ? 16 : len - key < 0 ? 0 : len - key);
    return h;
  };

  constexpr int kLoads = kCodes ? 4 : 8;  // 16-byte pieces a lane and half tile
  u32x4_t kr[2][kLoads], vr[2][kLoads];
  RowScales<SDT> ks[2], kb[2], vs[2], vb[2];
  auto load_k = [&](const Half* h) {
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const auto w = rows_window(a.k, h[u].row, kRowBytes, h[u].rows);
#pragma unroll
      for (int j = 0; j < kLoads; j++) kr[u][j] = window_load16(w, n * kRowBytes + 16 * g, 64 * j);
      if constexpr (kCodes) {
        ks[u].load(rows_window(a.k_scales, h[u].row, 4 * RowScales<SDT>::kBytes, h[u].rows), 16 * g + n);
        kb[u].load(rows_window(a.k_biases, h[u].row, 4 * RowScales<SDT>::kBytes, h[u].rows), 4 * n + g);
      }
    }
  };
  auto load_v = [&](const Half* h) {
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const auto w = rows_window(a.v, h[u].row, kRowBytes, h[u].rows);
#pragma unroll
      for (int j = 0; j < kLoads; j++) vr[u][j] = window_load16(w, 16 * lane, 1024 * j);
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
  __builtin_amdgcn_sched_barrier(0);  // the first tile is on its way before the queries are fetched

  // ---- Q^T operands, in LDS for all waves: [blocks][8 steps][terms][64 lanes]
  u32x4_t* qt = reinterpret_cast<u32x4_t*>(lds + kWaves * kVTileBytes) + lane;
  float q_unit[NB], qsum[NB];
#pragma unroll
  for (int b = 0; b < NB; b++) {
    q_unit[b] = a.scale_log2;
    qsum[b] = 0.0f;
  }
  if constexpr (!kCodes) {
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
      for (int i = 0; i < kSteps; i++)
        qt[64 * (8 * b + kSteps * wave + i)] = mine[b] ? qraw[b][i] : u32x4_t{0u, 0u, 0u, 0u};
  } else {
    auto element = [&](int b, int i, float* x) {
      if constexpr (QDT == MSPR_F32) {
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = __uint_as_float(qraw[b][2 * i + j / 4][j % 4]);
      } else {
        widen8<QDT>(qraw[b][i], x);
      }
#pragma unroll
      for (int j = 0; j < 8; j++) x[j] = mine[b] ? x[j] : 0.0f;
    };
    float* shared = reinterpret_cast<float*>(lds);  // [2][blocks][waves][16 columns], where the V tiles will be
    int e[NB] = {};
    if constexpr (QDT != MSPR_F16) {  // a power of two brings the column's largest element to [2^14, 2^15)
#pragma unroll
      for (int b = 0; b < NB; b++) {
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < kSteps; i++) {
          float x[8];
          element(b, i, x);
#pragma unroll
          for (int j = 0; j < 8; j++) top = fmaxf(top, fabsf(x[j]));
        }
        top = half_wave_max(row_pair_max(top));
        if (g == 0) shared[64 * b + 16 * wave + n] = top;
      }
      __syncthreads();
#pragma unroll
      for (int b = 0; b < NB; b++) {
        float top = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; w++) top = fmaxf(top, shared[64 * b + 16 * w + n]);
        if (top > 0.0f && top < __builtin_inff()) e[b] = __builtin_amdgcn_frexp_expf(top) - 15;
      }
    }
    static_assert(kSteps == 2, "a wave makes the operands of one group of 64 channels");
#pragma unroll
    for (int b = 0; b < NB; b++) {
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < kSteps; i++) {
        float x[8];
        element(b, i, x);
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = __builtin_amdgcn_ldexpf(x[j], -e[b]);
        u32x4_t terms[kQTerms];
        split_terms<MSPR_F16, kQTerms>(x, terms);
#pragma unroll
        for (int t = 0; t < kQTerms; t++) {  // (of the terms, as the products are)
          float y[8];
          widen8<MSPR_F16>(terms[t], y);
#pragma unroll
          for (int j = 0; j < 8; j++) sum += y[j];
          qt[64 * ((8 * b + kSteps * wave + i) * kQTerms + t)] = terms[t];
        }
      }
      q_unit[b] = __builtin_amdgcn_ldexpf(a.scale_log2, e[b]);
      sum += __shfl_xor(sum, 16, MSPR_WAVE);
      sum += __shfl_xor(sum, 32, MSPR_WAVE);
      if (g == 0) shared[64 * kBlocks + 64 * b + 16 * wave + n] = sum;
    }
    __syncthreads();
#pragma unroll
    for (int b = 0; b < NB; b++) qsum[b] = shared[64 * kBlocks + 64 * b + 16 * g + n];
  }
  __syncthreads();

  const int tr_off = (4 * g + ((lane & 15) >> 2)) * kVPitch + 4 * (lane & 3) * 2;
  for (int it0 = 0; it0 < n_mine; it0 += 31) {
    const int it_end = min(it0 + 31, n_mine);
    for (int it = it0; it < it_end; it++) {
      nxt[0] = half_at(ids, it0, it + 1, 0);
      nxt[1] = half_at(ids, it0, it + 1, 1);

      // ---- S^T = K . Q^T
      float s[NB][8];  // key 16 u + 4 g + i at 4 u + i
      if constexpr (!kCodes) {
        f32x4_t acc[2][NB];
#pragma unroll
        for (int b = 0; b < NB; b++) acc[0][b] = acc[1][b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 8; j++)
#pragma unroll
          for (int b = 0; b < NB; b++) {
            const u32x4_t qf = qt[64 * (8 * b + j)];
            acc[0][b] = mfma<FMT>(kr[0][j], qf, acc[0][b]);
            acc[1][b] = mfma<FMT>(kr[1][j], qf, acc[1][b]);
          }
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
          for (int i = 0; i < 8; i++) s[b][i] = acc[i >> 2][b][i & 3] * q_unit[b];
      } else {
#pragma unroll
        for (int u = 0; u < 2; u++) {
          const f32x4_t zero = {0.f, 0.f, 0.f, 0.f};
          const float ksf = ks[u].value(n);
          const float of_bias = __int_as_float(__builtin_amdgcn_ds_bpermute(4 * (4 * n + g), __float_as_int(ksf)));
          const float bias = fmaf(128.0f, of_bias, kb[u].value(g));
          f32x4_t sum[NB];
#pragma unroll
          for (int b = 0; b < NB; b++) sum[b] = __builtin_amdgcn_mfma_f32_16x16x4f32(bias, qsum[b], zero, 0, 0, 0);
          static_for<4>([&](auto jc) {
            constexpr int j = decltype(jc)::value;
            f32x4_t acc[NB];
#pragma unroll
            for (int b = 0; b < NB; b++) acc[b] = zero;
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
              for (int t = 0; t < kQTerms; t++)
#pragma unroll
                for (int b = 0; b < NB; b++) acc[b] = mfma<MSPR_F16>(c, qt[64 * ((8 * b + 2 * j + h) * kQTerms + t)], acc[b]);
            }
            static_for<4>([&](auto ic) {
              constexpr int i = decltype(ic)::value;
              const float by = of_lane<4 * i + j>(ksf);
#pragma unroll
              for (int b = 0; b < NB; b++) sum[b][i] = fmaf(by, acc[b][i], sum[b][i]);
            });
          });
#pragma unroll
          for (int b = 0; b < NB; b++)
#pragma unroll
            for (int i = 0; i < 4; i++) s[b][4 * u + i] = sum[b][i] * q_unit[b];
        }
      }
      load_k(nxt);
      __builtin_amdgcn_sched_barrier(0);

      // ---- online softmax (powers of two), the reference maximum moves only past 2^4
      float tmax[NB];
      bool grow = false;
#pragma unroll
      for (int b = 0; b < NB; b++) {
        tmax[b] = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < 8; i++) {
          if (4 * g + (i & 3) >= cur[i >> 2].rows) s[b][i] = -__builtin_inff();
          tmax[b] = fmaxf(tmax[b], s[b][i]);
        }
        tmax[b] = half_wave_max(row_pair_max(tmax[b]));
        grow |= tmax[b] > m_run[b] + kLag;
      }
      if (__any(grow)) {
#pragma unroll
        for (int b = 0; b < NB; b++) {
          const bool up = tmax[b] > m_run[b] + kLag;
          const float m_new = up ? tmax[b] : m_run[b];
          if (it > 0) {  // (sums of nothing need no new scale)
            const float alpha = up ? __builtin_amdgcn_exp2f(m_run[b] - m_new) : 1.0f;
            l_run[b] *= alpha;
#pragma unroll
            for (int mt = 0; mt < 16; mt++) oacc[b][mt] = oacc[b][mt] * alpha;
            bacc[b] = bacc[b] * alpha;
          }
          m_run[b] = m_new;
        }
      }
#pragma unroll
      for (int b = 0; b < NB; b++) {
        const float m_safe = (m_run[b] == -__builtin_inff() ? 0.0f : m_run[b]) - kUp;
#pragma unroll
        for (int i = 0; i < 8; i++) {
          s[b][i] = __builtin_amdgcn_exp2f(s[b][i] - m_safe);
          l_run[b] += s[b][i];
        }
      }

      // ---- V rows to LDS (zeros in the place of rows that do not count)
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int j = 0; j < kLoads; j++) {
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

      // ---- O^T += V^T . P^T (the tile was written by this wave only: LDS operations of one wave complete in order)
      __builtin_amdgcn_wave_barrier();
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
      u32x4_t pf[NB][kPTerms];
      auto accumulate = [&](int q4) {
        if (q4 < 3) read_v(q4 + 1);
#pragma unroll
        for (int t = 0; t < kPTerms; t++)
#pragma unroll
          for (int m = 0; m < 4; m++)
#pragma unroll
            for (int b = 0; b < NB; b++) oacc[b][4 * q4 + m] = mfma<kVType>(vf[q4 & 1][m], pf[b][t], oacc[b][4 * q4 + m]);
      };
      read_v(0);
      if constexpr (!kCodes) {
#pragma unroll
        for (int b = 0; b < NB; b++) split_terms<kVType, kPTerms>(s[b], pf[b]);
#pragma unroll
        for (int q4 = 0; q4 < 4; q4++) accumulate(q4);
      } else {
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
#pragma unroll
            for (int b = 0; b < NB; b++)
              static_for<16>([&](auto mt) { oacc[b][mt] = oacc[b][mt] * of_lane<decltype(mt)::value / 4>(by); });
          }
          v_unit = unit;
        }
        const float per_unit = 1.0f / v_unit;
        vsf[0] *= per_unit;
        vsf[1] *= per_unit;
        const float vbf[2] = {fmaf(128.0f, vs[0].value(n), vb[0].value(n)), fmaf(128.0f, vs[1].value(n), vb[1].value(n))};
        static_for<8>([&](auto ic) {
          constexpr int i = decltype(ic)::value;
          float bias = vbf[i >> 2];
          if constexpr ((i & 3) != 0)
            bias = __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(bias), 0x100 + 4 * (i & 3), 0xF, 0xF, true));  // row_shl
#pragma unroll
          for (int b = 0; b < NB; b++) bacc[b] = __builtin_amdgcn_mfma_f32_16x16x4f32(bias, s[b][i], bacc[b], 0, 0, 0);
        });
        static_for<4>([&](auto jc) {  // the weights of group j, which has channels 64 j on
          constexpr int j = decltype(jc)::value;
          float of_key[8];
          static_for<8>([&](auto ic) {
            constexpr int i = decltype(ic)::value;
            of_key[i] = of_lane<4 * (i & 3) + j>(vsf[i >> 2]);
          });
#pragma unroll
          for (int b = 0; b < NB; b++) {
            float w[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
              w[i] = of_key[i] * s[b][i];
              asm("" : "+v"(w[i]));  // (a rounded product, see paged_decode.hip)
            }
            split_terms<kVType, kPTerms>(w, pf[b]);
          }
          accumulate(j);
        });
      }
      if constexpr (kCodes) load_v_scales(nxt);
      __builtin_amdgcn_wave_barrier();
    }
    ids = ids_next;
    ids_next = load_ids(it_end + 31);
  }

  // ---- the four waves meet in LDS, a block of columns at a time (the V tiles are free now)
  float* xo = reinterpret_cast<float*>(lds);   // [waves][16 mt][64 lanes][4]
  float* xml = xo + kWaves * 16 * 64 * 4;      // [waves][16 columns][2]
  const int width = p.prefix >= 0 ? a.block : rep;  // columns of a partial
  const auto po = store_window((p.prefix >= 0 ? a.ws_pre : a.ws_own) + (int64_t)p.slot * width * kD, width * kD * (int)sizeof(float));
  float* ml = p.prefix >= 0 ? a.ws_pre_ml + (int64_t)p.slot * a.block * 4 : a.ws_own_ml + (int64_t)p.slot * 16 * 2;
  const int ml_pitch = p.prefix >= 0 ? 4 : 2;
#pragma unroll
  for (int b = 0; b < NB; b++) {
    l_run[b] += __shfl_xor(l_run[b], 16, MSPR_WAVE);
    l_run[b] += __shfl_xor(l_run[b], 32, MSPR_WAVE);
    if constexpr (kCodes) {
      float bias[4];
#pragma unroll
      for (int j = 0; j < 4; j++) bias[j] = __shfl(bacc[b][j], n, MSPR_WAVE);
      static_for<16>([&](auto mt) { oacc[b][mt] = oacc[b][mt] * of_lane<decltype(mt)::value / 4>(v_unit) + bias[mt >> 2]; });
    }
    __syncthreads();
#pragma unroll
    for (int mt = 0; mt < 16; mt++) *reinterpret_cast<f32x4_t*>(xo + ((wave * 16 + mt) * 64 + lane) * 4) = oacc[b][mt];
    if (g == 0) {
      xml[(wave * 16 + n) * 2] = m_run[b];
      xml[(wave * 16 + n) * 2 + 1] = l_run[b];
    }
    __syncthreads();
    float mw[kWaves], m_all = -__builtin_inff(), l_all = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; w++) {
      mw[w] = xml[(w * 16 + n) * 2];
      m_all = fmaxf(m_all, mw[w]);
    }
    const float m_safe = m_all == -__builtin_inff() ? 0.0f : m_all;
#pragma unroll
    for (int w = 0; w < kWaves; w++) {
      mw[w] = __builtin_amdgcn_exp2f(mw[w] - m_safe);
      l_all += xml[(w * 16 + n) * 2 + 1] * mw[w];
    }
    const int column = 16 * b + n;
#pragma unroll
    for (int q4 = 0; q4 < 16 / kWaves; q4++) {
      const int mt = wave * (16 / kWaves) + q4;
      f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kWaves; w++) acc += *reinterpret_cast<const f32x4_t*>(xo + ((w * 16 + mt) * 64 + lane) * 4) * mw[w];
      if (!mine[b]) continue;
      if (whole) store_out<QDT>(a.out, (((int64_t)p.row * n_kv + p.kvh) * rep + column) * kD + 16 * mt + 4 * g, acc, l_all);
      else window_store<kStoreThrough>(po, (column * kD + 16 * mt + 4 * g) * 4, __builtin_bit_cast(u32x4_t, acc));
    }
    if (!whole && wave == 0 && g == 0 && mine[b]) *reinterpret_cast<f32x2_t*>(ml + ml_pitch * column) = f32x2_t{m_all, l_all};
  }
}

// QDT: type of queries and output; FMT: page format; SDT: type of scales and biases (8-bit pages). A piece a workgroup.
template <int QDT, int FMT, int SDT>
__global__ __launch_bounds__(kThreads, 1) void paged_shared_kernel(const int32_t* requests, const int32_t* groups, const int32_t* lens,
                                                                   const int32_t* prefix_lens, int batch, int n_prefixes,
                                                                   int n_tables, int n_kv, int rep, SharedRest a) {
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  __shared__ int wave_sums[3][kWaves];
  __shared__ int members[kColumns];
  __shared__ Piece found;
  const int t = threadIdx.x;
  const int lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int number = blockIdx.x;

  // ---- the plan: which query belongs to which prefix, and how many tiles there are
  int* row_group = reinterpret_cast<int*>(lds);       // [batch]
  int* row_request = row_group + kMaxRows;            // [batch]
  int* length = row_request + kMaxRows;               // [n_prefixes, then batch]
  int* count = length + 2 * kMaxRows;                 // [n_prefixes]
  const int prefix_cap = a.prefix_width << a.page_shift, cap = a.width << a.page_shift;
  // (what a thread's first query and prefix need is asked for at once; the plan keeps all of it, so that a piece asks for no length again)
  auto request_of = [&](int r) { return r >= batch ? -1 : requests ? requests[r] : r; };
  auto group_of = [&](int request) { return request >= 0 && request < n_tables ? groups[request] : -1; };
  int request = request_of(t);
  int row_length = t < batch ? length_of(lens, batch, t, cap) : 0;
  const int first_length = t < n_prefixes ? length_of(prefix_lens, n_prefixes, t, prefix_cap) : 0;
  int group = group_of(request);
  for (int i = t; i < n_prefixes; i += kThreads) {
    length[i] = i == t ? first_length : length_of(prefix_lens, n_prefixes, i, prefix_cap);
    count[i] = 0;
  }
  __syncthreads();
  for (int r = t; r < batch; r += kThreads) {
    if (r > t) {
      request = request_of(r);
      group = group_of(request);
      row_length = length_of(lens, batch, r, cap);
    }
    if (group < 0 || group >= n_prefixes || length[group] == 0) group = -1;
    row_group[r] = group;
    const bool known = request >= 0 && request < n_tables;
    row_request[r] = known ? request : 0;
    length[n_prefixes + r] = known ? row_length : 0;
    if (group >= 0) atomicAdd(&count[group], 1);
  }
  auto tiles_of = [&](int e) { return ceil_div(length[e], kTileKeys); };
  if (t == 0) found.kvh = -1;
  __syncthreads();
  const int rows_a_block = kColumns / rep;
  auto blocks_of = [&](int e) { return e >= n_prefixes ? 1 : ceil_div(count[e], rows_a_block); };
  const int entries = n_prefixes + batch, per = ceil_div(entries, kThreads);
  const int e0 = min(t * per, entries), e1 = min(e0 + per, entries);
  int sum = 0, units = 0;
  for (int e = e0; e < e1; e++) {
    const int blocks = blocks_of(e);
    sum += blocks * tiles_of(e);
    units += blocks;
  }
  sum = wave_scan(sum);
  units = wave_scan(units);
  if (lane == 63) {
    wave_sums[0][wave] = sum;
    wave_sums[1][wave] = units;
  }
  __syncthreads();
  int all = 0, all_units = 0;
#pragma unroll
  for (int w = 0; w < kWaves; w++) {
    all += wave_sums[0][w];
    all_units += wave_sums[1][w];
  }
  all = __builtin_amdgcn_readfirstlane(all) * n_kv;
  all_units = __builtin_amdgcn_readfirstlane(all_units) * n_kv;
  // A range's tiles: no more pieces than compute units, as a unit has at most one piece that is not full; where there are too
  // many units for that, half as many again.
  const int share = max(kMinShare, ceil_div(all, max(kGroups - all_units, kGroups / 2)));
  int pieces = 0, of_prefixes = 0;
  for (int e = e0; e < e1; e++) {
    const int ranges = max(1, ceil_div(tiles_of(e), share));
    const int blocks = blocks_of(e);
    pieces += n_kv * blocks * ranges;
    if (e < n_prefixes) of_prefixes += n_kv * blocks * ranges;
  }
  const int upto = wave_scan(pieces);
  of_prefixes = wave_scan(of_prefixes);
  __syncthreads();
  if (lane == 63) {
    wave_sums[0][wave] = upto;
    wave_sums[2][wave] = of_prefixes;
  }
  __syncthreads();
  int before = upto - pieces, prefix_pieces = 0;
#pragma unroll
  for (int w = 0; w < kWaves; w++) {
    if (w < wave) before += wave_sums[0][w];
    prefix_pieces += wave_sums[2][w];
  }
  if (number >= before && number < before + pieces) {
    for (int e = e0; e < e1; e++) {
      const int ranges = max(1, ceil_div(tiles_of(e), share));
      const int blocks = blocks_of(e);
      const int own = n_kv * blocks * ranges;
      if (number < before + own) {
        Piece p;
        p.blocks = blocks;
        p.ranges = ranges;
        const int i = number - before;
        int bundle;
        if (e < n_prefixes) {
          const int bundles = n_kv * ranges, q = i / (8 * blocks), j = i - 8 * blocks * q, m = min(8, bundles - 8 * q);
          p.prefix = e;
          p.row = 0;
          p.block = j / m;
          bundle = 8 * q + j % m;
          p.first = before;
          p.slot = number;
        } else {
          p.prefix = -1;
          p.row = e - n_prefixes;
          p.block = 0;
          bundle = i;
          p.slot = number - prefix_pieces;
          p.first = p.slot - i % ranges;
        }
        p.kvh = bundle / ranges;
        p.range = bundle - p.kvh * ranges;
        found = p;
        break;
      }
      before += own;
    }
  }
  __syncthreads();
  Piece p;
  p.kvh = __builtin_amdgcn_readfirstlane(found.kvh);
  if (p.kvh < 0) return;  // (more workgroups than pieces)
  p.prefix = __builtin_amdgcn_readfirstlane(found.prefix);
  p.row = __builtin_amdgcn_readfirstlane(found.row);
  p.block = __builtin_amdgcn_readfirstlane(found.block);
  p.blocks = __builtin_amdgcn_readfirstlane(found.blocks);
  p.range = __builtin_amdgcn_readfirstlane(found.range);
  p.ranges = __builtin_amdgcn_readfirstlane(found.ranges);
  p.first = __builtin_amdgcn_readfirstlane(found.first);
  p.slot = __builtin_amdgcn_readfirstlane(found.slot);

  // ---- the queries of the piece
  int n_members = 1, n_tiles, len;
  const int32_t* table;
  bool whole = false;
  if (p.prefix >= 0) {
    const int per_row = ceil_div(batch, kThreads);
    const int r0 = min(t * per_row, batch), r1 = min(r0 + per_row, batch);
    int mine = 0;
    for (int r = r0; r < r1; r++) mine += row_group[r] == p.prefix;
    const int scanned = wave_scan(mine);
    if (lane == 63) wave_sums[1][wave] = scanned;
    __syncthreads();
    int rank = scanned - mine - p.block * rows_a_block;
#pragma unroll
    for (int w = 0; w < kWaves; w++)
      if (w < wave) rank += wave_sums[1][w];
    for (int r = r0; r < r1; r++)
      if (row_group[r] == p.prefix) {
        if (rank >= 0 && rank < rows_a_block) {
          members[rank] = r;
          if (p.range == 0) {
            int32_t* at = a.parts + 8 * ((int64_t)r * n_kv + p.kvh);
            at[2] = p.first;
            at[3] = p.ranges;
            at[4] = p.blocks;
            at[5] = p.block * a.block + rank * rep;
          }
        }
        rank++;
      }
    n_members = min(rows_a_block, __builtin_amdgcn_readfirstlane(count[p.prefix]) - p.block * rows_a_block);
    len = __builtin_amdgcn_readfirstlane(length[p.prefix]);
    n_tiles = ceil_div(len, kTileKeys);
    table = a.prefix_tables + (int64_t)p.prefix * a.prefix_width;
  } else {
    len = __builtin_amdgcn_readfirstlane(length[n_prefixes + p.row]);
    n_tiles = ceil_div(len, kTileKeys);
    const bool alone = __builtin_amdgcn_readfirstlane(row_group[p.row]) < 0;
    whole = alone && p.ranges == 1;
    const bool some = !whole && n_tiles > 0;
    table = a.tables + (int64_t)__builtin_amdgcn_readfirstlane(row_request[p.row]) * a.width;
    if (t == 0) {
      members[0] = p.row;
      if (p.range == 0) {
        int32_t* at = a.parts + 8 * ((int64_t)p.row * n_kv + p.kvh);
        at[0] = p.first;
        at[1] = some ? p.ranges : 0;
        if (alone) at[3] = 0;
      }
    }
    if (!whole && !some) return;  // (no rows of its own behind a prefix)
  }
  __syncthreads();  // (the plan lies where the V tiles will be)
  if (p.slot >= (p.prefix >= 0 ? a.prefix_slots : a.own_slots)) return;  // (cannot be, unless lengths change meanwhile)
  const int tile0 = (int)((int64_t)n_tiles * p.range / p.ranges), tile1 = (int)((int64_t)n_tiles * (p.range + 1) / p.ranges);
  const int columns = n_members * rep;
  if (columns <= 16)
    attend_piece<QDT, FMT, SDT, 1>(a, p, table, len, tile0, tile1, n_kv, rep, columns, whole, members, lds);
  else
    attend_piece<QDT, FMT, SDT, 2>(a, p, table, len, tile0, tile1, n_kv, rep, columns, whole, members, lds);
}

// ---------------------------------------------------------------------------------------------- prefixes of 16-bit rows

constexpr int kRowBytes = kD * 2;
constexpr int kTileBytes = kTileKeys * kRowBytes;  // 16 KB, K and V each
constexpr int kStageBytes = 2 * kTileBytes;
constexpr int kStages = 4;                         // tiles of the ring
constexpr int kWideLds = kStages * kStageBytes;    // 128 KB
constexpr int kChunk = 30;                         // tiles whose pages a wave has at hand, with two more behind them
static_assert(2 * kStageBytes >= 3 * kMaxRows * 4, "the plan fits into half of the ring");

__device__ const uint32_t g_no_rows[kRowBytes / 4] = {};  // what half tiles without rows are copied from

template <int FMT>
__device__ __forceinline__ f32x16_t mfma32(u32x4_t a, u32x4_t b, f32x16_t c) {
  if constexpr (FMT == MSPR_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}

template <int N>
__device__ __forceinline__ void wait_copies_and_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}
// The waves' LDS accesses only: copies and loads stay under way.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
// Lane i's 16 bytes at base + offset land at lds_base + 16 i. In an asm statement, so that the compiler does not wait for it in
// front of other LDS reads (s_nop: an instruction has to lie between the scalar write of M0 and the copy).
__device__ __forceinline__ void copy_16(uint64_t base, uint32_t offset, uint32_t lds_base) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %0" ::"s"(base), "v"(offset), "s"(lds_base) : "memory", "m0");
}
__device__ __forceinline__ uint32_t lds_address(const unsigned char* p) {
  return (uint32_t)(uintptr_t)MSPR_LDS_PTR(const unsigned char, p);
}
// Sixteen-byte piece p of tile row r lies at place (p & 16) | ((p ^ swizzle(r)) & 15): neither the K operand's reads (lane = row) nor the
// transposed ones of V meet a bank twice.
__device__ __forceinline__ int swizzle(int r) { return ((r & 7) << 1) | ((r >> 3) & 1); }

// One piece: `columns` columns (head rows of q in `column_row`) over tiles [tile0, tile1), two at a time: wave w has columns 32 (w % 4)
// on and every second tile. (Blocks of 256 columns, which read a prefix half as often, a tile at a time: 2048 query heads a KV head over
// 8192 rows 0.5 % less time, over 20000 rows 2 % less, but 256 over 32768 rows 7 % more, 200 ragged queries 3 % more. One tile at a time for
// blocks of 128: 1 % more for 16 queries over 32768 rows.)
template <int FMT, typename F>
__device__ __forceinline__ void prefix_piece(const SharedRest& a, const int32_t* table, int len, int tile0, int tile1, int n_kv, int kvh,
                                             int slot, int columns, const int* column_row, F&& find_members, unsigned char* lds,
                                             float (*xml)[32][2]) {
  constexpr float kLag = 4.0f;                              // (as in paged_decode.hip)
  constexpr float kUp = FMT == MSPR_F16 ? 11.0f : 0.0f;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 31, g = lane >> 5;  // column within the wave's; key of the K operand
  constexpr int kColumnWaves = kWideWaves / kAtATime;
  const int column0 = 32 * (wave % kColumnWaves), part = wave / kColumnWaves;
  const int mine = __builtin_amdgcn_readfirstlane(min(max(columns - column0, 0), 32));  // columns of this wave
  const int page_mask = (1 << a.page_shift) - 1;

  // ---- copies: a thread has row tid / 32 of both half tiles of 16 keys, of K and of V
  const int c_row = tid >> 5;
  const int c_piece = (tid & 16) | ((tid ^ swizzle(c_row)) & 15);  // (row 16 + c_row has the same swizzle)
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_address(lds)) + wave * 1024;
  auto load_ids = [&](int t0) {  // lane i: page of half tile i from tile t0 on
    const int t = t0 + (lane >> 1), key = t * kTileKeys + 16 * (lane & 1);
    const int e = t < tile1 && key < len ? key >> a.page_shift : -1;
    return e >= 0 ? table[e] : -1;
  };
  // Rows of tile t that count, of its first half and (from bit 8 on) of its second. Rows behind them are copies of the last: they
  // are masked, and must not be what is no number where that is not.
  auto issue_tile = [&](int ids, int t0, int t, int stage) {
    uint32_t rows = 0;
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const int page = __builtin_amdgcn_readlane(ids, 2 * (t - t0) + u);
      const int key = t * kTileKeys + 16 * u;
      const bool good = page >= 0 && page < a.n_pages && t < tile1;
      const int count = !good ? 0 : len - key >= 16 ? 16 : len - key < 0 ? 0 : len - key;
      const int64_t row = ((((int64_t)(good ? page : 0) * n_kv + kvh) << a.page_shift) + (key & page_mask));
      const uint64_t none = (uint64_t)(const void*)g_no_rows;
      const uint64_t kb = count > 0 ? (uint64_t)a.k + row * kRowBytes : none, vb = count > 0 ? (uint64_t)a.v + row * kRowBytes : none;
      const uint32_t offset = (uint32_t)(min(c_row, max(count, 1) - 1) * kRowBytes + c_piece * 16);
      const uint32_t to = lds0 + stage * kStageBytes + u * 8192;
      copy_16(kb, offset, to);
      copy_16(vb, offset, to + kTileBytes);
      rows |= (uint32_t)count << 8 * u;
    }
    return rows;
  };
  auto issue_step = [&](int ids, int t0, int step) {
    uint32_t rows = 0;
#pragma unroll
    for (int i = 0; i < kAtATime; i++) {
      const int t = tile0 + step * kAtATime + i;
      const uint32_t r = issue_tile(ids, t0, t, (step * kAtATime + i) % kStages);
      if (i == part) rows = r;
    }
    return rows;
  };
  const int n_steps = __builtin_amdgcn_readfirstlane((tile1 - tile0 + kAtATime - 1) / kAtATime);
  int ids = load_ids(tile0);
  uint32_t ahead = issue_step(ids, tile0, 0);  // rows of this wave's tile in the step under way
  int ids_next = load_ids(tile0 + kChunk);
  find_members();  // (under the first copies)

  // ---- Q^T operand: lane (n, g) holds q[column][16 s + 8 g ...] for step s. The wave's rows come in halves of 128 channels, in whole
  //      runs of 256 bytes, and change lanes in 8 KB of LDS that no tile uses yet (piece p of row r at p ^ (r & 15)).
  u32x4_t qf[16];
  {
    const int xr = lane / 16, xc = lane % 16;
    u32x4_t raw[2][8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const int column = column0 + 4 * i + xr;
      const int64_t row = column_row[column < columns ? column : 0];
#pragma unroll
      for (int h = 0; h < 2; h++) raw[h][i] = reinterpret_cast<const u32x4_t*>(a.q)[row * 32 + h * 16 + xc];
    }
    lds_barrier();  // (the plan lies there)
    unsigned char* xq = lds + 2 * kStageBytes + (wave << 13);
#pragma unroll
    for (int h = 0; h < 2; h++) {
#pragma unroll
      for (int i = 0; i < 8; i++) *reinterpret_cast<u32x4_t*>(xq + (4 * i + xr) * 256 + 16 * (xc ^ ((4 * i + xr) & 15))) = raw[h][i];
#pragma unroll
      for (int s = 0; s < 8; s++) qf[8 * h + s] = *reinterpret_cast<const u32x4_t*>(xq + n * 256 + 16 * ((2 * s + g) ^ (n & 15)));
    }
#pragma unroll
    for (int s = 0; s < 16; s++) asm volatile("" : "+v"(qf[s]));
  }

  f32x16_t oacc[8];
#pragma unroll
  for (int mt = 0; mt < 8; mt++) oacc[mt] = f32x16_t{0};
  float m_run = -__builtin_inff(), l_run = 0.0f;

  const int k_off = n * kRowBytes + 32 * (n & 7) + 16 * (g ^ ((n >> 3) & 1));
  const int tr_s = lane & 15;
  const int tr_row = 4 * g + (tr_s >> 2);                          // + 8 h + 16 half
  const int tr_piece = 2 * ((lane >> 4) & 1) + ((tr_s & 3) >> 1);  // of the 64 bytes that 32 channels take
  int v_off[2];
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const int r = tr_row + 8 * h;
    v_off[h] = kTileBytes + r * kRowBytes + 16 * ((tr_piece ^ swizzle(r)) & 15) + 8 * (tr_s & 1);
  }

  auto attend_tile = [&](const unsigned char* st, uint32_t rows) {
    // ---- S^T = K . Q^T: register i is key 8 (i / 4) + 4 g + i % 4
    f32x16_t s = f32x16_t{0};
    {
      constexpr int kReadAhead = 4;
      const uint32_t kb = lds_address(st) + (uint32_t)k_off;
      u32x4_t af[16];
#pragma unroll
      for (int j = 0; j < 16; j++)
        af[j] = *MSPR_LDS_PTR(const u32x4_t, (uintptr_t)((kb ^ (uint32_t)((j & 7) << 5)) + (uint32_t)((j >> 3) * 256)));
#pragma unroll
      for (int j = 0; j < 16; j++) s = mfma32<FMT>(af[j], qf[j], s);
      __builtin_amdgcn_sched_group_barrier(0x100, kReadAhead, 0);  // LDS reads
#pragma unroll
      for (int j = 0; j < 16 - kReadAhead; j++) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // matrix instructions
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, kReadAhead, 0);
    }
    // ---- online softmax
    float tmax = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < 16; i++) s[i] *= a.scale_log2;
    if (rows != 0x1010u) {
      const int first = (int)(rows & 0xFFu) - 4 * g, second = (int)(rows >> 8) - 4 * g;
#pragma unroll
      for (int i = 0; i < 16; i++)
        if (8 * ((i & 7) / 4) + i % 4 >= (i < 8 ? first : second)) s[i] = -__builtin_inff();
    }
#pragma unroll
    for (int i = 0; i < 16; i++) tmax = fmaxf(tmax, s[i]);
    tmax = half_wave_max(tmax);
    const bool grow = tmax > m_run + kLag;
    if (__any(grow)) {
      const float m_new = grow ? tmax : m_run;
      const float alpha = grow ? __builtin_amdgcn_exp2f(m_run - m_new) : 1.0f;
      l_run *= alpha;
      m_run = m_new;
#pragma unroll
      for (int mt = 0; mt < 8; mt++) oacc[mt] = oacc[mt] * alpha;
    }
    const float m_safe = (m_run == -__builtin_inff() ? 0.0f : m_run) - kUp;
#pragma unroll
    for (int i = 0; i < 16; i++) {
      s[i] = __builtin_amdgcn_exp2f(s[i] - m_safe);
      l_run += s[i];
    }
    // ---- O^T += V^T . P^T, half a tile at a time (of whose weights only one half's terms take registers then)
    const uint32_t vb0 = lds_address(st) + (uint32_t)v_off[0], vb1 = lds_address(st) + (uint32_t)v_off[1];
#pragma unroll
    for (int h = 0; h < 2; h++) {
      constexpr int kReadAhead = 3;
      float p[8];
#pragma unroll
      for (int i = 0; i < 8; i++) p[i] = s[8 * h + i];
      u32x4_t pf[2];
      split_terms<FMT, 2>(p, pf);
      u32x4_t vf[8];
#pragma unroll
      for (int mt = 0; mt < 8; mt++) {
        const uint32_t lo_a = (vb0 ^ (uint32_t)((mt & 3) << 6)) + (uint32_t)((mt >> 2) * 256 + h * 16 * kRowBytes);
        const uint32_t hi_a = (vb1 ^ (uint32_t)((mt & 3) << 6)) + (uint32_t)((mt >> 2) * 256 + h * 16 * kRowBytes);
        const u32x2_t lo = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(MSPR_LDS_PTR(s16x4_t, (uintptr_t)lo_a)));
        const u32x2_t hi = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(MSPR_LDS_PTR(s16x4_t, (uintptr_t)hi_a)));
        vf[mt] = u32x4_t{lo.x, lo.y, hi.x, hi.y};
      }
#pragma unroll
      for (int mt = 0; mt < 8; mt++) {
        oacc[mt] = mfma32<FMT>(vf[mt], pf[0], oacc[mt]);
        oacc[mt] = mfma32<FMT>(vf[mt], pf[1], oacc[mt]);
      }
      __builtin_amdgcn_sched_group_barrier(0x100, 2 * kReadAhead, 0);
#pragma unroll
      for (int i = 0; i < 8 - kReadAhead; i++) {
        __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, 2 * kReadAhead, 0);
    }
  };

  for (int s0 = 0; s0 < n_steps; s0 += kChunk / kAtATime) {
    const int s_end = min(s0 + kChunk / kAtATime, n_steps), t0 = tile0 + s0 * kAtATime;
    for (int step = s0; step < s_end; step++) {
      // This step's tiles have landed once the wave's copies of them have and every wave got here; the stages of the step before are
      // free then.
      wait_copies_and_barrier<0>();
      const uint32_t rows = ahead;
      ahead = issue_step(ids, t0, step + 1);  // (behind the last, tiles without rows)
      if (mine > 0 && rows != 0) attend_tile(lds + ((step * kAtATime + part) % kStages) * kStageBytes, rows);
    }
    ids = ids_next;
    ids_next = load_ids(t0 + 2 * kChunk);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (the last copies must not outlive the piece)

  // ---- the waves of one block of columns meet in LDS; rows of the partial leave in whole runs, through 16 KB a wave
  l_run += __shfl_xor(l_run, 32, MSPR_WAVE);
  __syncthreads();  // every wave has left the tiles
  int tl = tid;
  asm volatile("" : "+v"(tl));  // (the offsets below are made here, not carried through the tile loop)
  const int en = tl & 31, eg = (tl >> 5) & 1;
  unsigned char* region = lds + (wave % kColumnWaves) * 32768;
  f32x4_t* xo = reinterpret_cast<f32x4_t*>(region) + (tl & 63);  // [32 quads][64 lanes]
  if (part == 1 && mine > 0) {
#pragma unroll
    for (int mt = 0; mt < 8; mt++)
#pragma unroll
      for (int c = 0; c < 4; c++)
        xo[64 * (4 * mt + c)] = f32x4_t{oacc[mt][4 * c], oacc[mt][4 * c + 1], oacc[mt][4 * c + 2], oacc[mt][4 * c + 3]};
    if (eg == 0) {
      xml[wave % kColumnWaves][en][0] = m_run;
      xml[wave % kColumnWaves][en][1] = l_run;
    }
  }
  __syncthreads();
  if (part == 1 || mine == 0) return;
  const float m2 = xml[wave][en][0], l2 = xml[wave][en][1];
  const float m_all = fmaxf(m_run, m2), m_safe = m_all == -__builtin_inff() ? 0.0f : m_all;
  const float w1 = __builtin_amdgcn_exp2f(m_run - m_safe), w2 = __builtin_amdgcn_exp2f(m2 - m_safe);
  int row0 = slot * a.block + column0;  // (a scalar by hand: with the lanes' addresses below, the compiler takes it for one of each lane's)
  asm volatile("" : "+s"(row0));
  if (eg == 0 && en < mine) *reinterpret_cast<f32x2_t*>(a.ws_pre_ml + 4 * (int64_t)(row0 + en)) = f32x2_t{m_all, l_run * w1 + l2 * w2};
  const auto to = store_window(a.ws_pre + (int64_t)row0 * kD, mine * kD * 4);
  // (half of the channels at a time: the first half's exchange is over when its rows take the place)
#pragma unroll
  for (int h = 0; h < 2; h++) {
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int mt = 0; mt < 4; mt++)
#pragma unroll
      for (int c = 0; c < 4; c++) {
        const f32x4_t other = xo[64 * (16 * h + 4 * mt + c)];
#pragma unroll
        for (int i = 0; i < 4; i++) oacc[4 * h + mt][4 * c + i] = oacc[4 * h + mt][4 * c + i] * w1 + other[i] * w2;
      }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int mt = 0; mt < 4; mt++)
#pragma unroll
      for (int c = 0; c < 4; c++) {
        const f32x16_t& o = oacc[4 * h + mt];
        *reinterpret_cast<f32x4_t*>(region + en * 512 + 16 * ((8 * mt + 2 * c + eg) ^ (en & 15))) =
            f32x4_t{o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]};
      }
#pragma unroll
    for (int i = 0; i < 16; i++) {
      const int r = 2 * i + eg;
      const f32x4_t v = *reinterpret_cast<const f32x4_t*>(region + r * 512 + 16 * (en ^ (r & 15)));
      window_store<kStoreThrough>(to, r * kD * 4 + 512 * h + 16 * en, __builtin_bit_cast(u32x4_t, v));
    }
  }
}

// What a workgroup of the kernels for prefixes does: the plan, in `plan` (LDS where no first copy goes), then its piece by `run`(table, rows,
// first tile, last, KV head, columns, what finds its members).
template <typename F>
__device__ __forceinline__ void prefix_workgroup(const int32_t* requests, const int32_t* groups, const int32_t* prefix_lens, int batch,
                                                 int n_prefixes, int n_tables, int n_kv, int rep, const SharedRest& a, int step,
                                                 unsigned char* plan, int* wave_members, int* column_row, F&& run) {
  const int t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int number = blockIdx.x;

  // ---- members of every prefix
  int* row_group = reinterpret_cast<int*>(plan);  // [batch]
  int* length = row_group + kMaxRows;             // [n_prefixes]
  int* count = length + kMaxRows;                 // [n_prefixes]
  const int prefix_cap = a.prefix_width << a.page_shift;
  auto group_of = [&](int r) {
    if (r >= batch) return -1;
    const int request = requests ? requests[r] : r;
    return request >= 0 && request < n_tables ? groups[request] : -1;
  };
  int group = group_of(t);  // (asked for together with the lengths)
  for (int i = t; i < n_prefixes; i += kWideThreads) {
    length[i] = length_of(prefix_lens, n_prefixes, i, prefix_cap);
    count[i] = 0;
  }
  lds_barrier();
  for (int r = t; r < batch; r += kWideThreads) {
    if (r > t) group = group_of(r);
    if (group < 0 || group >= n_prefixes || length[group] == 0) group = -1;
    row_group[r] = group;
    if (group >= 0) atomicAdd(&count[group], 1);
    else if (number == 0)
      for (int kvh = 0; kvh < n_kv; kvh++) a.parts[8 * ((int64_t)r * n_kv + kvh) + 3] = 0;
  }
  lds_barrier();

  // ---- the plan, by every wave for itself: 64 prefixes at a time, one a lane
  const int most = a.block / rep;  // members of a block
  const int chunks = ceil_div(n_prefixes, MSPR_WAVE);
  struct Load {
    int blocks, tiles;
  };
  auto load_of = [&](int chunk) {
    const int e = chunk * MSPR_WAVE + lane;
    return e < n_prefixes ? Load{ceil_div(count[e], most), ceil_div(length[e], kTileKeys)} : Load{0, 0};
  };
  Load first = load_of(0);
  int all = 0, units = 0;
  for (int c = 0; c < chunks; c++) {
    const Load p = c == 0 ? first : load_of(c);
    all += __builtin_amdgcn_readlane(wave_scan(p.blocks * p.tiles), 63);
    units += __builtin_amdgcn_readlane(wave_scan(p.blocks), 63);
  }
  if (all == 0) return;
  all *= n_kv;
  units *= n_kv;
  // A range's tiles: so many that there are no more pieces than compute units, as a unit has at most one piece that is not full; where
  // there are too many units for that, half as many again. Of few prefixes the least of 64 lengths that does it, tried one a lane (256
  // queries over 8192 rows of two KV heads: 256 pieces of 32 tiles, not 224 of 37; 12 % of the kernel's time).
  int share = max(kMinShare, ceil_div(all, max(kGroups - units, kGroups / 2)));
  if (n_prefixes <= 16 && all < (1 << 21)) {
    const int tried = (max(kMinShare, ceil_div(all, kGroups)) + step - 1) / step * step + step * lane;
    const float inverse = 1.0f / (float)tried;  // (exact enough: quotients below 2^21, a half away from whole numbers)
    int pieces = 0;
    for (int e = 0; e < n_prefixes; e++) {
      const int tiles = __builtin_amdgcn_readlane(first.tiles, e), blocks = __builtin_amdgcn_readlane(first.blocks, e);
      pieces += blocks * (int)(((float)(tiles + tried - 1) + 0.5f) * inverse);
    }
    const uint64_t fits = __ballot(pieces * n_kv <= kGroups);
    if (fits) share = min(share, __builtin_amdgcn_readlane(tried, __builtin_ctzll(fits)));
  }
  int before = 0, prefix = -1, blocks = 0, ranges = 0;
  for (int c = 0; c < chunks && prefix < 0; c++) {
    const Load p = c == 0 ? first : load_of(c);
    const int p_ranges = ceil_div(p.tiles, share), pieces = n_kv * p.blocks * p_ranges;
    const int upto = before + wave_scan(pieces);
    const uint64_t beyond = __ballot(upto > number);
    if (beyond) {
      const int i = __builtin_ctzll(beyond);
      prefix = c * MSPR_WAVE + i;
      blocks = __builtin_amdgcn_readlane(p.blocks, i);
      ranges = __builtin_amdgcn_readlane(p_ranges, i);
      before = __builtin_amdgcn_readlane(upto - pieces, i);
    } else {
      before = __builtin_amdgcn_readlane(upto, 63);
    }
  }
  if (prefix < 0 || number >= a.prefix_slots) return;  // (more workgroups than pieces)
  const int piece = number - before, bundles = n_kv * ranges;
  const int eights = piece / (8 * blocks), in_eights = piece - 8 * blocks * eights, wide = min(8, bundles - 8 * eights);
  const int block = __builtin_amdgcn_readfirstlane(in_eights / wide);
  const int bundle = 8 * eights + in_eights - block * wide;
  const int kvh = __builtin_amdgcn_readfirstlane(bundle / ranges), range = __builtin_amdgcn_readfirstlane(bundle - kvh * ranges);

  // ---- its queries: members block by block, as many in each as it takes to have them about equal
  const int members = __builtin_amdgcn_readfirstlane(count[prefix]);
  const int a_block = __builtin_amdgcn_readfirstlane(ceil_div(members, blocks));
  const int n_members = min(a_block, members - block * a_block);
  const int len = __builtin_amdgcn_readfirstlane(length[prefix]), n_tiles = ceil_div(len, kTileKeys);
  auto find_members = [&]() {
    const int per_row = ceil_div(batch, kWideThreads);
    const int r0 = min(t * per_row, batch), r1 = min(r0 + per_row, batch);
    int mine = 0;
    for (int r = r0; r < r1; r++) mine += row_group[r] == prefix;
    const int sum = wave_scan(mine);
    if (lane == 63) wave_members[wave] = sum;
    lds_barrier();
    int rank = sum - mine - block * a_block;
#pragma unroll
    for (int w = 0; w < kWideWaves; w++)
      if (w < wave) rank += wave_members[w];
    for (int r = r0; r < r1; r++)
      if (row_group[r] == prefix) {
        if (rank >= 0 && rank < a_block) {
          for (int h = 0; h < rep; h++) column_row[rank * rep + h] = (r * n_kv + kvh) * rep + h;
          if (range == 0) {
            int32_t* at = a.parts + 8 * ((int64_t)r * n_kv + kvh);
            at[2] = before;
            at[3] = ranges;
            at[4] = blocks;
            at[5] = block * a.block + rank * rep;
          }
        }
        rank++;
      }
    lds_barrier();
  };
  const int32_t* table = a.prefix_tables + (int64_t)prefix * a.prefix_width;
  const int tile0 = __builtin_amdgcn_readfirstlane((int)((int64_t)n_tiles * range / ranges));
  const int tile1 = __builtin_amdgcn_readfirstlane((int)((int64_t)n_tiles * (range + 1) / ranges));
  const int columns = __builtin_amdgcn_readfirstlane(n_members * rep);
  run(table, len, tile0, tile1, kvh, columns, find_members);
}

// A piece of a prefix of 16-bit rows a workgroup.
template <int FMT>
__global__ __launch_bounds__(kWideThreads, 1) void paged_prefix_kernel(const int32_t* requests, const int32_t* groups,
                                                                       const int32_t* prefix_lens, int batch, int n_prefixes,
                                                                       int n_tables, int n_kv, int rep, SharedRest a) {
  // (a name of its own: declarations of one name share an alignment, and the tiles' bases need zero low bits under the address XORs)
  extern __shared__ __attribute__((aligned(256))) unsigned char ring[];
  __shared__ int wave_members[kWideWaves];
  __shared__ int column_row[kWideColumns];
  __shared__ float xml[kWideWaves / 2][32][2];
  prefix_workgroup(requests, groups, prefix_lens, batch, n_prefixes, n_tables, n_kv, rep, a, kAtATime, ring + 2 * kStageBytes, wave_members, column_row,
                   [&](const int32_t* table, int len, int tile0, int tile1, int kvh, int columns, auto&& find_members) {
                     prefix_piece<FMT>(a, table, len, tile0, tile1, n_kv, kvh, blockIdx.x, columns, column_row, find_members, ring, xml);
                   });
}

// ---------------------------------------------------------------------------------------------- prefixes of 8-bit rows

// Sixteen columns a wave by 16x16x32 products of codes and queries, as paged_decode.hip makes them. Raw rows come by
// asynchronous copies into a ring of four tiles; the eight waves together make a tile's codes float16 numbers, a tile ahead of the
// one they multiply, so that what unpacking costs is shared. Scales and biases are read where the copies put them.
static_assert(kWideColumns == 16 * kWideWaves && kWideColumns == 32 * kWideWaves / kAtATime, "a block's columns are the waves'");
constexpr int kCodeTile = kTileKeys * kD;                  // 8 KB of codes, K and V each
constexpr int kScaleBytes = 256;                           // sixteen rows of scales or biases (of 16-bit ones half of it)
constexpr int kRawBytes = 2 * kCodeTile + 8 * kScaleBytes;
constexpr int kRawSlots = 4;
constexpr int kRawBase = 2 * kStageBytes;
constexpr int kCodeLds = kRawBase + kRawSlots * kRawBytes;  // 136 KB
constexpr int kCodeChunk = 28;                             // tiles whose pages a wave has at hand, with three more behind them

// Lane i's four bytes at base + offset land at lds_base + 4 i.
__device__ __forceinline__ void copy_4(uint64_t base, uint32_t offset, uint32_t lds_base) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %1, %0" ::"s"(base), "v"(offset), "s"(lds_base) : "memory", "m0");
}
// Sixteen-byte piece p of row r lies at place p ^ turn(r): eight rows' pieces, and four rows' pairs of pieces, on all banks.
__device__ __forceinline__ int turn(int r) { return ((r & 3) << 1) | (r >> 2 & 1); }

// Eight weights as two float16 terms each: the first cut off instead of rounded (half the instructions), which the second, a rounded
// rest of at most 2^-10 of the weight, makes up for.
__device__ __forceinline__ void cut_terms(const float* x, u32x4_t* t) {
  // (unknown to the compiler, which else makes two conversions and a difference of one mixed multiplication: 1.3 % of the call for 33
  // queries over 20001 rows; of 16-bit rows, whose kernel has fewer registers to spare, it cost 1.4 % for 61 ragged ones)
  float minus = -1.0f;
  asm("" : "+s"(minus));
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const h2_t h = __builtin_bit_cast(h2_t, __builtin_amdgcn_cvt_pkrtz(x[2 * j], x[2 * j + 1]));
    t[0][j] = h2_bits(h);
    const h2_t rest = {(_Float16)fmaf((float)h.x, minus, x[2 * j]), (_Float16)fmaf((float)h.y, minus, x[2 * j + 1])};
    t[1][j] = h2_bits(rest);
  }
}

template <int SDT>
__device__ __forceinline__ float scale_at(const unsigned char* region, int i) { return load_as_f32<SDT>(region, i); }

template <int QDT, int SDT, typename F>
__device__ __forceinline__ void codes_piece(const SharedRest& a, const int32_t* table, int len, int tile0, int tile1, int n_kv, int kvh,
                                            int slot, int columns, const int* column_row, F&& find_members, unsigned char* lds) {
  constexpr float kLag = 4.0f, kUp = 11.0f;           // (as in paged_decode.hip)
  constexpr int kQTerms = QDT == MSPR_F32 ? 2 : 1;
  constexpr int kSB = SDT == MSPR_F32 ? 4 : 2;
  constexpr int kCopies = 3;                           // of a wave and tile
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, g = lane >> 4;  // column of the wave's sixteen, key of the K operand; quarter of an operand's depth
  const int column0 = 16 * wave;
  const int mine = __builtin_amdgcn_readfirstlane(min(max(columns - column0, 0), 16));
  const int page_mask = (1 << a.page_shift) - 1;

  // ---- copies: a wave has a quarter of half a tile's K and V codes, and one of the four kinds of scales of that half
  const int half = wave >> 2, kind = wave & 3;
  const int c_row = (tid & 255) >> 4, s_row = kSB == 4 ? lane >> 2 : (lane & 31) >> 1;
  const uint64_t scales = (uint64_t)(kind == 0 ? a.k_scales : kind == 1 ? a.k_biases : kind == 2 ? a.v_scales : a.v_biases);
  const uint32_t raw0 = __builtin_amdgcn_readfirstlane(lds_address(lds)) + kRawBase;
  auto load_ids = [&](int t0) {  // lane i: page of half tile i from tile t0 on
    const int t = t0 + (lane >> 1), key = t * kTileKeys + 16 * (lane & 1);
    const int e = t < tile1 && key < len ? key >> a.page_shift : -1;
    return e >= 0 ? table[e] : -1;
  };
  // (rows that count, as of the 16-bit form; rows behind them are copies of the last, of half tiles without any codes and scales of zero)
  auto issue_tile = [&](int ids, int t0, int t) {
    uint32_t rows = 0;
    int64_t row = 0;
    int count = 0;
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const int page = __builtin_amdgcn_readlane(ids, 2 * (t - t0) + u);
      const int key = t * kTileKeys + 16 * u;
      const bool good = page >= 0 && page < a.n_pages && t < tile1;
      const int c = !good ? 0 : len - key >= 16 ? 16 : len - key < 0 ? 0 : len - key;
      if (u == half) {
        row = ((((int64_t)(good ? page : 0) * n_kv + kvh) << a.page_shift) + (key & page_mask));
        count = c;
      }
      rows |= (uint32_t)c << 8 * u;
    }
    const uint64_t none = (uint64_t)(const void*)g_no_rows;
    const uint64_t kb = count > 0 ? (uint64_t)a.k + row * kD : none, vb = count > 0 ? (uint64_t)a.v + row * kD : none;
    const uint64_t sb = count > 0 ? scales + row * 4 * kSB : none;
    const int last = max(count, 1) - 1;
    const uint32_t offset = (uint32_t)(min(c_row, last) * kD + (tid & 15) * 16);
    const uint32_t s_offset = (uint32_t)(min(s_row, last) * 4 * kSB + (lane & (kSB - 1)) * 4);
    const uint32_t to = raw0 + ((t - tile0) % kRawSlots) * kRawBytes;
    copy_16(kb, offset, to + wave * 1024);
    copy_16(vb, offset, to + kCodeTile + wave * 1024);
    copy_4(sb, s_offset, to + 2 * kCodeTile + (2 * kind + half) * kScaleBytes);
    return rows;
  };
  uint32_t ahead[4];  // rows of the present tile and of the three behind it
  int ids = load_ids(tile0);
#pragma unroll
  for (int i = 0; i < 3; i++) ahead[i] = issue_tile(ids, tile0, tile0 + i);
  int ids_next = load_ids(tile0 + kCodeChunk);
  find_members();  // (under the first copies)

  // ---- Q^T operands in registers: lane (n, g) has channels 32 s + 8 g on of step s, scaled by a power of two that brings the
  //      column's largest element to [2^14, 2^15) (float16 queries as they are)
  u32x4_t qf[8][kQTerms];
  float q_unit = a.scale_log2, qsum = 0.0f;  // (sums of the query over group g, for the biases)
  {
    constexpr int kWords = QDT == MSPR_F32 ? 2 : 1;
    u32x4_t raw[8][kWords];
    const int64_t row = column_row[column0 + n < columns ? column0 + n : 0];
#pragma unroll
    for (int s = 0; s < 8; s++)
#pragma unroll
      for (int w = 0; w < kWords; w++)
        raw[s][w] = reinterpret_cast<const u32x4_t*>(reinterpret_cast<const uint8_t*>(a.q) +
                                                     (row * kD + 32 * s + 8 * g) * (QDT == MSPR_F32 ? 4 : 2))[w];
    auto element = [&](int s, float* x) {
      if constexpr (QDT == MSPR_F32) {
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = __uint_as_float(raw[s][j / 4][j % 4]);
      } else {
        widen8<QDT>(raw[s][0], x);
      }
    };
    int e = 0;
    if constexpr (QDT != MSPR_F16) {
      float top = 0.0f;
#pragma unroll
      for (int s = 0; s < 8; s++) {
        float x[8];
        element(s, x);
#pragma unroll
        for (int j = 0; j < 8; j++) top = fmaxf(top, fabsf(x[j]));
      }
      top = half_wave_max(row_pair_max(top));
      if (top > 0.0f && top < __builtin_inff()) e = __builtin_amdgcn_frexp_expf(top) - 15;
    }
    float sums[4] = {};
#pragma unroll
    for (int s = 0; s < 8; s++) {
      float x[8];
      element(s, x);
#pragma unroll
      for (int j = 0; j < 8; j++) x[j] = __builtin_amdgcn_ldexpf(x[j], -e);
      split_terms<MSPR_F16, kQTerms>(x, qf[s]);
#pragma unroll
      for (int t = 0; t < kQTerms; t++) {  // (of the terms, as the products are)
        float y[8];
        widen8<MSPR_F16>(qf[s][t], y);
#pragma unroll
        for (int j = 0; j < 8; j++) sums[s / 2] += y[j];
      }
    }
    q_unit = __builtin_amdgcn_ldexpf(q_unit, e);
#pragma unroll
    for (int j = 0; j < 4; j++) {
      sums[j] += __shfl_xor(sums[j], 16, MSPR_WAVE);
      sums[j] += __shfl_xor(sums[j], 32, MSPR_WAVE);
    }
    qsum = g == 0 ? sums[0] : g == 1 ? sums[1] : g == 2 ? sums[2] : sums[3];
  }

  f32x4_t oacc[16], bacc = {0.f, 0.f, 0.f, 0.f};  // bacc: weighted biases, lane n (g = 0) has those of column n and the four groups
#pragma unroll
  for (int mt = 0; mt < 16; mt++) oacc[mt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  float m_run = -__builtin_inff(), l_run = 0.0f, v_unit = 0x1p-126f, per_unit = 0x1p126f;
  bool begun = false;

  // A tile's codes as float16 numbers, less 128: a thread has sixteen of K and of V in each eighth that its wave unpacks.
  auto unpack_part = [&](int i, int part) {
    int tl = lane + 64 * part;
    asm volatile("" : "+v"(tl));  // (offsets are made here, not carried through the loop)
    const unsigned char* raw = lds + kRawBase + (i % kRawSlots) * kRawBytes + tl * 16;
    const int row = tl >> 4, piece = 2 * (tl & 15), f = turn(row);
    unsigned char* to = lds + (i & 1) * kStageBytes + row * kRowBytes;
#pragma unroll
    for (int side = 0; side < 2; side++) {
      const u32x4_t c = *reinterpret_cast<const u32x4_t*>(raw + side * kCodeTile);
      u32x4_t p[2];
#pragma unroll
      for (int w = 0; w < 4; w++) {
        h2_t lo, hi;
        centred_to_h(c[w], lo, hi);
        p[w >> 1][2 * (w & 1)] = h2_bits(lo);
        p[w >> 1][2 * (w & 1) + 1] = h2_bits(hi);
      }
      *reinterpret_cast<u32x4_t*>(to + side * kTileBytes + 16 * (piece ^ f)) = p[0];
      *reinterpret_cast<u32x4_t*>(to + side * kTileBytes + 16 * ((piece + 1) ^ f)) = p[1];
    }
  };

  const int busy = (columns + 15) >> 4, idle = kWideWaves - busy;
  auto unpack = [&](int i) {
    if (idle == 0) {
      unpack_part(i, wave);
    } else {  // (waves without columns unpack for the others: 33 queries, of which six waves have 88 heads, 5 % of the call)
      for (int part = wave - busy; part >= 0 && part < kWideWaves; part += idle) unpack_part(i, part);
    }
  };

  const int k_off0 = n * kRowBytes + 16 * (g ^ turn(n)), k_off1 = n * kRowBytes + 16 * ((4 + g) ^ turn(n));  // + 8192 half + 128 group
  const int tr_row = 4 * g + (n >> 2);
  const uint32_t v_off = kTileBytes + tr_row * kRowBytes + 16 * (((n & 3) >> 1) ^ turn(tr_row)) + 8 * (n & 1);
  // K operands of half a tile: [step]
  auto read_k = [&](int i, int u, u32x4_t* kf) {
    const unsigned char* st = lds + (i & 1) * kStageBytes + 8192 * u;
#pragma unroll
    for (int s = 0; s < 8; s++) kf[s] = *reinterpret_cast<const u32x4_t*>(st + ((s & 1) ? k_off1 : k_off0) + 128 * (s >> 1));
  };
  auto attend_tile = [&](int i, uint32_t rows, u32x4_t (*kf)[8]) {
    const unsigned char* st = lds + (i & 1) * kStageBytes;
    const unsigned char* sc = lds + kRawBase + (i % kRawSlots) * kRawBytes + 2 * kCodeTile;
    // ---- S^T = K . Q^T: a group's sum takes its scale, biases are products with the query's sums
    float s[8];  // key 16 u + 4 g + i at 4 u + i
    read_k(i, 1, kf[1]);
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const f32x4_t zero = {0.f, 0.f, 0.f, 0.f};
      const float ksf = scale_at<SDT>(sc + u * kScaleBytes, 16 * g + n);
      const float bias = fmaf(128.0f, scale_at<SDT>(sc + u * kScaleBytes, 4 * n + g), scale_at<SDT>(sc + (2 + u) * kScaleBytes, 4 * n + g));
      f32x4_t acc[4];
#pragma unroll
      for (int j = 0; j < 4; j++) acc[j] = zero;
#pragma unroll
      for (int h = 0; h < 2; h++)
#pragma unroll
        for (int t = 0; t < kQTerms; t++)
#pragma unroll
          for (int j = 0; j < 4; j++) acc[j] = mfma<MSPR_F16>(kf[u][2 * j + h], qf[2 * j + h][t], acc[j]);
      f32x4_t sum = __builtin_amdgcn_mfma_f32_16x16x4f32(bias, qsum, zero, 0, 0, 0);
      static_for<4>([&](auto jc) {
        constexpr int j = decltype(jc)::value;
        static_for<4>([&](auto ic) {
          constexpr int k = decltype(ic)::value;
          sum[k] = fmaf(of_lane<4 * k + j>(ksf), acc[j][k], sum[k]);
        });
      });
#pragma unroll
      for (int k = 0; k < 4; k++) s[4 * u + k] = sum[k] * q_unit;
    }
    // ---- online softmax
    float tmax = -__builtin_inff();
    if (rows != 0x1010u) {
#pragma unroll
      for (int k = 0; k < 8; k++)
        if (4 * g + (k & 3) >= (int)(k < 4 ? rows & 0xFFu : rows >> 8)) s[k] = -__builtin_inff();
    }
#pragma unroll
    for (int k = 0; k < 8; k++) tmax = fmaxf(tmax, s[k]);
    tmax = half_wave_max(row_pair_max(tmax));
    const bool grow = tmax > m_run + kLag;
    if (__any(grow)) {
      const float m_new = grow ? tmax : m_run;
      if (begun) {
        const float alpha = grow ? __builtin_amdgcn_exp2f(m_run - m_new) : 1.0f;
        l_run *= alpha;
#pragma unroll
        for (int mt = 0; mt < 16; mt++) oacc[mt] = oacc[mt] * alpha;
        bacc = bacc * alpha;
      }
      m_run = m_new;
    }
    const float m_safe = (m_run == -__builtin_inff() ? 0.0f : m_run) - kUp;
#pragma unroll
    for (int k = 0; k < 8; k++) {
      s[k] = __builtin_amdgcn_exp2f(s[k] - m_safe);
      l_run += s[k];
    }
    // ---- O^T += V^T . P^T: weights take V's scales, as multiples of a power of two that is as large as any of their group
    float vsf[2], vbf[2];
#pragma unroll
    for (int u = 0; u < 2; u++) {
      vsf[u] = scale_at<SDT>(sc + (4 + u) * kScaleBytes, 16 * g + n);
      vbf[u] = fmaf(128.0f, vsf[u], scale_at<SDT>(sc + (6 + u) * kScaleBytes, 16 * g + n));
    }
    const float largest = fmaxf(fabsf(vsf[0]), fabsf(vsf[1]));
    if (__any(largest > v_unit)) {
      float top = largest;
      top = fmaxf(top, lane_xor<4>(top));
      top = fmaxf(top, lane_xor<8>(top));
      top = half_wave_max(row_pair_max(top));
      const int e = top < 0x1p126f ? __builtin_amdgcn_frexp_expf(top) : 126;
      const float unit = top > v_unit ? __builtin_amdgcn_ldexpf(1.0f, e) : v_unit;
      if (begun) {
        const float by = v_unit / unit;
        static_for<16>([&](auto mt) { oacc[mt] = oacc[mt] * of_lane<decltype(mt)::value / 4>(by); });
      }
      v_unit = unit;
      per_unit = 1.0f / unit;
    }
    begun = true;
    vsf[0] *= per_unit;
    vsf[1] *= per_unit;
    static_for<8>([&](auto ic) {
      constexpr int k = decltype(ic)::value;
      float bias = vbf[k >> 2];
      if constexpr ((k & 3) != 0)
        bias = __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(bias), 0x100 + 4 * (k & 3), 0xF, 0xF, true));  // row_shl
      bacc = __builtin_amdgcn_mfma_f32_16x16x4f32(bias, s[k], bacc, 0, 0, 0);
    });
    // (operands of the next group of channels are read while this one's weights are made)
    const uint32_t vb = lds_address(st) + v_off;
    u32x4_t vf[2][4];
    auto read_v = [&](int j) {
#pragma unroll
      for (int m = 0; m < 4; m++) {
        const uint32_t at = (vb ^ (uint32_t)(m << 5)) + 128 * j;
        const u32x2_t lo = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(MSPR_LDS_PTR(s16x4_t, (uintptr_t)at)));
        const u32x2_t hi =
            __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(MSPR_LDS_PTR(s16x4_t, (uintptr_t)(at + 16 * kRowBytes))));
        vf[j & 1][m] = u32x4_t{lo.x, lo.y, hi.x, hi.y};
      }
    };
    read_v(0);
    static_for<4>([&](auto jc) {  // the weights of group j, which has channels 64 j on
      constexpr int j = decltype(jc)::value;
      if constexpr (j < 3) read_v(j + 1);
      float w[8];
      static_for<8>([&](auto ic) {
        constexpr int k = decltype(ic)::value;
        w[k] = of_lane<4 * (k & 3) + j>(vsf[k >> 2]) * s[k];
        asm("" : "+v"(w[k]));  // (a rounded product, see paged_decode.hip)
      });
      u32x4_t pf[2];
      cut_terms(w, pf);
#pragma unroll
      for (int t = 0; t < 2; t++)
#pragma unroll
        for (int m = 0; m < 4; m++) oacc[4 * j + m] = mfma<MSPR_F16>(vf[j & 1][m], pf[t], oacc[4 * j + m]);
    });
  };

  // Steps of a wave: what tile i + 1 is made of has landed once its copies have (three a tile, in order) and every wave got here; the
  // stage and the slot of tile i - 1 are free then.
  wait_copies_and_barrier<2 * kCopies>();  // (and the plan, where the stages lie, is no longer read)
  unpack_part(0, wave);
  const int n_tiles = tile1 - tile0;
  for (int i0 = 0; i0 < n_tiles; i0 += kCodeChunk) {
    const int i_end = min(i0 + kCodeChunk, n_tiles);
    for (int i = i0; i < i_end; i++) {
      wait_copies_and_barrier<kCopies>();
      ahead[3] = issue_tile(ids, tile0 + i0, tile0 + i + 3);  // (behind the last, tiles without rows: what is under way is the same)
      u32x4_t kf[2][8];
      if (mine > 0) read_k(i, 0, kf[0]);  // (under the unpacking)
      if (i + 1 < n_tiles) unpack(i + 1);
      const uint32_t rows = ahead[0];
#pragma unroll
      for (int k = 0; k < 3; k++) ahead[k] = ahead[k + 1];
      if (mine > 0 && rows != 0) attend_tile(i, rows, kf);
    }
    ids = ids_next;
    ids_next = load_ids(tile0 + i0 + 2 * kCodeChunk);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (the last copies must not outlive the piece)

  // ---- a wave's columns leave in whole rows, through 16 KB of LDS
  __syncthreads();  // every wave has left the tiles
  if (mine == 0) return;
  l_run += __shfl_xor(l_run, 16, MSPR_WAVE);
  l_run += __shfl_xor(l_run, 32, MSPR_WAVE);
  float bias[4];
#pragma unroll
  for (int j = 0; j < 4; j++) bias[j] = __shfl(bacc[j], n, MSPR_WAVE);
  int row0 = slot * a.block + column0;  // (a scalar by hand, as of the 16-bit form)
  asm volatile("" : "+s"(row0));
  if (g == 0 && n < mine) *reinterpret_cast<f32x4_t*>(a.ws_pre_ml + 4 * (int64_t)(row0 + n)) = f32x4_t{m_run, l_run, 0.0f, 0.0f};
  unsigned char* xo = lds + (wave << 14);
  static_for<16>([&](auto mt) {
    constexpr int m = decltype(mt)::value;
    *reinterpret_cast<f32x4_t*>(xo + n * 1024 + 16 * ((4 * m + g) ^ n)) = oacc[m] * of_lane<m / 4>(v_unit) + bias[m / 4];
  });
  const auto to = store_window(a.ws_pre + (int64_t)row0 * kD, mine * kD * 4);
#pragma unroll
  for (int r = 0; r < 16; r++)
    window_store<kStoreThrough>(to, r * 1024 + 16 * lane, *reinterpret_cast<const u32x4_t*>(xo + r * 1024 + 16 * (lane ^ r)));
}

// A piece of a prefix of 8-bit rows a workgroup.
template <int QDT, int SDT>
__global__ __launch_bounds__(kWideThreads, 1) void paged_prefix_codes_kernel(const int32_t* requests, const int32_t* groups,
                                                                             const int32_t* prefix_lens, int batch, int n_prefixes,
                                                                             int n_tables, int n_kv, int rep, SharedRest a) {
  extern __shared__ __attribute__((aligned(256))) unsigned char ring[];
  __shared__ int wave_members[kWideWaves];
  __shared__ int column_row[kWideColumns];
  prefix_workgroup(requests, groups, prefix_lens, batch, n_prefixes, n_tables, n_kv, rep, a, 1, ring, wave_members, column_row,
                   [&](const int32_t* table, int len, int tile0, int tile1, int kvh, int columns, auto&& find_members) {
                     codes_piece<QDT, SDT>(a, table, len, tile0, tile1, n_kv, kvh, blockIdx.x, columns, column_row, find_members, ring);
                   });
}

constexpr int kAtOnce = 16;  // pieces that a wave joins at a time
typedef __attribute__((address_space(1))) u32x4_t global_quads_t;

// Joins the pieces of one query head: WAVES of them a head take every WAVES-th, and meet in LDS. PARTS: own rows are
// paged_decode.hip's parts (own: of rows that are not cut), else pieces of paged_shared_kernel.
// grid: heads / (kMergeWaves / WAVES)
constexpr int kMergeWaves = 8;
template <int ODT, int WAVES, bool PARTS>
__global__ __launch_bounds__(64 * kMergeWaves) void paged_shared_merge_kernel(const int32_t* parts, const int32_t* cuts, int rep, int n_kv,
                                                                              int rows, int block, int prefix_slots, int own_slots,
                                                                              int shares, bool cut_rows, const float* ws_pre, const float* ws_pre_ml,
                                                                              const float* ws_own, const float* ws_own_ml,
                                                                              const float* part_o, const float* part_ml, void* out) {
  __shared__ __attribute__((aligned(16))) float xo[kMergeWaves][kD + 2];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int head = (int)blockIdx.x * (kMergeWaves / WAVES) + wave / WAVES;
  const int part = wave % WAVES;
  const bool here = head < rows * rep;
  const int row = here ? head / rep : 0, hn = here ? head - row * rep : 0;
  // (both entries of the row are read at once, whether it has a cut or not: waits one behind the other are what this kernel's time
  // is made of)
  const int32_t* at = parts + 8 * (int64_t)row;
  const int own_first = PARTS ? 0 : at[0], own_count = at[1], pre_first = at[2], pre_ranges = at[3], blocks = at[4], column = at[5] + hn;
  Cut cut = {-1, 0, 0};
  if constexpr (PARTS) cut.load(cuts, row, rows, shares);
  const bool is_cut = PARTS && cut_rows && cut.count > 0;
  const int n_own = !here ? 0 : !PARTS ? own_count : is_cut ? cut.count : 1, ranges = here ? pre_ranges : 0;
  const int total = n_own + ranges;
  const int kvh = row % n_kv, column_block = column / block, column_at = column - column_block * block;
  struct From {
    const float *o, *ml;
  };
  // Sums and statistics of own piece i, of prefix piece i (bounded by the workspace, whatever is there)
  auto own_piece = [&](int i) {
    if (is_cut) {
      const int64_t p = part_of(cut.first, i);
      return From{part_o + (p * rep + hn) * kD, part_ml + (p * 16 + hn) * 2};
    }
    if constexpr (PARTS) return From{ws_own + (int64_t)head * kD, ws_own_ml + (int64_t)head * 2};
    const int s = own_first + i >= 0 && own_first + i < own_slots ? own_first + i : 0;
    return From{ws_own + ((int64_t)s * rep + hn) * kD, ws_own_ml + ((int64_t)s * 16 + hn) * 2};
  };
  auto prefix_piece = [&](int i) {
    const int s = pre_first + bundle_piece(kvh * ranges + i, column_block, n_kv * ranges, blocks);
    const int64_t r = (int64_t)(s >= 0 && s < prefix_slots ? s : 0) * block + column_at;
    return From{ws_pre + r * kD, ws_pre_ml + 4 * r};
  };
  float m = -__builtin_inff(), l = 0.0f;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  for (int p0 = part; p0 < total; p0 += kAtOnce * WAVES) {
    // Lane j finds piece j, of those past the end the last. (One load of either kind of piece, so that none waits for the other.)
    const int mine = p0 + WAVES * (lane % kAtOnce), near = min(mine, total - 1);
    const From from = near >= n_own ? prefix_piece(near - n_own) : own_piece(near);
    f32x2_t stat = *reinterpret_cast<const f32x2_t*>(from.ml);
    if (mine >= total) stat = f32x2_t{-__builtin_inff(), 0.0f};
    const uint64_t o_at = reinterpret_cast<uint64_t>(from.o);
    u32x4_t ov[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; j++) {  // (wave-uniform: pieces past the end cost no load)
      const int i = p0 + WAVES * j;
      if (i >= total) continue;
      const uint64_t o_j = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)o_at, j) |
                           (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(o_at >> 32), j) << 32;
      ov[j] = reinterpret_cast<const global_quads_t*>(o_j)[lane];
    }
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
    for (int j = 0; j < kAtOnce; j++) {
      const int i = p0 + WAVES * j;
      if (i >= total) continue;
      o += __builtin_bit_cast(f32x4_t, ov[j]) * __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), j));
    }
    m = m_new;
  }
  if constexpr (WAVES > 1) {
    if (lane == 0) {
      xo[wave][kD] = m;
      xo[wave][kD + 1] = l;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) xo[wave][4 * lane + i] = o[i];
    __syncthreads();
    if (part != 0) return;
    float m_all = -__builtin_inff();
#pragma unroll
    for (int w = 0; w < WAVES; w++) m_all = fmaxf(m_all, xo[wave + w][kD]);
    const float m_safe = m_all == -__builtin_inff() ? 0.0f : m_all;
    l = 0.0f;
    o = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < WAVES; w++) {
      const float wt = __builtin_amdgcn_exp2f(xo[wave + w][kD] - m_safe);
      l += xo[wave + w][kD + 1] * wt;
#pragma unroll
      for (int i = 0; i < 4; i++) o[i] += xo[wave + w][4 * lane + i] * wt;
    }
  }
  if (total > 0) store_out<ODT>(out, ((int64_t)row * rep + hn) * kD + 4 * lane, o, l);
}

// Whether prefixes are a kernel's own: from so many columns times rows that their tables hold (the lengths are on the device) on, and of
// many columns always. A second kernel costs 9 to 11 us; blocks of 32 columns read a prefix again and again, and own rows of many
// queries are better dealt out by paged_decode.hip. In us a call of a captured graph, one launch and two, two KV heads of 8 query heads: 16-bit
// rows, 8 queries over 32768 rows 36.1 and 37.2, 12 over them 44.9 and 40.6; 32 over 4000 29.2 and 38.7, 128 over 1000 43.3 and 49.3, 256 over
// 1000 65.4 either way; 20 ragged ones behind 5 prefixes of up to 9001 33.4 and 38.9, 40 such 59.3 and 51.0. 8-bit rows: 24 queries over 20000
// rows 59.7 and 61.9, 32 over them 77.3 and 67.6, 48 over 4000 47.6 and 50.0, 96 over 1000 34.0 and 50.1, 200 over 1000 52.0 and 55.6. The number of
// KV heads is not in the rule, though with more of them two launches are better earlier: eight of 4 query heads, 16 queries over 4096 rows 32.6
// and 33.1, 32 over them 44.8 and 42.0, 16 over 16384 rows 73.6 and 52.2, 32 over them 127 and 69, where the rule takes one launch.
constexpr int kManyColumns = 1024;
bool wide_prefixes(int batch, int rep, int64_t prefix_cap, bool codes) {
  const int64_t columns = (int64_t)batch * rep;
  return columns > kManyColumns || (columns > kColumns && columns * prefix_cap >= (codes ? 4 << 20 : 5 << 19));
}

// Columns of a block of members: 32, or as many as eight waves hold, but no more than twice what a prefix has members on the
// average, so that the scratch, a place for every column of a block, does not grow with what blocks leave empty.
int block_columns(int batch, int n_prefixes, int rep, bool wide) {
  if (!wide) return kColumns;
  const int64_t used = n_prefixes < batch ? n_prefixes : batch;
  const int64_t mean = ((used > 1 ? 2 : 1) * (int64_t)batch * rep + used - 1) / used;
  const int64_t n = (mean + 31) / 32 * 32;
  return (int)(n < kWideColumns ? n : kWideColumns);
}

// Pieces of `units` units: a call has at most max(kGroups, kGroups / 2 + units), see `share`.
int64_t pieces_of(int64_t units) { return kGroups / 2 + units > kGroups ? kGroups / 2 + units : kGroups; }

// Blocks of members, at most (every prefix may have one that is not full), of every KV head.
int64_t prefix_units(int batch, int n_prefixes, int n_kv, int rep, int block) {
  const int rows_a_block = block / rep;
  const int used = n_prefixes < batch ? n_prefixes : batch;
  return (int64_t)n_kv * ((batch + (int64_t)used * (rows_a_block - 1)) / rows_a_block);
}

struct SharedScratch {
  bool wide;
  int block;
  int64_t pieces;                                  // workgroups: of prefixes, and of own rows where one launch has both
  int64_t prefix_slots, own_slots;                 // places for partials; wide: own_slots query heads
  size_t pre, pre_ml, own, own_ml, parts, decode;  // bytes
  size_t total() const { return pre + pre_ml + own + own_ml + parts + decode; }
};
SharedScratch shared_scratch(int batch, int n_prefixes, int n_kv, int rep, int page_size, int width, bool wide) {
  SharedScratch s;
  s.wide = wide;
  s.block = block_columns(batch, n_prefixes, rep, s.wide);
  const int64_t own = (int64_t)batch * n_kv, blocks = prefix_units(batch, n_prefixes, n_kv, rep, s.block);
  s.pieces = pieces_of(s.wide ? blocks : own + blocks);
  s.prefix_slots = s.wide ? s.pieces : s.pieces - own;  // (every query has a piece of its own, at least)
  s.own_slots = s.wide ? own * rep : pieces_of(own);
  s.pre = (size_t)s.prefix_slots * s.block * kD * sizeof(float);
  s.pre_ml = (size_t)s.prefix_slots * s.block * 4 * sizeof(float);
  s.own = (size_t)s.own_slots * (s.wide ? 1 : rep) * kD * sizeof(float);
  s.own_ml = ((size_t)s.own_slots * (s.wide ? 1 : 16) * 2 * sizeof(float) + 15) / 16 * 16;
  s.parts = (size_t)own * 8 * sizeof(int32_t);
  s.decode = s.wide ? mspr_sdpa_decode_paged_workspace_bytes(batch, n_kv * rep, n_kv, page_size, width) : 0;
  return s;
}

// The LDS of a kernel beyond what every launch may have, asked for once a device.
template <typename K>
int reserve_lds(K* kernel, int bytes, bool (&done)[64]) {
  int device = 0;
  if (hipGetDevice(&device) != hipSuccess || device < 0 || device >= 64 || !done[device]) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != hipSuccess) {
      mspr_set_error("sdpa_decode_paged_shared: cannot reserve %d bytes of LDS: %s", bytes, hipGetErrorString(e));
      return MSPR_ERR_LAUNCH;
    }
    if (device >= 0 && device < 64) done[device] = true;
  }
  return MSPR_OK;
}

// Joins the pieces of `heads` query heads: eight waves a head where they are few and have many pieces, else one. (In us, with eight and with
// one: 256 heads of 129 pieces 44.4 and 50.1 the call, 1024 of 33 85.4 and 84.1, 2048 137.5 and 135.3, 4096 116.6 and 109.9.)
template <int QDT, bool PARTS>
int merge_launch(const SharedArgs& a, const PagedParts& own, hipStream_t st) {
  const SharedRest& r = a.rest;
  const int heads = a.batch * a.n_kv * a.rep;
  auto merge = [&](auto waves) {
    constexpr int kWavesAHead = decltype(waves)::value, kHeads = kMergeWaves / kWavesAHead;
    paged_shared_merge_kernel<QDT, kWavesAHead, PARTS><<<dim3((unsigned)((heads + kHeads - 1) / kHeads)), dim3(64 * kMergeWaves), 0, st>>>(
        r.parts, own.cut ? own.cut : r.parts, a.rep, a.n_kv, a.batch * a.n_kv, r.block, r.prefix_slots, r.own_slots, own.shares,
        own.cut != nullptr, r.ws_pre, r.ws_pre_ml, r.ws_own, r.ws_own_ml, own.o, own.ml, r.out);
  };
  // (a head has as many pieces as compute units divided by blocks: few where heads are many)
  if (heads <= 1024) merge(std::integral_constant<int, 8>{});
  else merge(std::integral_constant<int, 1>{});
  MSPR_CHECK_LAUNCH("sdpa_decode_paged_shared (merge)");
  return MSPR_OK;
}

template <int QDT, int FMT, int SDT>
int shared_launch(const SharedArgs& a, hipStream_t st) {
  constexpr int kLds = shared_lds(QDT, FMT);
  static bool reserved[64] = {};
  if (int rc = reserve_lds(&paged_shared_kernel<QDT, FMT, SDT>, kLds, reserved)) return rc;
  paged_shared_kernel<QDT, FMT, SDT><<<dim3((unsigned)a.pieces), dim3(kThreads), kLds, st>>>(
      a.requests, a.groups, a.lens, a.prefix_lens, a.batch, a.n_prefixes, a.n_tables, a.n_kv, a.rep, a.rest);
  MSPR_CHECK_LAUNCH("sdpa_decode_paged_shared");
  return merge_launch<QDT, false>(a, PagedParts{}, st);
}

// Own rows, then prefixes by `kernel`.
template <int QDT, typename K>
int wide_launch(const char* what, const SharedArgs& a, int sb_dtype, K* kernel, int lds, bool (&reserved)[64], hipStream_t st) {
  if (int rc = reserve_lds(kernel, lds, reserved)) return rc;
  const SharedRest& r = a.rest;
  PagedPartsCall c = {};
  c.q = r.q;
  c.k = r.k;
  c.v = r.v;
  c.k_scales = r.k_scales;
  c.k_biases = r.k_biases;
  c.v_scales = r.v_scales;
  c.v_biases = r.v_biases;
  c.q_dtype = QDT;
  c.sb_dtype = sb_dtype;
  c.tables = r.tables;
  c.lens = a.lens;
  c.requests = a.requests;
  c.batch = a.batch;
  c.n_kv = a.n_kv;
  c.rep = a.rep;
  c.n_pages = r.n_pages;
  c.page_shift = r.page_shift;
  c.n_tables = a.n_tables;
  c.width = r.width;
  c.scale_log2 = r.scale_log2;
  c.own = r.ws_own;
  c.own_ml = r.ws_own_ml;
  c.workspace = a.decode;
  c.workspace_bytes = a.decode_bytes;
  PagedParts own;
  if (int rc = mspr_paged_decode_parts(what, c, &own, st)) return rc;
  kernel<<<dim3((unsigned)a.pieces), dim3(kWideThreads), lds, st>>>(a.requests, a.groups, a.prefix_lens, a.batch, a.n_prefixes, a.n_tables,
                                                                    a.n_kv, a.rep, r);
  MSPR_CHECK_LAUNCH("sdpa_decode_paged_shared (prefixes)");
  return merge_launch<QDT, true>(a, own, st);
}
template <int FMT>
int rows_launch(const SharedArgs& a, hipStream_t st) {
  static bool reserved[64] = {};
  if (!a.wide) return shared_launch<FMT, FMT, FMT>(a, st);
  return wide_launch<FMT>("sdpa_decode_paged_shared", a, FMT, &paged_prefix_kernel<FMT>, kWideLds, reserved, st);
}
template <int QDT, int SDT>
int codes_launch(const SharedArgs& a, hipStream_t st) {
  static bool reserved[64] = {};
  if (!a.wide) return shared_launch<QDT, kAffine, SDT>(a, st);
  return wide_launch<QDT>("sdpa_decode_paged_shared_q8", a, SDT, &paged_prefix_codes_kernel<QDT, SDT>, kCodeLds, reserved, st);
}

int shared_fill(const char* what, SharedArgs& a, bool codes, const void* q, const void* k, const void* v, const int32_t* prefix_tables,
                const int32_t* prefix_lens, const int32_t* groups, const int32_t* tables, const int32_t* lens,
                const int32_t* requests, int batch, int n_q_heads, int n_kv_heads, int head_dim, int n_pages, int page_size,
                int n_prefixes, int prefix_width, int n_tables, int table_width, float scale, void* out, void* workspace,
                size_t workspace_bytes) {
  MSPR_REQUIRE(q && k && v && prefix_tables && prefix_lens && groups && tables && lens && out, "%s: null pointer", what);
  MSPR_REQUIRE(head_dim == kD, "%s: head_dim must be 256", what);
  MSPR_REQUIRE(batch >= 1 && batch <= kMaxRows, "%s: 1 to %d queries", what, kMaxRows);
  MSPR_REQUIRE(n_prefixes >= 1 && n_prefixes <= kMaxRows, "%s: 1 to %d prefixes", what, kMaxRows);
  MSPR_REQUIRE(n_tables >= 1 && (requests || n_tables == batch), "%s: a table for every query, or the requests they belong to",
               what);
  MSPR_REQUIRE(n_kv_heads >= 1 && n_kv_heads <= 1024 && n_q_heads >= n_kv_heads && n_q_heads % n_kv_heads == 0,
               "%s: bad head counts", what);
  MSPR_REQUIRE(n_q_heads / n_kv_heads <= 16, "%s: at most 16 query heads per KV head", what);
  MSPR_REQUIRE(page_size >= 16 && (page_size & (page_size - 1)) == 0, "%s: page_size must be a power of two from 16 on", what);
  MSPR_REQUIRE(n_pages >= 1 && (int64_t)n_pages * page_size <= 0x7FFFFFFF, "%s: the pool must hold fewer than 2^31 tokens", what);
  MSPR_REQUIRE(table_width >= 1 && (int64_t)table_width * page_size <= 0x40000000 && prefix_width >= 1 &&
                   (int64_t)prefix_width * page_size <= 0x40000000,
               "%s: a table must hold 1 page or more and at most 2^30 tokens", what);
  const int rep = n_q_heads / n_kv_heads;
  const int64_t most = (int64_t)table_width * page_size > (int64_t)prefix_width * page_size ? (int64_t)table_width * page_size
                                                                                           : (int64_t)prefix_width * page_size;
  const SharedScratch s = shared_scratch(batch, n_prefixes, n_kv_heads, rep, page_size, table_width,
                                         wide_prefixes(batch, rep, (int64_t)prefix_width * page_size, codes));
  MSPR_REQUIRE((prefix_units(batch, n_prefixes, n_kv_heads, rep, s.block) + (int64_t)batch * n_kv_heads) * ((most + kTileKeys - 1) / kTileKeys + 1) <= 0x3FFFFFFF,
               "%s: the tables hold too many tokens together", what);
  MSPR_REQUIRE(mspr_aligned(q, 16) && mspr_aligned(k, 16) && mspr_aligned(v, 16) && mspr_aligned(out, 16),
               "%s: pointers must be 16-byte aligned", what);
  MSPR_REQUIRE(workspace && workspace_bytes >= s.total() && mspr_aligned(workspace, 16),
               "%s: workspace of %zu bytes (16-byte aligned) needed, %zu given", what, s.total(), workspace_bytes);
  a = SharedArgs{};
  a.requests = requests;
  a.groups = groups;
  a.lens = lens;
  a.prefix_lens = prefix_lens;
  a.batch = batch;
  a.n_prefixes = n_prefixes;
  a.n_tables = n_tables;
  a.n_kv = n_kv_heads;
  a.rep = rep;
  a.pieces = (int)s.pieces;
  a.wide = s.wide;
  a.decode_bytes = s.decode;
  SharedRest& r = a.rest;
  r.q = q;
  r.k = k;
  r.v = v;
  r.prefix_tables = prefix_tables;
  r.tables = tables;
  r.n_pages = n_pages;
  r.page_shift = __builtin_ctz(page_size);
  r.prefix_width = prefix_width;
  r.width = table_width;
  r.prefix_slots = (int)s.prefix_slots;
  r.own_slots = (int)s.own_slots;
  r.block = s.block;
  r.scale_log2 = (float)((double)scale * 1.4426950408889634);
  uint8_t* at = reinterpret_cast<uint8_t*>(workspace);
  r.ws_pre = reinterpret_cast<float*>(at);
  r.ws_pre_ml = reinterpret_cast<float*>(at += s.pre);
  r.ws_own = reinterpret_cast<float*>(at += s.pre_ml);
  r.ws_own_ml = reinterpret_cast<float*>(at += s.own);
  r.parts = reinterpret_cast<int32_t*>(at += s.own_ml);
  a.decode = at + s.parts;
  r.out = out;
  return MSPR_OK;
}

template <int QDT>
int shared_q8_launch(const SharedArgs& a, int sb_dtype, hipStream_t st) {
  if (sb_dtype == MSPR_F32) return codes_launch<QDT, MSPR_F32>(a, st);
  if (sb_dtype == MSPR_F16) return codes_launch<QDT, MSPR_F16>(a, st);
  return codes_launch<QDT, MSPR_BF16>(a, st);
}

}  // namespace

// (of both forms, whichever needs more: which it is depends on the prefixes' tables too)
extern "C" size_t mspr_sdpa_decode_paged_shared_workspace_bytes(int batch, int n_q_heads, int n_kv_heads, int page_size,
                                                                int table_width, int n_prefixes) {
  if (batch < 1 || n_kv_heads < 1 || n_q_heads < n_kv_heads || n_q_heads / n_kv_heads > 16 || n_prefixes < 1 || page_size < 1 ||
      table_width < 1)
    return 0;
  const int rep = n_q_heads / n_kv_heads;
  const size_t narrow = shared_scratch(batch, n_prefixes, n_kv_heads, rep, page_size, table_width, false).total();
  if ((int64_t)batch * rep <= kColumns) return narrow;
  const size_t wide = shared_scratch(batch, n_prefixes, n_kv_heads, rep, page_size, table_width, true).total();
  return narrow > wide ? narrow : wide;
}

extern "C" int mspr_sdpa_decode_paged_shared(const void* queries, const void* k_pages, const void* v_pages, int dtype,
                                             const int32_t* prefix_tables, const int32_t* prefix_lens, const int32_t* groups,
                                             const int32_t* tables, const int32_t* lens, const int32_t* requests, int batch,
                                             int n_q_heads, int n_kv_heads, int head_dim, int n_pages, int page_size,
                                             int n_prefixes, int prefix_width, int n_tables, int table_width, float scale,
                                             void* out, void* workspace, size_t workspace_bytes, void* stream) {
  MSPR_REQUIRE(dtype == MSPR_F16 || dtype == MSPR_BF16, "sdpa_decode_paged_shared: dtype must be f16 or bf16");
  SharedArgs a;
  if (int rc = shared_fill("sdpa_decode_paged_shared", a, false, queries, k_pages, v_pages, prefix_tables, prefix_lens, groups, tables,
                           lens, requests, batch, n_q_heads, n_kv_heads, head_dim, n_pages, page_size, n_prefixes, prefix_width,
                           n_tables, table_width, scale, out, workspace, workspace_bytes))
    return rc;
  hipStream_t st = (hipStream_t)stream;
  return dtype == MSPR_F16 ? rows_launch<MSPR_F16>(a, st) : rows_launch<MSPR_BF16>(a, st);
}

extern "C" int mspr_sdpa_decode_paged_shared_q8(const void* queries, int q_dtype, const void* k_wq, const void* k_scales,
                                                const void* k_biases, const void* v_wq, const void* v_scales,
                                                const void* v_biases, int sb_dtype, const int32_t* prefix_tables,
                                                const int32_t* prefix_lens, const int32_t* groups, const int32_t* tables,
                                                const int32_t* lens, const int32_t* requests, int batch, int n_q_heads,
                                                int n_kv_heads, int head_dim, int n_pages, int page_size, int n_prefixes,
                                                int prefix_width, int n_tables, int table_width, float scale, int group_size,
                                                int bits, void* out, void* workspace, size_t workspace_bytes, void* stream) {
  MSPR_REQUIRE(group_size == 64 && bits == 8, "sdpa_decode_paged_shared_q8: only group_size=64, bits=8 is supported");
  MSPR_REQUIRE(q_dtype >= MSPR_F32 && q_dtype <= MSPR_BF16, "sdpa_decode_paged_shared_q8: queries must be f32, f16 or bf16");
  MSPR_REQUIRE(sb_dtype >= MSPR_F32 && sb_dtype <= MSPR_BF16, "sdpa_decode_paged_shared_q8: scales must be f32, f16 or bf16");
  MSPR_REQUIRE(k_scales && k_biases && v_scales && v_biases, "sdpa_decode_paged_shared_q8: null pointer");
  MSPR_REQUIRE(mspr_aligned(k_scales, 16) && mspr_aligned(k_biases, 16) && mspr_aligned(v_scales, 16) &&
                   mspr_aligned(v_biases, 16),
               "sdpa_decode_paged_shared_q8: pointers must be 16-byte aligned");
  SharedArgs a;
  if (int rc = shared_fill("sdpa_decode_paged_shared_q8", a, true, queries, k_wq, v_wq, prefix_tables, prefix_lens, groups, tables, lens,
                           requests, batch, n_q_heads, n_kv_heads, head_dim, n_pages, page_size, n_prefixes, prefix_width,
                           n_tables, table_width, scale, out, workspace, workspace_bytes))
    return rc;
  a.rest.k_scales = k_scales;
  a.rest.k_biases = k_biases;
  a.rest.v_scales = v_scales;
  a.rest.v_biases = v_biases;
  hipStream_t st = (hipStream_t)stream;
  if (q_dtype == MSPR_F32) return shared_q8_launch<MSPR_F32>(a, sb_dtype, st);
  if (q_dtype == MSPR_F16) return shared_q8_launch<MSPR_F16>(a, sb_dtype, st);
  return shared_q8_launch<MSPR_BF16>(a, sb_dtype, st);
}
