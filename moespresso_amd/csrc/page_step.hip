// Tables of one step of a paged cache, from the requests' lengths.
//
// The pages of a pool that no request holds lie on a stack (`free_pages` from `head` on). A step gives every request the
// pages that its new rows begin, takes those of ended requests back first, and names a slot (page * page_size + row in the
// page) for every new row. Four running sums over the requests decide everything: rows asked for, pages needed, pages given
// back; each page that moves and each row then finds its request by bisection of a sum.
//
// Bound by latency: a step of 16 requests reads 128 bytes and writes 500. One launch; every workgroup makes the sums anew
// (2048 requests are two a thread) rather than wait for another's, and writes its share of the rows. What one workgroup
// writes no other reads: pages given back go below `head` and pages taken from there are read where they come from, the table
// of the ended request; new table entries lie behind those that rows of the last started page read.
#include "common.h"

namespace {

constexpr int kMaxRequests = 2048;  // (five sums of them in 40 KB of LDS)

struct StepArgs {
  const int32_t* lens;
  const int32_t* add;
  int32_t* tables;
  int32_t* free_pages;
  const int32_t* head;
  int batch, width, n_pages, page_shift, n_rows;
  int32_t* lens_out;
  int32_t* head_out;
  int32_t* starts;
  int32_t* slots;
  int32_t* positions;
  int32_t* visible;
  int32_t* requests;
  int32_t* counts;
};

// a + b of values from 0 on, at most 2^31 - 1: asked-for rows may add up to more
__device__ __forceinline__ int sat_add(int a, int b) {
  const uint32_t s = (uint32_t)a + (uint32_t)b;
  return s > 0x7FFFFFFFu ? 0x7FFFFFFF : (int)s;
}

// Sums of `v` over the threads before this one, and of all of them in `total`.
template <int THREADS>
__device__ __forceinline__ int block_scan(int v, int* wave_sums, int& total) {
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  int s = v;
#pragma unroll
  for (int m = 1; m < MSPR_WAVE; m <<= 1) {
    const int o = __shfl_up(s, m, MSPR_WAVE);
    if (lane >= m) s = sat_add(s, o);
  }
  if (lane == 63) wave_sums[wave] = s;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / MSPR_WAVE; w++) {
    if (w == wave) before = total;
    total = sat_add(total, wave_sums[w]);
  }
  const int up = __shfl_up(s, 1, MSPR_WAVE);
  return sat_add(before, lane == 0 ? 0 : up);
}

// The last index in [0, n) whose sum is at most x (sums ascend, sums[0] = 0).
__device__ __forceinline__ int last_at_most(const int* sums, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (sums[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// grid: workgroups that share rows and returned pages; LDS: five arrays of `batch` integers
template <int THREADS, int ITEMS>
__global__ __launch_bounds__(THREADS) void page_step_kernel(StepArgs a) {
  extern __shared__ int lds[];
  __shared__ int wave_sums[3][THREADS / MSPR_WAVE];
  const int tid = threadIdx.x;
  const int B = a.batch;
  int* s_start = lds;           // first row
  int* s_first = lds + B;       // pages needed by the requests before
  int* s_back = lds + 2 * B;    // pages given back by the requests before
  int* s_old = lds + 3 * B;     // length before
  int* s_len = lds + 4 * B;     // length after
  const int page = 1 << a.page_shift;
  const int cap = a.width << a.page_shift;

  int old_[ITEMS], add_[ITEMS];
  int rows = 0;
#pragma unroll
  for (int i = 0; i < ITEMS; i++) {
    const int b = tid * ITEMS + i;
    old_[i] = b < B ? a.lens[b] : 0;
    add_[i] = b < B ? a.add[b] : 0;
  }
  int head = *a.head;
  head = head < 0 ? 0 : head > a.n_pages ? a.n_pages : head;
#pragma unroll
  for (int i = 0; i < ITEMS; i++) {
    old_[i] = old_[i] < 0 ? 0 : old_[i] > cap ? cap : old_[i];
    rows = sat_add(rows, add_[i] > 0 ? add_[i] : 0);
  }
  int all_rows, all_need, all_back;
  int start = block_scan<THREADS>(rows, wave_sums[0], all_rows);
  // rows behind n_rows are not part of the step: what a request may add ends there, and at its table's end
  int start_[ITEMS], goal_[ITEMS], need = 0, back = 0;
#pragma unroll
  for (int i = 0; i < ITEMS; i++) {
    const int asked = add_[i] > 0 ? add_[i] : 0;
    start_[i] = start < a.n_rows ? start : a.n_rows;
    const int room = a.n_rows - start_[i];
    goal_[i] = old_[i] + min(min(asked, room), cap - old_[i]);
    start = sat_add(start, asked);
    const int held = (old_[i] + page - 1) >> a.page_shift;
    if (add_[i] < 0) back += held;
    else need += ((goal_[i] + page - 1) >> a.page_shift) - held;
  }
  int first = block_scan<THREADS>(need, wave_sums[1], all_need);
  int given = block_scan<THREADS>(back, wave_sums[2], all_back);
  const int base = head - all_back;  // the stack's new top, before pages are taken (below 0 only if pages were lent twice)
  const int avail = a.n_pages - base;
  int placed = 0;
#pragma unroll
  for (int i = 0; i < ITEMS; i++) {
    const int b = tid * ITEMS + i;
    const int held = (old_[i] + page - 1) >> a.page_shift;
    const bool ended = add_[i] < 0;
    const int want = ended ? 0 : ((goal_[i] + page - 1) >> a.page_shift) - held;
    const int got = max(0, min(want, avail - first));
    const int len = ended ? 0 : got == want ? goal_[i] : (held + got) << a.page_shift;
    if (b < B) {
      s_start[b] = start_[i];
      s_first[b] = first;
      s_back[b] = given;
      s_old[b] = old_[i];
      s_len[b] = len;
      if (blockIdx.x == 0) {
        a.lens_out[b] = len;
        a.starts[b] = start_[i];
        if (!ended) placed += len - old_[i];
      }
    }
    first += want;
    given += ended ? held : 0;
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    int all_placed;
    block_scan<THREADS>(placed, wave_sums[0], all_placed);
    if (tid == 0) {
      const int taken = max(0, min(all_need, avail));
      const int top = base + taken;
      a.starts[B] = min(all_rows, a.n_rows);
      *a.head_out = top < 0 ? 0 : top;
      a.counts[0] = all_rows;
      a.counts[1] = all_rows - all_placed;
      a.counts[2] = taken;
      a.counts[3] = all_back;
    }
  }

  const int stride = gridDim.x * THREADS;
  for (int k = blockIdx.x * THREADS + tid; k < all_back; k += stride) {
    const int b = last_at_most(s_back, B, k);
    const int at = base + k;
    if (at >= 0) a.free_pages[at] = a.tables[(int64_t)b * a.width + (k - s_back[b])];
  }
  for (int t = blockIdx.x * THREADS + tid; t < a.n_rows; t += stride) {
    int slot = -1, position = 0, request = -1;
    if (t < all_rows) {
      const int b = last_at_most(s_start, B, t);
      const int old = s_old[b];
      request = b;
      position = old + (t - s_start[b]);
      if (position < s_len[b]) {
        const int held = (old + page - 1) >> a.page_shift;
        const int i = position >> a.page_shift;
        int p;
        if (i < held) {
          p = a.tables[(int64_t)b * a.width + i];
        } else {
          const int k = s_first[b] + (i - held);
          if (k < all_back) {
            const int from = last_at_most(s_back, B, k);
            p = a.tables[(int64_t)from * a.width + (k - s_back[from])];
          } else {
            p = a.free_pages[base + k];  // (k < avail, and from all_back on at or behind the old head)
          }
          if ((position & (page - 1)) == 0) a.tables[(int64_t)b * a.width + i] = p;
        }
        if (p >= 0 && p < a.n_pages) slot = (p << a.page_shift) + (position & (page - 1));
      }
    }
    a.slots[t] = slot;
    a.positions[t] = position;
    a.visible[t] = slot >= 0 ? position + 1 : 0;
    a.requests[t] = request;
  }
}

template <int THREADS, int ITEMS>
int step_launch(const StepArgs& a, hipStream_t st) {
  // one row a thread, and no more workgroups than a row each of 64 keeps busy: each makes the sums
  int grid = (a.n_rows + THREADS - 1) / THREADS;
  grid = grid < 1 ? 1 : grid > 64 ? 64 : grid;
  const int bytes = 5 * a.batch * (int)sizeof(int);
  page_step_kernel<THREADS, ITEMS><<<dim3(grid), dim3(THREADS), bytes, st>>>(a);
  MSPR_CHECK_LAUNCH("page_step");
  return MSPR_OK;
}

}  // namespace

extern "C" int mspr_page_step(const int32_t* lens, const int32_t* new_lens, int32_t* tables, int32_t* free_pages,
                              const int32_t* head, int batch, int table_width, int n_pages, int page_size, int n_rows,
                              int32_t* lens_out, int32_t* head_out, int32_t* starts, int32_t* slots, int32_t* positions,
                              int32_t* visible, int32_t* requests, int32_t* counts, void* stream) {
  MSPR_REQUIRE(lens && new_lens && tables && free_pages && head && lens_out && head_out && starts && counts &&
                   (n_rows == 0 || (slots && positions && visible && requests)),
               "page_step: null pointer");
  MSPR_REQUIRE(batch >= 1 && batch <= kMaxRequests, "page_step: 1 to %d requests", kMaxRequests);
  MSPR_REQUIRE(page_size >= 16 && (page_size & (page_size - 1)) == 0, "page_step: page_size must be a power of two from 16 on");
  MSPR_REQUIRE(table_width >= 1 && (int64_t)table_width * page_size <= 0x40000000,
               "page_step: a request's table must hold 1 page or more and at most 2^30 tokens");
  MSPR_REQUIRE((int64_t)batch * table_width <= 0x40000000, "page_step: too many table entries");
  MSPR_REQUIRE(n_pages >= 1 && (int64_t)n_pages * page_size <= 0x7FFFFFFF, "page_step: the pool must hold fewer than 2^31 tokens");
  MSPR_REQUIRE(n_rows >= 0 && n_rows <= 0x3FFFFFFF, "page_step: n_rows out of range");
  MSPR_REQUIRE(lens_out != lens && head_out != head, "page_step: lengths and head are not updated in place");
  const StepArgs a{lens, new_lens, tables, free_pages, head, batch, table_width, n_pages, __builtin_ctz(page_size), n_rows,
                   lens_out, head_out, starts, slots, positions, visible, requests, counts};
  hipStream_t st = (hipStream_t)stream;
  if (batch <= 256) return step_launch<256, 1>(a, st);
  if (batch <= 1024) return step_launch<1024, 1>(a, st);
  return step_launch<1024, 2>(a, st);
}
