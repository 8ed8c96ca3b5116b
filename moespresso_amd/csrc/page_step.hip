// Tables of one step of a paged cache, from the requests' lengths.
//
// The pages of a pool that no request holds lie on a stack (`free_pages` from `head` on). A step gives every request the
// pages that its new rows begin, takes those of ended requests back first, and names a slot (page * page_size + row in the
// page) for every new row. Four running sums over the requests decide everything: rows asked for, pages needed, pages given
// back; each page that moves and each row then finds its request by bisection of a sum.
//
// Bound by latency: a step of 16 requests reads 128 bytes and writes 500, in 2.9 us; one of 1000, of which some end, takes 6.7.
// One launch; every workgroup makes the sums anew (2048 requests are eight a thread) rather than wait for another's, and writes
// its share of the rows. What one workgroup writes no other reads: pages given back go below `head` and pages taken from there
// are read where they come from, the table of the ended request; new table entries lie behind those that rows of the last
// started page read.
#include "common.h"

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / MSPR_WAVE;
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

// a + b of values from 0 on, at most 2^32 - 1: asked-for rows may add up to more
__device__ __forceinline__ uint32_t sat_add(uint32_t a, uint32_t b) { return __builtin_elementwise_add_sat(a, b); }

template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t scan_step(uint32_t v) {
  return sat_add(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false));
}

// Sums over this lane and those before it, by data-parallel moves.
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
  v = scan_step<0x111, 0xF>(v);  // row_shr 1, 2, 4, 8
  v = scan_step<0x112, 0xF>(v);
  v = scan_step<0x114, 0xF>(v);
  v = scan_step<0x118, 0xF>(v);
  v = scan_step<0x142, 0xA>(v);  // row_bcast 15, 31
  return scan_step<0x143, 0xC>(v);
}

// Sums of N values over the threads before this one (in place), and over all of them in `total`, at most 2^31 - 1.
template <int N>
__device__ __forceinline__ void block_scan(uint32_t* v, uint32_t (*wave_sums)[N], int* total) {
  const int wave = threadIdx.x >> 6;
  uint32_t s[N];
#pragma unroll
  for (int k = 0; k < N; k++) {
    s[k] = wave_scan(v[k]);
    if ((threadIdx.x & 63) == 63) wave_sums[wave][k] = s[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < N; k++) {
    uint32_t all = 0, before = 0;
#pragma unroll
    for (int w = 0; w < kWaves; w++) {
      if (w == wave) before = all;
      all = sat_add(all, wave_sums[w][k]);
    }
    v[k] = sat_add(before, s[k] - v[k]);
    total[k] = all > 0x7FFFFFFFu ? 0x7FFFFFFF : (int)all;
  }
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

// grid: workgroups that share rows and returned pages; LDS: five arrays of `batch` integers. ITEMS requests a thread.
template <int ITEMS>
__global__ __launch_bounds__(kThreads) void page_step_kernel(StepArgs a) {
  extern __shared__ int lds[];
  __shared__ uint32_t wave_sums[3][kWaves][2];
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
#pragma unroll
  for (int i = 0; i < ITEMS; i++) {
    const int b = tid * ITEMS + i;
    old_[i] = b < B ? a.lens[b] : 0;
    add_[i] = b < B ? a.add[b] : 0;
  }
  int head = *a.head;
  head = head < 0 ? 0 : head > a.n_pages ? a.n_pages : head;
  uint32_t rows[1] = {0};
#pragma unroll
  for (int i = 0; i < ITEMS; i++) {
    old_[i] = old_[i] < 0 ? 0 : old_[i] > cap ? cap : old_[i];
    rows[0] = sat_add(rows[0], add_[i] > 0 ? add_[i] : 0);
  }
  rows[0] = min(rows[0], 0x7FFFFFFFu);  // (so that a sum that is cut off stays far above n_rows without this thread's)
  int all_rows;
  block_scan<1>(rows, reinterpret_cast<uint32_t(*)[1]>(wave_sums[0]), &all_rows);
  // rows behind n_rows are not part of the step: what a request may add ends there, and at its table's end
  int start_[ITEMS], goal_[ITEMS];
  uint32_t pages[2] = {0, 0};  // needed, given back
#pragma unroll
  for (int i = 0; i < ITEMS; i++) {
    const int asked = add_[i] > 0 ? add_[i] : 0;
    start_[i] = rows[0] < (uint32_t)a.n_rows ? (int)rows[0] : a.n_rows;
    goal_[i] = old_[i] + min(min(asked, a.n_rows - start_[i]), cap - old_[i]);
    rows[0] = sat_add(rows[0], asked);
    const int held = (old_[i] + page - 1) >> a.page_shift;
    if (add_[i] < 0) pages[1] += held;
    else pages[0] += ((goal_[i] + page - 1) >> a.page_shift) - held;
  }
  int all_pages[2];
  block_scan<2>(pages, wave_sums[1], all_pages);
  const int all_need = all_pages[0], all_back = all_pages[1];
  int first = (int)pages[0], given = (int)pages[1];
  const int base = head - all_back;  // the stack's new top, before pages are taken (below 0 only if pages were lent twice)
  const int avail = a.n_pages - base;
  uint32_t placed[1] = {0};
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
        if (!ended) placed[0] += len - old_[i];
      }
    }
    first += want;
    given += ended ? held : 0;
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    int all_placed;
    block_scan<1>(placed, reinterpret_cast<uint32_t(*)[1]>(wave_sums[2]), &all_placed);
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

  const int stride = gridDim.x * kThreads;
  for (int k = blockIdx.x * kThreads + tid; k < all_back; k += stride) {
    const int b = last_at_most(s_back, B, k);
    const int at = base + k;
    if (at >= 0) a.free_pages[at] = a.tables[(int64_t)b * a.width + (k - s_back[b])];
  }
  for (int t = blockIdx.x * kThreads + tid; t < a.n_rows; t += stride) {
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

template <int ITEMS>
int step_launch(const StepArgs& a, hipStream_t st) {
  // A row a thread; pages given back, of which the host knows no number, get a workgroup per sixteen requests. Each workgroup
  // makes the sums, so there are no more of them than half the compute units.
  const int for_rows = (a.n_rows + kThreads - 1) / kThreads, for_pages = (a.batch + 15) / 16;
  const int most = for_rows > for_pages ? for_rows : for_pages;
  const int grid = most < 1 ? 1 : most > 128 ? 128 : most;
  const int bytes = 5 * a.batch * (int)sizeof(int);
  page_step_kernel<ITEMS><<<dim3(grid), dim3(kThreads), bytes, st>>>(a);
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
  MSPR_REQUIRE(n_pages >= 1 && (int64_t)n_pages * page_size <= 0x7FFFFFFF,
               "page_step: the pool must hold fewer than 2^31 tokens");
  MSPR_REQUIRE(n_rows >= 0 && n_rows <= 0x3FFFFFFF, "page_step: n_rows out of range");
  MSPR_REQUIRE(lens_out != lens && head_out != head, "page_step: lengths and head are not updated in place");
  const StepArgs a{lens, new_lens, tables, free_pages, head, batch, table_width, n_pages, __builtin_ctz(page_size), n_rows,
                   lens_out, head_out, starts, slots, positions, visible, requests, counts};
  hipStream_t st = (hipStream_t)stream;
  if (batch <= 256) return step_launch<1>(a, st);
  if (batch <= 512) return step_launch<2>(a, st);
  if (batch <= 1024) return step_launch<4>(a, st);
  return step_launch<8>(a, st);
}
