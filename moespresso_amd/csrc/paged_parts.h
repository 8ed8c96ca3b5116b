// Decode attention over pages (paged_decode.hip) whose results are joined with attention over other keys of the same queries: what
// is left of every row instead of its output.
#pragma once
#include "paged_rows.h"

// The call's operands (checked as those of mspr_sdpa_decode_paged are), and where rows that are not cut go: sums relative to their
// reference maximum [batch * n_kv * rep][256], maximum (powers of two) and sum of weights [..][2].
struct PagedPartsCall {
  const void *q, *k, *v, *k_scales, *k_biases, *v_scales, *v_biases;  // scales and biases: null of 16-bit rows
  int q_dtype, sb_dtype;
  const int32_t *tables, *lens, *requests;
  int batch, n_kv, rep, n_pages, page_shift, n_tables, width;
  float scale_log2;
  float *own, *own_ml;
  void* workspace;  // of mspr_sdpa_decode_paged_workspace_bytes
  size_t workspace_bytes;
};

// Rows that are cut: row by row {the row or -1, its first share, its last}, null where none is; their parts' sums
// [2 shares][rep][256] and statistics [2 shares][16][2].
struct PagedParts {
  const int32_t* cut;
  const float *o, *ml;
  int shares;
};

int mspr_paged_decode_parts(const char* what, const PagedPartsCall& call, PagedParts* parts, hipStream_t st);

namespace {

// Where part i of a row lies whose first part is share `first`'s: that began the row, the others go on with it.
__device__ __forceinline__ int64_t part_of(int first, int i) { return 2 * (int64_t)(first + i) + (i == 0 ? 1 : 0); }

// An entry of `cut`: a row and how many parts it has, none where no row was cut. (Bounded by the call's rows and shares,
// whatever is there.)
struct Cut {
  int row, first, count;
  __device__ __forceinline__ void load(const int32_t* cut, int entry, int rows, int shares) {
    row = cut[3 * entry];
    first = cut[3 * entry + 1];
    const int last = min(cut[3 * entry + 2], shares - 1);
    count = ((row < 0) | (row >= rows) | (first < 0) | (first > last)) ? 0 : last - first + 1;  // (one wait for the three)
  }
};

}  // namespace
