// kv_view.h -- what the paged-cache kernels (kv_ops.hip, kv_attend.h) share: the
// cache, its new rows, and how a row finds its sequence.
#pragma once

#include "device_common.h"

namespace mit2hip {

typedef __bf16 bf16_t;

// What the kernels take of a cache and of its new rows.
struct CacheView {
  char* k;
  char* v;
  const int32_t* table;
  int pages, page_shift, kv_heads, table_stride;

  // Page that holds a sequence's cached row j (0 <= j < capacity()), or -1.
  __host__ __device__ int page_of(int seq, int j) const {
    const int p = table[(size_t)seq * table_stride + (j >> page_shift)];
    return (unsigned)p < (unsigned)pages ? p : -1;
  }
  __host__ __device__ int capacity() const { return table_stride << page_shift; }
  // Element index of head 0's row j in a page.
  __host__ __device__ int64_t row_in(int page, int j, int D) const {
    return ((((int64_t)page * kv_heads) << page_shift) + (j & ((1 << page_shift) - 1))) * D;
  }
  __host__ __device__ int64_t head_stride(int D) const { return (int64_t)D << page_shift; }
};
struct RowView {
  const int32_t* start;
  const int32_t* length;
  int seqs, rows;
};

// The sequence that new row `row` belongs to, or -1 (a wave's lanes look at 64
// bounds at a time; all return the same).
__device__ __forceinline__ int seq_of_row(const RowView& r, int row) {
  const int lane = threadIdx.x & 63;
  int n = 0;
  for (int base = 0; base < r.seqs; base += 64) {
    const bool before = base + lane < r.seqs && r.start[base + lane + 1] <= row;
    const int c = __popcll(__ballot(before));
    n += c;
    if (c < 64) break;
  }
  return n < r.seqs && row >= r.start[n] ? n : -1;
}

}  // namespace mit2hip
