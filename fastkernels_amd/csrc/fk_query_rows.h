// Query rows of a batch: which sequence a row belongs to and how many keys it sees.
#pragma once

#include "fk_common.h"

namespace fk {

// Sequence of row t (cu[b] <= t < cu[b + 1]), or -1 for a row of none.  Sequences without rows are
// skipped by taking the last b with cu[b] <= t.  Whole waves call it, with one t each.
__device__ __forceinline__ int sequence_of(const int32_t* __restrict__ cu, int batch, int t) {
  if (batch <= 0 || t < cu[0] || t >= cu[batch]) return -1;
  // The lanes look at 64 places at a time: one load's latency for up to 64 sequences, where
  // halving takes six.
  const int lane = threadIdx.x & 63;
  int lo = 0, len = batch;
  while (len > 1) {
    const int step = (len + 63) >> 6;
    const bool before = lane * step < len && cu[lo + lane * step] <= t;
    const int last = max(__builtin_popcountll(__ballot(before)) - 1, 0) * step;
    lo += last;
    len = min(step, len - last);
  }
  return lo;
}

// Rows of a work-group of such a copy: two work-groups a CU at least, if there are the rows, and at
// most `most` rows each.
inline int dense_rows_of_wg(int64_t rows, int most) {
  const int64_t per = rows / (2 * num_cus());
  return static_cast<int>(per < 1 ? 1 : per < most ? per : most);
}

// Slots (page * block size + place) of the tokens that rows t0 .. t0 + per - 1 (at most kRows) of a
// dense copy of the sequences stand for, into LDS: -1 at a masked page, -2 for a row of no sequence.  cu may
// not ascend; what is read stays inside the table.
template <int kRows>
__device__ __forceinline__ void dense_slots(const int32_t* __restrict__ cu, int batch, int64_t t0,
                                            int per, int64_t rows, const int32_t* __restrict__ bt,
                                            int64_t bt_row_stride, int bt_width,
                                            int block_size_log2, int64_t num_blocks,
                                            int64_t (&slot)[kRows]) {
  if (threadIdx.x < per) {
    const int64_t t = t0 + threadIdx.x;
    int64_t at = -2;
    if (t < rows && t >= cu[0] && t < cu[batch]) {
      int lo = 0, hi = batch;  // the last sequence that begins at t or before
      while (hi - lo > 1) {
        const int mid = lo + ((hi - lo) >> 1);
        if (cu[mid] <= t) lo = mid; else hi = mid;
      }
      const int64_t pos = t - cu[lo], j = pos >> block_size_log2;
      const int page = j < bt_width ? bt[lo * bt_row_stride + j] : -1;
      at = page >= 0 && page < num_blocks
               ? (static_cast<int64_t>(page) << block_size_log2) +
                     (pos & ((int64_t{1} << block_size_log2) - 1))
               : -1;
    }
    slot[threadIdx.x] = at;
  }
  __syncthreads();
}

// Sequence b of query row t and the keys the row sees, vis = ctx - n + i + 1 for the i-th
// of the sequence's n rows (aligned to the end of its tokens; at most ctx).  cu == nullptr:
// one row per sequence.  False for a row behind the last sequence.  Whole waves call it, with one
// t each.
__device__ __forceinline__ bool query_row(const int32_t* __restrict__ cu,
                                          const int32_t* __restrict__ ctx, int batch, int t,
                                          int& b, int& vis) {
  if (cu == nullptr) {
    b = t;
    vis = t < batch ? ctx[t] : 0;
    return t < batch;
  }
  b = sequence_of(cu, batch, t);
  if (b < 0) return false;
  const int c = ctx[b];
  // (cu[b + 1] > t here, so at least one of the sequence's rows is not before this one.)
  vis = c - (cu[b + 1] - 1 - t);
  vis = vis < c ? vis : c;
  return true;
}

// Pages that hold the first `vis` keys (0 for none).
__device__ __forceinline__ int pages_of(int vis, int block_size_log2) {
  return vis > 0 ? ((vis - 1) >> block_size_log2) + 1 : 0;
}

// A store past the caches, for dense copies larger than they are: the lines that a copy is read
// from stay.
__device__ __forceinline__ void store_past(uint16_t* p, const uint4& v) {
  typedef uint32_t words __attribute__((ext_vector_type(4)));
  __builtin_nontemporal_store(words{v.x, v.y, v.z, v.w}, reinterpret_cast<words*>(p));
}

}  // namespace fk
