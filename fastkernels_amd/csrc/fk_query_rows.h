// Query rows of a batch: which sequence a row belongs to and how many keys it sees.
#pragma once

#include "fk_common.h"

namespace fk {

// Sequence b of query row t and the keys the row sees, vis = ctx - n + i + 1 for the i-th
// of the sequence's n rows (aligned to the end of its tokens; at most ctx).  cu == nullptr:
// one row per sequence.  False for a row behind the last sequence.  Sequences without rows
// are skipped by taking the last b with cu[b] <= t.  Whole waves call it, with one t each.
__device__ __forceinline__ bool query_row(const int32_t* __restrict__ cu,
                                          const int32_t* __restrict__ ctx, int batch, int t,
                                          int& b, int& vis) {
  if (cu == nullptr) {
    b = t;
    vis = t < batch ? ctx[t] : 0;
    return t < batch;
  }
  if (batch <= 0 || t < cu[0] || t >= cu[batch]) return false;
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
  b = lo;
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

}  // namespace fk
