// Lines of work: items laid end to end, counted in steps, and cut into equal ranges, one per
// work-group, so that lengths need not be known on the host and none waits for the longest.
#pragma once

#include "fk_common.h"

namespace fk {

__device__ __forceinline__ int64_t lane64(int64_t v, int src) {
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(v), src);
  const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(v >> 32), src);
  return static_cast<int64_t>((static_cast<uint64_t>(hi) << 32) | lo);
}
// Inclusive sums over the lanes of a wave: within rows of 16, then across them.
template <int kCtrl, int kRows>
__device__ __forceinline__ int64_t plus_moved(int64_t v) {
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(v), kCtrl, kRows, 0xf, false);
  const uint32_t hi =
      __builtin_amdgcn_update_dpp(0, static_cast<int>(v >> 32), kCtrl, kRows, 0xf, false);
  return v + static_cast<int64_t>((static_cast<uint64_t>(hi) << 32) | lo);
}
__device__ __forceinline__ int64_t scan64(int64_t v) {
  v = plus_moved<0x111, 0xf>(v);     // from the lane 1 before, 2, 4, 8
  v = plus_moved<0x112, 0xf>(v);
  v = plus_moved<0x114, 0xf>(v);
  v = plus_moved<0x118, 0xf>(v);
  v = plus_moved<0x142, 0xa>(v);     // from lane 15 of the row before, into rows 1 and 3
  return plus_moved<0x143, 0xc>(v);  // from lane 31, into rows 2 and 3
}
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
// A line of `total` tiles is cut into ranges of the least multiple of `quantum` (a power of two)
// that makes them at most n.
__device__ __forceinline__ int64_t range_of(int64_t total, int n, int quantum) {
  int64_t range = static_cast<int64_t>(static_cast<double>(total) / n);
  range += range * n < total;  // (the quotient is off by less than one)
  range = (range + quantum - 1) & -static_cast<int64_t>(quantum);
  return max(range, static_cast<int64_t>(quantum));
}
// a / b (0 <= a, 0 < b) by way of a float estimate, off by one at most for quotients below 2^21.
__device__ __forceinline__ int quotient(int64_t a, int64_t b) {
  int64_t q = static_cast<int64_t>(static_cast<float>(a) *
                                   __builtin_amdgcn_rcpf(static_cast<float>(b)));
  while (q * b > a) --q;
  while ((q + 1) * b <= a) ++q;
  return static_cast<int>(q);
}
// The share of a line that work-group `wg` of n takes, when it has `shares` of them (n or more:
// none).  They are dealt out to the 8 XCDs in runs (work-groups go to XCDs in turn), so that
// neighbouring ranges, which read the same keys for the column blocks of a group, share an L2;
// `last`: the work-groups are counted from the end.
__device__ __forceinline__ int64_t share_of(int wg, int n, int64_t shares, bool last) {
  if (n % 8) return last ? n - 1 - wg : wg;
  const int per = static_cast<int>(shares + 7) / 8;
  const int i = last ? n / 8 - 1 - (wg >> 3) : wg >> 3;
  return i < per ? (wg & 7) * per + i : n;
}

// Query rows of sequence b (cu == nullptr: one each), inside [0, rows) whatever cu says, and at
// most `most`; and the keys they see: row i of n the last window_left + 1 (all: -1) before
// ctx - n + i + 1, whether the rows processed are all n or not.
struct SeqRows {
  int row0, rows, all, ctx;
  int64_t start;  // its first step on the line (filled where that is walked)
};
__device__ __forceinline__ SeqRows seq_rows(const int32_t* __restrict__ cu,
                                            const int32_t* __restrict__ ctx, int b, int rows,
                                            int most) {
  SeqRows s;
  s.start = 0;
  s.ctx = max(ctx[b], 0);
  if (cu == nullptr) {
    s.row0 = b;
    s.rows = s.all = b < rows ? 1 : 0;
    return s;
  }
  const int64_t lo = cu[b], hi = cu[b + 1];
  s.all = static_cast<int>(max(min(hi - lo, int64_t{0x7fffffff}), int64_t{0}));
  s.row0 = static_cast<int>(max(lo, int64_t{0}));
  s.rows = lo < 0 ? 0 : static_cast<int>(max(min(min(lo + s.all, static_cast<int64_t>(rows)) - lo,
                                                 static_cast<int64_t>(most)), int64_t{0}));
  return s;
}
// Keys that row i of such a sequence sees: [lo, hi).
__device__ __forceinline__ void row_keys(const SeqRows& s, int i, int window_left, int& lo,
                                         int& hi) {
  hi = static_cast<int>(max(min(static_cast<int64_t>(s.ctx) - s.all + i + 1,
                                static_cast<int64_t>(s.ctx)), int64_t{0}));
  lo = window_left >= 0 ? max(0, hi - 1 - window_left) : 0;
}

// Its items on a line: `items` of `steps` steps each, laid end to end, over the keys [from, to)
// that any of its rows sees.  Each has `pad` steps before its own that stand for what a part of it
// costs besides them, so that a range of many short items has fewer steps.
struct LineItems {
  int from, to;
  int steps, items;
};
// Where the merge finds a sequence's items on the line.
struct LineRecord {
  int64_t start, range;
  int steps, pad_;
};
// Partial states of the items that ranges cut: a range has one slot for an item that begins
// before it and one for an item that begins in it and goes on behind it.
__device__ __forceinline__ int64_t line_slot(int64_t wg, bool begins) {
  return 2 * wg + (begins ? 1 : 0);
}

// What walk_line holds in LDS: kSeqs sequences at a time.
template <int kThreads, int kSeqs = kThreads>
struct LineLds {
  SeqRows seq[kSeqs];
  int64_t sum[kThreads / 64];
  uint64_t hits[kSeqs / 64];
};

// Walks the share of work-group `wg` of `wgs` on the line of `batch` sequences, seq_at(b) their
// rows and items_of(rows) their items: body(b, rows, items, item, first step, end step, slot, free)
// for each item's part in it, uniform over the work-group; slot: -1 where the part is the whole
// item, otherwise where its partial state goes; free: a slot that is not in use yet where the part
// is a whole item.  Work-group wgs writes every sequence's record instead.
// Every thread of the work-group calls it; items have at least one step.
template <int kThreads, int kSeqs, class SeqAt, class ItemsOf, class Body>
__device__ __forceinline__ void walk_line(LineLds<kThreads, kSeqs>& lds, int batch, int wgs, int wg,
                                          int quantum, int pad,
                                          LineRecord* __restrict__ records,
                                          SeqAt seq_at, ItemsOf items_of, Body body) {
  constexpr int kWaves = kThreads / 64;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  auto scan_all = [&](int64_t v, int64_t& total) {
    const int64_t x = scan64(v);
    if (lane == 63) lds.sum[wave] = x;
    __syncthreads();
    int64_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      before += w < wave ? lds.sum[w] : 0;
      total += lds.sum[w];
    }
    __syncthreads();
    return before + x;
  };
  auto at = [&](int b) {
    SeqRows x{};
    if (tid < kSeqs && b < batch) x = seq_at(b);
    return x;
  };
  auto length = [&](const SeqRows& x) {
    if (x.rows == 0) return int64_t{0};
    const LineItems it = items_of(x);
    return static_cast<int64_t>(it.steps + pad) * it.items;
  };
  int64_t sum = 0, total;
  for (int b = tid; b < batch; b += kSeqs) sum += length(at(b));
  scan_all(sum, total);
  if (total == 0) return;
  const int64_t S = range_of(total, wgs, quantum);
  const bool writes = wg == wgs;
  const int64_t w = writes ? 0 : share_of(wg, wgs, quotient(total + S - 1, S), false);
  const int64_t t_lo = writes ? 0 : w * S;
  const int64_t t_hi = writes ? total : min(total, t_lo + S);
  int64_t line = 0;
  for (int b0 = 0; t_lo < total && b0 < batch && line < t_hi; b0 += kSeqs) {
    SeqRows x = at(b0 + tid);
    const int64_t mine = length(x);
    const int64_t end = line + scan_all(mine, sum);
    line += sum;
    x.start = end - mine;
    if (writes) {
      if (mine > 0) records[b0 + tid] = LineRecord{x.start, S, items_of(x).steps, 0};
      continue;
    }
    const bool in = mine > 0 && end > t_lo && x.start < t_hi;
    if (in) lds.seq[tid] = x;
    const uint64_t hits = __ballot(in);
    if (lane == 0 && wave < kSeqs / 64) lds.hits[wave] = hits;
    __syncthreads();
#pragma unroll 1
    for (int k = 0; k < kSeqs / 64; ++k) {
      uint64_t hit = lane64(lds.hits[k], 0);
      while (hit) {
        const int src = 64 * k + __builtin_ctzll(hit);
        hit &= hit - 1;
        SeqRows y = lds.seq[src];
        y.row0 = uniform(y.row0);
        y.rows = uniform(y.rows);
        y.all = uniform(y.all);
        y.ctx = uniform(y.ctx);
        y.start = lane64(y.start, 0);
        const LineItems z = items_of(y);
        const int length = z.steps + pad;
        for (int it = t_lo > y.start ? quotient(t_lo - y.start, length) : 0;
             it < z.items && y.start + static_cast<int64_t>(it) * length < t_hi; ++it) {
          const int64_t s0 = y.start + static_cast<int64_t>(it) * length + pad;
          const int lo = static_cast<int>(max(t_lo - s0, int64_t{0}));
          const int hi = static_cast<int>(min(t_hi - s0, static_cast<int64_t>(z.steps)));
          if (hi <= 0) continue;
          const bool whole = lo == 0 && hi == z.steps;
          body(b0 + src, y, z, it, lo, hi, whole ? int64_t{-1} : line_slot(w, lo == 0),
               line_slot(w, true));
        }
      }
    }
    __syncthreads();
  }
}

// The pieces of item `it` of a sequence: their number (1: the item was whole in its range), and
// the slot of piece k.
struct LinePieces {
  int64_t first;
  int n;
  __device__ __forceinline__ LinePieces(const LineRecord& r, int it, int pad) {
    const int64_t s0 = r.start + static_cast<int64_t>(it) * (r.steps + pad) + pad;
    first = quotient(s0, r.range);
    n = quotient(s0 + r.steps - 1, r.range) - static_cast<int>(first) + 1;
  }
  __device__ __forceinline__ int64_t slot(int k) const { return line_slot(first + k, k == 0); }
};

}  // namespace fk
