// Decode attention of a batch whose sequences come in groups that share a prefix.
//
// Rows cu_groups[g] .. cu_groups[g + 1] - 1 hold the same keys at positions below
// prefix_lens[g], which are read through the block table of the group's first row; every
// other key is read through the row's own table.  The result is that of paged decode: row b
// attends to its keys [lo, ctx_lens[b]), lo = 0 or ctx - 1 - window_left under a sliding
// window.  Rows outside every group share nothing.
//
// Work.  A group's rows times the query heads of one kv head are the columns of one matrix
// product with the prefix's keys: blocks of kCols columns stream the prefix's 16-token tiles
// once each (where paged decode would stream them once per row), and what a row has of its own
// is streamed like decode's, 16 columns at most.  Both kinds are lines of tiles,
//   prefix line: (group, kv head, block of columns) x tiles of the prefix
//   own line:    (row, kv head, block of 16 query heads) x tiles from the prefix's end on
// cut into equal ranges, one per work-group of the first and one per wave of the second, so that
// lengths need not be known on the host and none waits for the longest.  The four waves of a
// work-group share a prefix range's tiles (fk_page_attn.h).  Each item and range leave one
// partial state; a second launch merges each row's partials of both kinds.
//
// What bounds it.  Own tiles are read once: memory.  A prefix tile is read once per 32 columns
// (at head size 128), from L2 where the column blocks' ranges are in phase (below), and costs the
// vector units as much as the matrix units.  One half of the CUs takes its prefix ranges first
// and the other half last, so that the chip does both at a time (both on each CU: 96 us where
// this took 87).
// Two waves a SIMD (O of 32 columns, the queries, and two tiles of K and V fill their registers)
// leave latencies that show.  Measured: 64 rows of 32 / 8 heads over a prefix of 8192 bf16
// tokens with 100 .. 2000 of their own 85.5 us and 5.6 for the merge (311 MB, 9.7 GFLOP); 128
// rows of 64 / 8 heads over three prefixes of 11000 .. 16400 fp8 tokens 137 us and 7.5 (250 MB,
// 60 GFLOP; little less with every page in L2); 8 rows over 1488 tokens 15.3 us and 4.0.  The
// set-up of a work-group has more live than its registers hold (132 .. 160 scalars go to vector
// registers, up to 48 vectors to scratch), which the smallest calls show; the tile loops touch
// no scratch.
// Variants that were slower there: 16 or 64 columns to a wave, 128 columns to a work-group
// with K and V staged in LDS (117 .. 136 and 185 .. 210 us), the four waves on four column blocks
// of the same tiles (98 and 152, 10 for the merge), two steps of loads ahead, items rounded up to
// whole ranges (101 and 160).
#include <limits.h>

#include "fk_page_attn.h"

namespace fk {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * 64;
// A prefix range is a multiple of this: in pages of 16 tokens two tiles per wave; in pages of 64
// and more two units of four tiles, which two of the waves take.
constexpr int kPreTiles = 8;
constexpr int kOwnTiles = 2;      // a wave's own range is a multiple of this: a step
constexpr int kMaxGroups = 2048;  // (their bounds are held in LDS)

// Column blocks of a prefix item.  (O takes 4 D / 16 registers per block.)
template <int D>
constexpr int col_blocks_of() { return D == 64 ? 4 : D == 128 ? 2 : 1; }
constexpr int cols_of(int d) { return 16 * (d == 64 ? 4 : d == 128 ? 2 : 1); }

// What the merge has to know of a row.
struct RowRecord {
  int64_t own_start;  // the row's first tile on the own line (its first head's)
  int64_t pre_start;  // its group's first tile on the prefix line
  int64_t own_range, pre_range;  // tiles of a range of each line
  int64_t pre_step;              // places of a prefix item
  int own_tiles;      // tiles per head (0: nothing of its own)
  int pre_tiles;      // tiles of the prefix (0: no shared prefix)
  int pre_item;       // its group's first prefix item
  int col_items;      // column blocks of its group, per kv head
  int index;          // row of its group
  int short_keys;     // keys of a row shorter than its group's prefix, otherwise -1
};

struct PrefixParams {
  PageAttnParams A;
  int num_groups;
  int max_prefix;          // tokens of a prefix that are shared at most
  int window_left;
  int unit_tiles_log2;
  int wgs;                 // work-groups that share the lines
  int vheads;              // kv heads x blocks of 16 query heads
  int own_cols;            // query columns of an own item: min(16, gqa)
  int merge_cols;          // of which a work-group of the merge takes so many
  float* pre_o;            // [pieces][kCols][D], then (maximum, sum) per column
  float* pre_ml;
  float* own_o;            // [pieces][own_cols][D]
  float* own_ml;
  int64_t pre_pieces;      // room for pieces of the prefix line
  RowRecord* rows;         // [batch]
};

// A group: its rows, and the prefix that they share in this launch: none where there is one
// row, or under a sliding window (each row then streams its own window).
struct Group {
  int first, rows, prefix;
};
// What a row streams of its own: positions [from, ctx), through its own table from position
// `border` on and through its group's first row's before.
struct Own {
  int from, ctx, border, first_row, tiles, pad_;
  int64_t start;  // on the own line (filled where the line is walked)
};

__device__ __forceinline__ int tiles_in(int tokens) {
  return tokens > 0 ? (tokens - 1) / kTile + 1 : 0;
}
// The places of a prefix item on its line: its tiles, rounded up so that the ranges of a short
// line do not span two items.
__device__ __forceinline__ int64_t places_of(int prefix) {
  return (tiles_in(prefix) + kPreTiles - 1) & -kPreTiles;
}
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
// v of the lane `off` places further on in the row of 16, round.
template <int kOff>
__device__ __forceinline__ uint32_t rotated(uint32_t v) {
  return __builtin_amdgcn_update_dpp(0, v, 0x120 + kOff, 0xf, 0xf, false);
}
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
  v = max(v, rotated<8>(v));
  v = max(v, rotated<4>(v));
  v = max(v, rotated<2>(v));
  return max(v, rotated<1>(v));
}
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
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// LDS: the merge's states (also the last work-group's tables), a chunk of rows, the groups.
template <int D>
constexpr int lds_rows_at() { return 4 * merge_lds_floats<kWaves, D>(cols_of(D)); }
template <int D>
constexpr int lds_groups_at() { return lds_rows_at<D>() + kThreads * static_cast<int>(sizeof(Own)); }
static_assert(kWaves * 2 * KChunks<false, 64>::kBytes <= lds_rows_at<64>() &&
                  kWaves * 2 * KChunks<false, 128>::kBytes <= lds_rows_at<128>() &&
                  kWaves * 2 * KChunks<false, 256>::kBytes <= lds_rows_at<256>(),
              "the waves' K rows fit");
static_assert(kMaxGroups * 12 <= lds_groups_at<64>(), "the last work-group's tables fit");

template <int D, bool kFp8>
__global__ __launch_bounds__(kThreads)
__attribute__((amdgpu_waves_per_eu((D == 256 ? 1 : 2)))) void shared_prefix_kernel(
    PrefixParams P, const int32_t* __restrict__ bt, const int32_t* __restrict__ ctx_lens,
    const int32_t* __restrict__ cu_groups, const int32_t* __restrict__ prefix_lens) {
  constexpr int kCB = col_blocks_of<D>();
  constexpr int kCols = 16 * kCB;
  extern __shared__ __align__(16) uint8_t lds_all[];
  __shared__ int64_t wave_sum[kWaves];
  __shared__ uint64_t wave_hits[kWaves];
  float* const lds = reinterpret_cast<float*>(lds_all);
  Own* const own_rows = reinterpret_cast<Own*>(lds_all + lds_rows_at<D>());
  int* const group_first = reinterpret_cast<int*>(lds_all + lds_groups_at<D>());
  int* const group_prefix = group_first + P.num_groups + 1;
  const PageAttnParams& A = P.A;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int r = lane & 15, g = lane >> 4;
  const int tok_log2 = 4 + P.unit_tiles_log2;
  // Row and head indexes, and so every address formed from them, stay inside the batch
  // whatever the groups say.  (Without groups there may be no cu_groups to read.)
  for (int i = threadIdx.x; i <= P.num_groups; i += kThreads) {
    group_first[i] = P.num_groups > 0 ? min(max(cu_groups[i], 0), A.batch) : 0;
    if (i < P.num_groups) {
      const int64_t most = static_cast<int64_t>(A.bt_width) << A.block_size_log2;
      group_prefix[i] =
          static_cast<int>(min(static_cast<int64_t>(max(prefix_lens[i], 0)), most));
    }
  }
  __syncthreads();
  auto group_at = [&](int i) {
    Group x{0, 0, 0};
    if (i >= P.num_groups) return x;
    x.first = group_first[i];
    x.rows = group_first[i + 1] - x.first;
    x.prefix = x.rows > 1 && P.window_left < 0 ? min(group_prefix[i], P.max_prefix) : 0;
    return x;
  };
  // Items (kv heads x column blocks) of a group and the tiles of each.
  auto group_items = [&](const Group& x) {
    return x.prefix > 0 ? A.num_kv_heads * ((x.rows * A.gqa + kCols - 1) / kCols) : 0;
  };
  // The group that holds row b (the last one with first <= b), or -1.
  auto group_of = [&](int b) {
    if (P.num_groups <= 0 || b < group_first[0] || b >= group_first[P.num_groups]) return -1;
    int lo = 0, hi = P.num_groups;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (group_first[mid] <= b) lo = mid; else hi = mid;
    }
    return lo;
  };
  auto own_at = [&](int b) {
    Own w{};
    if (b >= A.batch) return w;
    w.ctx = max(ctx_lens[b], 0);
    const int grp = group_of(b);
    w.first_row = b;
    w.from = P.window_left >= 0 ? max(0, w.ctx - 1 - P.window_left) : 0;
    if (grp >= 0) {
      const Group x = group_at(grp);
      w.border = min(group_prefix[grp], w.ctx);
      w.first_row = x.first;
      if (x.prefix > 0) w.from = min(x.prefix, w.ctx);
    }
    // counted from the tile of `from`
    w.tiles = w.ctx > w.from ? (w.ctx - 1) / kTile - w.from / kTile + 1 : 0;
    return w;
  };
  // Inclusive sums over the work-group's threads; total: over all of them.
  auto scan_all = [&](int64_t v, int64_t& total) {
    const int64_t x = scan64(v);
    if (lane == 63) wave_sum[wave] = x;
    __syncthreads();
    int64_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      before += w < wave ? wave_sum[w] : 0;
      total += wave_sum[w];
    }
    __syncthreads();
    return before + x;
  };
  auto prefix_length = [&] {
    int64_t sum = 0;
    for (int i = lane; i < P.num_groups; i += 64) {
      const Group x = group_at(i);
      sum += group_items(x) * places_of(x.prefix);
    }
    return lane64(scan64(sum), 63);
  };
  // Streams positions [from, to) of one item through the table `table`: unit `first` and every
  // step-th after it.
  auto stream = [&](auto& st, const int32_t* table, int from, int to, int first, int step,
                    auto limits, int kvh, float s2) {
    const int u0 = from >> tok_log2;
    auto unit_at = [&](int u, int& page, int& tok) {
      tok = (u0 + u) << tok_log2;
      const int j = tok >> A.block_size_log2;
      page = j < A.bt_width ? table[j] : -1;
    };
    stream_units(A, st, unit_at, from < to ? ((to - 1) >> tok_log2) + 1 - u0 : 0, first, step,
                 P.unit_tiles_log2, from, to, limits, kvh, s2,
                 lds_all + wave * 2 * KChunks<kFp8, D>::kBytes, lane);
  };
  auto factor = [&](int kvh) {
    return kFp8 && A.k_scale ? A.scale_log2 * A.k_scale[kvh] : A.scale_log2;
  };

  const int wg = blockIdx.x;
  auto run_prefix = [&] {
    const int64_t total = prefix_length();
    const int64_t S = range_of(total, P.wgs, kPreTiles);
    int64_t line = 0;  // tiles and items of the groups before the chunk
    int64_t item0 = 0;
    const int64_t w = share_of(wg, P.wgs, quotient(total + S - 1, S), false);
    const int64_t t_lo = w * S, t_hi = min(total, t_lo + S);
    for (int g0 = 0; t_lo < total && g0 < P.num_groups && line < t_hi; g0 += 64) {
      const Group x = group_at(g0 + lane);
      const int items = group_items(x);
      const int64_t mine = items * places_of(x.prefix);
      const int64_t end = line + scan64(mine);
      const int64_t item_end = item0 + scan64(items);
      uint64_t hit = __ballot(mine > 0 && end > t_lo && end - mine < t_hi);
      while (hit) {
        const int src = __builtin_ctzll(hit);
        hit &= hit - 1;
        const int row0 = __builtin_amdgcn_readlane(x.first, src);
        const int n_cols = __builtin_amdgcn_readlane(x.rows, src) * A.gqa;
        const int prefix = __builtin_amdgcn_readlane(x.prefix, src);
        const int n_items = __builtin_amdgcn_readlane(items, src);
        const int64_t start = lane64(end - mine, src);
        const int64_t first_item = lane64(item_end, src) - n_items;
        const int64_t step = places_of(prefix);
        const int col_items = n_items / A.num_kv_heads;
        for (int it = t_lo > start ? quotient(t_lo - start, step) : 0;
             it < n_items && start + it * step < t_hi; ++it) {
          const int64_t at = start + it * step;
          const int from = static_cast<int>(
              min(static_cast<int64_t>(prefix), (max(t_lo, at) - at) * kTile));
          const int to = static_cast<int>(
              min(static_cast<int64_t>(prefix), (min(t_hi, at + step) - at) * kTile));
          const int kvh = it / col_items;
          const int col0 = (it - kvh * col_items) * kCols;
          const float s2 = factor(kvh);
          ColumnState<kCB, D, kFp8> st;
          st.reset();
          int seen[kCB];  // keys of this lane's column, all of them for a column that is none
#pragma unroll
          for (int cb = 0; cb < kCB; ++cb) {
            const int c = col0 + 16 * cb + r;
            const bool ok = c < n_cols;
            const int b = row0 + (ok ? c / A.gqa : 0);
            const int hq = kvh * A.gqa + (ok ? c % A.gqa : 0);
            seen[cb] = ok ? ctx_lens[b] : -1;
            st.load_q(cb, A.q + b * A.q_row_stride + static_cast<int64_t>(hq) * D, ok,
                      s2 < 0.f ? 0x80008000u : 0u, g);
          }
          // From the first multiple of the range's length on, then what is before it: so that
          // at any time all ranges are as far past such a multiple, and the column blocks of a
          // kv head, whose ranges begin anywhere, read the same tiles while the L2 holds them.
          const int64_t length = S * kTile;
          const int turn = static_cast<int>(min(
              static_cast<int64_t>(to), quotient(from + length - 1, length) * length));
#pragma unroll 1
          for (int part = 0; part < 2; ++part) {
            const int lo = part ? from : turn, hi = part ? turn : to;
            if (lo >= hi) continue;
            auto limits = [&] {
              Limits<kCB> x;
              x.span = 0;
              x.least = hi - lo;
#pragma unroll
              for (int cb = 0; cb < kCB; ++cb) {
                const bool ok = col0 + 16 * cb + r < n_cols;
                x.lim[cb] = ok ? max(min(hi, seen[cb]) - lo, 0) : hi - lo;
                x.span = max(x.span, ok ? x.lim[cb] : 0u);
                x.least = min(x.least, x.lim[cb]);
              }
              x.span = uniform(row_max(x.span));
              x.least = ~uniform(row_max(~x.least));
              return x;
            };
            stream(st, bt + row0 * A.bt_row_stride, lo, hi, wave, kWaves, limits, kvh,
                   __builtin_fabsf(s2));
          }
          const int64_t piece = w + first_item + it;
          if (piece >= P.pre_pieces) continue;  // (groups that overlap: beyond the plan)
          float* po = P.pre_o + piece * kCols * D;
          float* pm = P.pre_ml + piece * kCols * 2;
          merge_waves<kWaves>(st, lds, wave, lane, min(kCols, n_cols - col0),
                              [&](int j, int dim, const float4& o, float M, float L) {
                                *reinterpret_cast<float4*>(po + j * D + dim) = o;
                                if (dim == 0)
                                  *reinterpret_cast<float2*>(pm + 2 * j) = make_float2(M, L);
                              });
          __syncthreads();
        }
      }
      line = lane64(end, 63);
      item0 = lane64(item_end, 63);
    }
  };

  // The own line: a wave's range is one of 4 wgs.
  const Own own0 = own_at(threadIdx.x);
  int64_t own_total;
  {
    int64_t sum = own0.tiles;
    for (int b = kThreads + threadIdx.x; b < A.batch; b += kThreads) sum += own_at(b).tiles;
    scan_all(sum, own_total);
  }
  own_total *= P.vheads;
  const int64_t own_range = range_of(own_total, kWaves * P.wgs, kOwnTiles);

  auto run_own = [&] {
    const int64_t S = own_range;
    const int64_t w0 =
        kWaves * share_of(wg, P.wgs, quotient(own_total + kWaves * S - 1, kWaves * S), true);
    const int64_t all_hi = min(own_total, (w0 + kWaves) * S);  // of the work-group
    const int64_t w = w0 + wave;
    const int64_t t_lo = w * S, t_hi = min(own_total, t_lo + S);
    int64_t line = 0;
    for (int b0 = 0; w0 * S < own_total && b0 < A.batch && line < all_hi; b0 += kThreads) {
      Own o = b0 == 0 ? own0 : own_at(b0 + threadIdx.x);
      const int64_t mine = static_cast<int64_t>(o.tiles) * P.vheads;
      int64_t sum;
      const int64_t end = line + scan_all(mine, sum);
      line += sum;
      o.start = end - mine;
      const bool in = mine > 0 && end > w0 * S && o.start < all_hi;
      if (in) own_rows[threadIdx.x] = o;
      const uint64_t hits = __ballot(in);
      if (lane == 0) wave_hits[wave] = hits;
      __syncthreads();
#pragma unroll 1
      for (int k = 0; k < kWaves; ++k) {
        uint64_t hit = lane64(wave_hits[k], 0);
        while (hit) {
          const int src = 64 * k + __builtin_ctzll(hit);
          hit &= hit - 1;
          const int b = b0 + src;
          Own x = own_rows[src];
          x.from = uniform(x.from);
          x.ctx = uniform(x.ctx);
          x.border = uniform(x.border);
          x.first_row = uniform(x.first_row);
          x.tiles = uniform(x.tiles);
          x.start = lane64(x.start, 0);
          const int tile0 = x.from / kTile;
          for (int v = t_lo > x.start ? quotient(t_lo - x.start, x.tiles) : 0;
               v < P.vheads && x.start + static_cast<int64_t>(v) * x.tiles < t_hi; ++v) {
            const int64_t at = x.start + static_cast<int64_t>(v) * x.tiles;
            const int64_t k_lo = max(t_lo, at) - at, k_hi = min(t_hi, at + x.tiles) - at;
            const int from = max(x.from, kTile * (tile0 + static_cast<int>(k_lo)));
            const int to = static_cast<int>(
                min(static_cast<int64_t>(x.ctx), (tile0 + k_hi) * int64_t{kTile}));
            const int kvh = v / A.col_blocks;
            const int qbase = kvh * A.gqa + 16 * (v - kvh * A.col_blocks);
            const int nc = min(16, (kvh + 1) * A.gqa - qbase);
            const float s2 = factor(kvh);
            ColumnState<1, D, kFp8> st;
            st.reset();
            st.load_q(0, A.q + b * A.q_row_stride + static_cast<int64_t>(qbase + r) * D, r < nc,
                      s2 < 0.f ? 0x80008000u : 0u, g);
            // before the border through the group's table, then through the row's own
            const int mid = min(max(x.border, from), to);
#pragma unroll 1
            for (int own = mid > from ? 0 : 1; own < 2; ++own) {
              const int lo = own ? mid : from, hi = own ? to : mid;
              const uint32_t span = hi - lo;
              stream(st, bt + (own ? b : x.first_row) * A.bt_row_stride, lo, hi, 0, 1,
                     [&] { return Limits<1>{{span}, span, span}; }, kvh, __builtin_fabsf(s2));
            }
            const int64_t piece = w + static_cast<int64_t>(b) * P.vheads + v;
            write_partial(st, P.own_o + piece * P.own_cols * D, P.own_ml + piece * P.own_cols * 2,
                          lane, nc);
          }
        }
      }
      __syncthreads();
    }
  };

  if (wg == P.wgs) {
    // The last work-group writes the merge's records: first each group's place on the prefix
    // line, into LDS, then the rows'.
    int64_t* const pre_start = reinterpret_cast<int64_t*>(lds_all);
    int* const pre_item = reinterpret_cast<int*>(pre_start + P.num_groups);
    const int64_t pre_range = range_of(prefix_length(), P.wgs, kPreTiles);
    if (wave == 0) {
      int64_t line = 0, item0 = 0;
      for (int g0 = 0; g0 < P.num_groups; g0 += 64) {
        const Group x = group_at(g0 + lane);
        const int items = group_items(x);
        const int64_t mine = items * places_of(x.prefix);
        const int64_t end = line + scan64(mine);
        const int64_t item_end = item0 + scan64(items);
        if (g0 + lane < P.num_groups) {
          pre_start[g0 + lane] = end - mine;
          pre_item[g0 + lane] = static_cast<int>(item_end) - items;
        }
        line = lane64(end, 63);
        item0 = lane64(item_end, 63);
      }
    }
    __syncthreads();
    int64_t line = 0;
    for (int b0 = 0; b0 < A.batch; b0 += kThreads) {
      const int b = b0 + threadIdx.x;
      const Own o = own_at(b);
      const int64_t mine = static_cast<int64_t>(o.tiles) * P.vheads;
      int64_t sum;
      const int64_t end = line + scan_all(mine, sum);
      line += sum;
      if (b >= A.batch) continue;
      RowRecord rec{};
      rec.own_start = end - mine;
      rec.own_range = own_range;
      rec.own_tiles = o.tiles;
      rec.short_keys = -1;
      rec.pre_range = pre_range;
      const int grp = group_of(b);
      if (grp >= 0) {
        const Group x = group_at(grp);
        rec.pre_start = pre_start[grp];
        rec.pre_tiles = tiles_in(x.prefix);
        rec.pre_step = places_of(x.prefix);
        rec.pre_item = pre_item[grp];
        rec.col_items = group_items(x) / A.num_kv_heads;
        rec.index = b - x.first;
        if (o.ctx < x.prefix) rec.short_keys = o.ctx;
      }
      P.rows[b] = rec;
    }
    return;
  }
  // (Work-groups go to the XCDs in turn and in each to its CUs, of which there is an even number.)
  const bool prefix_first = !((wg >> 3) & 1);
#pragma unroll 1
  for (int phase = 0; phase < 2; ++phase) {
    if ((phase == 0) == prefix_first)
      run_prefix();
    else
      run_own();
  }
}

// A step of 256 keys in attend_plainly: where they are in the caches, and their weights.
struct PlainLds {
  int64_t row[kMergeThreads];
  float weight[kMergeThreads], top[kMergeThreads / 64];
};
// Attention of query head hq of row b over positions [0, keys) read through `table`, by a merge's
// work-group: a key a thread for the scores, a dim a thread for the sums.
template <int D, bool kFp8>
__device__ void attend_plainly(const PageAttnParams& A, const int32_t* __restrict__ table, int keys,
                               int b, int hq, PlainLds& lds) {
  constexpr int kElt = kFp8 ? 1 : 2;
  static_assert(D <= kMergeThreads, "a dim a thread");
  const int tid = threadIdx.x, kvh = hq / A.gqa;
  const uint16_t* const q = A.q + b * A.q_row_stride + static_cast<int64_t>(hq) * D;
  const float s2 = kFp8 && A.k_scale ? A.scale_log2 * A.k_scale[kvh] : A.scale_log2;
  // Index of position t's first element in the caches, -1 at a masked page.
  auto row_at = [&](int t) -> int64_t {
    const int j = t >> A.block_size_log2;
    const int page = j < A.bt_width ? table[j] : -1;
    if (page < 0 || page >= A.num_blocks) return -1;
    const int64_t slot = (static_cast<int64_t>(page) << A.block_size_log2) +
                         (t & ((1 << A.block_size_log2) - 1));
    return (slot * A.num_kv_heads + kvh) * D;
  };
  auto value = [&](int64_t i) {
    if constexpr (kFp8) return __builtin_amdgcn_cvt_f32_fp8(A.v_cache[i], 0);
    return bf16_to_f32(reinterpret_cast<const uint16_t*>(A.v_cache)[i]);
  };
  float m = kNegInf, l = 0.f, o = 0.f;
  for (int t0 = 0; t0 < keys; t0 += kMergeThreads) {
    const int64_t row = t0 + tid < keys ? row_at(t0 + tid) : -1;
    float s = kNegInf;
    if (row >= 0) {
      const uint8_t* const k = A.k_cache + row * kElt;
      float dot = 0.f;
      for (int d = 0; d < D; d += 16 / kElt) {
        const uint4 x = ld16(k + d * kElt);
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (kFp8) {
            const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(w[i], false);
            const auto b = __builtin_amdgcn_cvt_pk_f32_fp8(w[i], true);
            dot = __builtin_fmaf(bf16_to_f32(q[d + 4 * i]), a[0], dot);
            dot = __builtin_fmaf(bf16_to_f32(q[d + 4 * i + 1]), a[1], dot);
            dot = __builtin_fmaf(bf16_to_f32(q[d + 4 * i + 2]), b[0], dot);
            dot = __builtin_fmaf(bf16_to_f32(q[d + 4 * i + 3]), b[1], dot);
          } else {
            dot = __builtin_fmaf(bf16_to_f32(q[d + 2 * i]), __uint_as_float(w[i] << 16), dot);
            dot = __builtin_fmaf(bf16_to_f32(q[d + 2 * i + 1]),
                                 __uint_as_float(w[i] & 0xffff0000u), dot);
          }
        }
      }
      s = dot * s2;
    }
    float most = s;
    for (int off = 32; off; off >>= 1) most = fmaxf(most, __shfl_xor(most, off, 64));
    if ((tid & 63) == 0) lds.top[tid >> 6] = most;
    __syncthreads();
    for (int w = 0; w < kMergeThreads / 64; ++w) most = fmaxf(most, lds.top[w]);
    const float m_new = fmaxf(m, most), used = m_new == kNegInf ? 0.f : m_new;
    const float alpha = __builtin_amdgcn_exp2f(m - used);
    m = m_new;
    lds.row[tid] = row;
    lds.weight[tid] = __builtin_amdgcn_exp2f(s - used);
    __syncthreads();
    l *= alpha;
    o *= alpha;
    // (in eights, whose loads are on their way together; without a row the weight is zero, and
    // the value read instead does not count)
    for (int k0 = 0; k0 < min(kMergeThreads, keys - t0); k0 += 8) {
      float x[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int64_t at = lds.row[k0 + k];
        const float y = value(max(at, int64_t{0}) + min(tid, D - 1));
        x[k] = at >= 0 ? y : 0.f;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        l += lds.weight[k0 + k];
        o = __builtin_fmaf(lds.weight[k0 + k], x[k], o);
      }
    }
    __syncthreads();
  }
  l = with_sink(l, m, A.sinks ? A.sinks[hq] * kLog2e : kNegInf);
  const float f = l > 0.f ? (kFp8 && A.v_scale ? A.v_scale[kvh] : 1.f) / l : 0.f;
  if (tid < D)
    A.out[b * A.out_row_stride + static_cast<int64_t>(hq) * D + tid] = f32_to_bf16(o * f);
}

// One work-group per (row, kv head, block of 16 query heads) merges the row's partials.
//
// A row shorter than its group's prefix has zero weights for the keys that only others see, but
// in the products with V these meet the others' values all the same: where one is infinite or
// NaN the row's sum is NaN.  Such a row that is not finite is computed again by itself (its 32
// heads over 65436 bf16 keys take 5 ms; a second pass over such ranges in the kernel above cost
// every call 2 us in set-up).
template <int D>
__global__ __launch_bounds__(kMergeThreads) void shared_prefix_merge_kernel(
    PrefixParams P, const int32_t* __restrict__ bt, int fp8) {
  constexpr int kCols = cols_of(D);
  __shared__ Folded folded[kMergeThreads];
  static_assert(sizeof(PlainLds) <= sizeof(folded), "the plain form's weights fit");
  __shared__ uint32_t again;  // bits: columns to compute again
  const PageAttnParams& A = P.A;
  const int b = blockIdx.y, v = blockIdx.x;
  const int kvh = v / A.col_blocks;
  const int in_group = 16 * (v - kvh * A.col_blocks);  // first query head, of the group
  const RowRecord rec = P.rows[b];
  const float vsc = fp8 && A.v_scale ? A.v_scale[kvh] : 1.f;
  // The row's pieces on its own line: ranges own_w, own_w + 1, ...
  const int64_t own_at = rec.own_start + static_cast<int64_t>(v) * rec.own_tiles;
  const int64_t own_w = rec.own_tiles ? quotient(own_at, rec.own_range) : 0;
  const int own_n = rec.own_tiles
                        ? static_cast<int>(
                              quotient(own_at + rec.own_tiles - 1, rec.own_range) - own_w) + 1
                        : 0;
  const int64_t own_col = (own_w + static_cast<int64_t>(b) * P.vheads + v) * P.own_cols;
  // ... and on the prefix line, found for each column.
  int pre_n = 0;
  int64_t pre_col = 0;
  const int j0 = blockIdx.z * P.merge_cols;
  if (rec.short_keys >= 0) {
    if (threadIdx.x == 0) again = 0;
    __syncthreads();
  }
  merge_pieces<D>(
      j0, min(P.merge_cols, min(16, A.gqa - in_group) - j0), folded,
      [&](int j) {
        if (rec.pre_tiles > 0) {
          const int c = rec.index * A.gqa + in_group + j;
          const int it = kvh * rec.col_items + c / kCols;
          const int64_t at = rec.pre_start + it * rec.pre_step;
          const int64_t w = quotient(at, rec.pre_range);
          const int64_t first = w + rec.pre_item + it;
          pre_n = static_cast<int>(max(
              int64_t{0},
              min(quotient(at + rec.pre_tiles - 1, rec.pre_range) - w + 1, P.pre_pieces - first)));
          pre_col = first * kCols + c % kCols;
        }
        return pre_n + own_n;
      },
      [&](int k, int j, const float*& ml, const float*& o) {
        const bool pre = k < pre_n;
        const int64_t col = pre ? pre_col + static_cast<int64_t>(k) * kCols
                                : own_col + static_cast<int64_t>(k - pre_n) * P.own_cols + j;
        ml = (pre ? P.pre_ml : P.own_ml) + 2 * col;
        o = (pre ? P.pre_o : P.own_o) + col * D;
      },
      [&](int j, int dim, const float4& o, float M, float L) {
        write_quad(A, b, kvh * A.gqa + in_group + j, D, dim, o, M, L, vsc);
        if (rec.short_keys >= 0 && !__builtin_isfinite((o.x + o.y) + (o.z + o.w)))
          atomicOr(&again, 1u << j);
      });
  if (rec.short_keys < 0) return;
  __syncthreads();
  const int32_t* const table = bt + (b - rec.index) * A.bt_row_stride;
  PlainLds& plain = *reinterpret_cast<PlainLds*>(folded);
  for (uint32_t left = __builtin_amdgcn_readfirstlane(again); left; left &= left - 1) {
    const int hq = kvh * A.gqa + in_group + __builtin_ctz(left);
    if (fp8)
      attend_plainly<D, true>(A, table, rec.short_keys, b, hq, plain);
    else
      attend_plainly<D, false>(A, table, rec.short_keys, b, hq, plain);
  }
}

// The bound on the shared tokens of a prefix that an argument of 0 (none) or more stands for.
int64_t prefix_bound(int64_t max_prefix_len) {
  return max_prefix_len == 0 || max_prefix_len > INT_MAX ? INT_MAX : max_prefix_len;
}

// Work-groups and workspace of a launch.
struct PrefixPlan {
  int wgs;
  int64_t pre_pieces, own_pieces;
  int64_t pre_o, pre_ml, own_o, own_ml, rows, bytes;  // offsets
};
PrefixPlan plan_of(int64_t batch, int64_t groups, int64_t max_prefix, int num_heads,
                   int num_kv_heads, int head_size) {
  PrefixPlan p{};
  const int gqa = num_heads / num_kv_heads;
  const int64_t cols = cols_of(head_size);
  const int64_t vheads = static_cast<int64_t>(num_kv_heads) * ((gqa + 15) / 16);
  const int own_cols = gqa < 16 ? gqa : 16;
  // Two work-groups per CU where the registers leave room for them.
  p.wgs = num_cus() * (head_size == 256 ? 1 : 2);
  // A group that shares has two rows at the least, and rounds its columns up once.
  const int64_t shared = groups < batch / 2 ? groups : batch / 2;
  if (shared > 0) {
    const int64_t items = num_kv_heads * (batch * gqa / cols + shared);
    const int64_t each = (max_prefix + kTile * kPreTiles - 1) / (kTile * kPreTiles);
    // An item and a range leave a piece where they meet: as many as both at the most.
    p.pre_pieces = items + (each < p.wgs && items * each < p.wgs ? items * each : p.wgs);
  }
  p.own_pieces = kWaves * p.wgs + batch * vheads;
  auto take = [&](int64_t bytes) {
    const int64_t at = p.bytes;
    p.bytes += (bytes + 255) / 256 * 256;
    return at;
  };
  p.pre_o = take(p.pre_pieces * cols * head_size * 4);
  p.pre_ml = take(p.pre_pieces * cols * 8);
  p.own_o = take(p.own_pieces * own_cols * head_size * 4);
  p.own_ml = take(p.own_pieces * own_cols * 8);
  p.rows = take(batch * static_cast<int64_t>(sizeof(RowRecord)));
  return p;
}

template <int D>
void launch_d(bool fp8, const PrefixParams& P, hipStream_t s, const int32_t* bt,
              const int32_t* ctx, const int32_t* cu, const int32_t* pre) {
  const dim3 grid(static_cast<unsigned>(P.wgs + 1));
  const unsigned lds = lds_groups_at<D>() + 4 * (2 * P.num_groups + 1);
  if (fp8)
    hipLaunchKernelGGL((shared_prefix_kernel<D, true>), grid, dim3(kThreads), lds, s, P, bt, ctx,
                       cu, pre);
  else
    hipLaunchKernelGGL((shared_prefix_kernel<D, false>), grid, dim3(kThreads), lds, s, P, bt, ctx,
                       cu, pre);
  hipLaunchKernelGGL((shared_prefix_merge_kernel<D>),
                     dim3(static_cast<unsigned>(P.vheads), static_cast<unsigned>(P.A.batch),
                          (P.own_cols + P.merge_cols - 1) / P.merge_cols),
                     dim3(kMergeThreads), 0, s, P, bt, fp8 ? 1 : 0);
}

}  // namespace
}  // namespace fk

using namespace fk;

extern "C" int fk_shared_prefix_decode(
    void* out, int64_t out_row_stride, const void* q, int64_t q_row_stride, const void* k_cache,
    const void* v_cache, int kv_dtype, const float* k_scale, const float* v_scale,
    const int32_t* block_tables, int64_t bt_row_stride, int64_t bt_width,
    const int32_t* cache_seqlens, int64_t batch, const int32_t* cu_groups,
    const int32_t* prefix_lens, int64_t num_groups, int64_t max_prefix_len, int num_heads,
    int num_kv_heads, int head_size, int block_size, int64_t num_blocks, float scale,
    int window_left, const float* sinks, void* workspace, int64_t workspace_bytes,
    void* stream) {
  const char* what = "fk_shared_prefix_decode";
  PageAttnParams A{};
  if (int rc = fill_page_attn(what, A, out, out_row_stride, q, q_row_stride, k_cache, v_cache,
                              kv_dtype, k_scale, v_scale, bt_row_stride, bt_width, batch,
                              num_heads, num_kv_heads, head_size, block_size, num_blocks, scale,
                              sinks))
    return rc;
  FK_REQUIRE(num_groups >= 0 && num_groups <= kMaxGroups, "%s: %lld groups outside [0, %d]", what,
             static_cast<long long>(num_groups), kMaxGroups);
  FK_REQUIRE(max_prefix_len >= 0, "%s: max_prefix_len %lld", what,
             static_cast<long long>(max_prefix_len));
  FK_REQUIRE(window_left >= -1, "%s: window_left %d must be -1 or >= 0", what, window_left);
  if (batch == 0) return FK_OK;
  max_prefix_len = prefix_bound(max_prefix_len);
  FK_REQUIRE(out && q && k_cache && v_cache && block_tables && cache_seqlens &&
                 (num_groups == 0 || (cu_groups && prefix_lens)),
             "%s: null pointer", what);
  const PrefixPlan plan = plan_of(batch, num_groups, max_prefix_len, num_heads, num_kv_heads, head_size);
  if (workspace_bytes < plan.bytes || !workspace)
    return set_error(FK_ERR_WORKSPACE, "%s: workspace of %lld bytes, %lld needed", what,
                     static_cast<long long>(workspace_bytes), static_cast<long long>(plan.bytes));
  FK_REQUIRE(aligned16(workspace), "%s: workspace must be 16-byte aligned", what);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  PrefixParams P{};
  P.A = A;
  P.num_groups = static_cast<int>(num_groups);
  P.max_prefix = static_cast<int>(max_prefix_len);
  P.window_left = window_left;
  P.unit_tiles_log2 = A.block_size_log2 - 4 < 2 ? A.block_size_log2 - 4 : 2;
  P.wgs = plan.wgs;
  P.pre_pieces = plan.pre_pieces;
  P.vheads = num_kv_heads * A.col_blocks;
  P.own_cols = A.gqa < 16 ? A.gqa : 16;
  P.merge_cols = merge_cols(batch, P.vheads, P.own_cols);
  P.pre_o = reinterpret_cast<float*>(ws + plan.pre_o);
  P.pre_ml = reinterpret_cast<float*>(ws + plan.pre_ml);
  P.own_o = reinterpret_cast<float*>(ws + plan.own_o);
  P.own_ml = reinterpret_cast<float*>(ws + plan.own_ml);
  P.rows = reinterpret_cast<RowRecord*>(ws + plan.rows);
  const bool fp8 = kv_dtype == FK_DTYPE_FP8_E4M3FN;
  hipStream_t s = as_stream(stream);
  if (head_size == 64)
    launch_d<64>(fp8, P, s, block_tables, cache_seqlens, cu_groups, prefix_lens);
  else if (head_size == 128)
    launch_d<128>(fp8, P, s, block_tables, cache_seqlens, cu_groups, prefix_lens);
  else
    launch_d<256>(fp8, P, s, block_tables, cache_seqlens, cu_groups, prefix_lens);
  return check_launch(what);
}

extern "C" int fk_shared_prefix_decode_plan(int64_t batch, int64_t num_groups,
                                            int64_t max_prefix_len, int num_heads,
                                            int num_kv_heads, int head_size,
                                            int64_t* workspace_bytes) {
  FK_REQUIRE(workspace_bytes, "fk_shared_prefix_decode_plan: null output pointer");
  FK_REQUIRE(batch >= 0 && batch <= 65535 && num_groups >= 0 && max_prefix_len >= 0 &&
                 num_kv_heads > 0 && num_heads > 0 && num_heads % num_kv_heads == 0,
             "fk_shared_prefix_decode_plan: invalid argument");
  *workspace_bytes = batch == 0 ? 0
                                : plan_of(batch, num_groups, prefix_bound(max_prefix_len),
                                          num_heads, num_kv_heads, head_size)
                                      .bytes;
  return FK_OK;
}
