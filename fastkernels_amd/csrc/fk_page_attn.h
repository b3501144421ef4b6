// Attention of blocks of 16 query columns over a list of page pieces, by the waves
// of one work-group: shared by the sparse and the shared-prefix decode kernels.
//
// A unit is a run of 16-token tiles inside one page.  The waves take the units in turn
// (wave w of n takes units w, w + n, ...), each keeps the softmax state of its units (a
// reference maximum, the sum, the unnormalised O, all fp32), and the states are merged through
// LDS with the log-sum-exp rule M = max m_w, L = sum l_w 2^(m_w - M), O = sum o_w 2^(m_w - M).
#pragma once

#include "fk_key_rows.h"

namespace fk {

struct PageAttnParams {
  uint16_t* out;
  int64_t out_row_stride;
  const uint16_t* q;
  int64_t q_row_stride;
  const uint8_t* k_cache;
  const uint8_t* v_cache;
  const float* k_scale;
  const float* v_scale;
  int num_heads;
  int num_kv_heads;
  int gqa;
  int col_blocks;  // blocks of 16 query heads per kv head
  int block_size_log2;
  int64_t num_blocks;
  float scale_log2;
  const float* sinks;
  int64_t bt_row_stride;
  int bt_width;
  int batch;
};

// Softmax state of one wave over kCB blocks of 16 query columns.  Lane (r, g) holds, for
// column r of each block, the reference maximum, its share of the sum (keys 4g .. 4g + 3 of
// every tile) and dims (D/4) g .. (D/4) g + D/4 - 1 of O: P V is computed transposed (A = V
// with row m = dim (D/16) m + slice, B = P), so that the column a lane rescales and divides
// is its own.  o[cb][d][i] is dim (D/4) g + (D/16) i + d.
//
// Two tiles go together: their scores' layouts side by side (keys 4g .. 4g + 3 of each) are
// the 32-key operand of the 16x16x32 MFMA once V's rows are paired alike, which does P V in
// half the instructions of the 16-key form.
//
// The maximum is only moved when a score exceeds it by more than kLazyMax: until then the
// weights grow to at most 2^8, which bf16 and the fp32 sums hold as exactly as smaller ones.
constexpr float kLazyMax = 8.f;
// The reference before a column's first visible key: no finite score lies below it.
constexpr float kNoMax = -__FLT_MAX__;

template <int kCB, int D, bool kFp8>
struct ColumnState {
  static constexpr int kKc = D / 32;
  static constexpr int kSl = D / 16;
  bf16x8_t qb[kCB][kKc];
  float m[kCB], l[kCB];
  floatx4_t o[kCB][kSl];

  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int cb = 0; cb < kCB; ++cb) {
      m[cb] = kNoMax;
      l[cb] = 0.f;
#pragma unroll
      for (int d = 0; d < kSl; ++d) o[cb][d] = floatx4_t{0.f, 0.f, 0.f, 0.f};
    }
  }
  // qp: the row of this lane's column of block cb (read where ok); its signs are flipped by
  // `flip` (0, or 0x80008000 where the scores' factor is negative: it is taken as positive).
  __device__ __forceinline__ void load_q(int cb, const uint16_t* qp, bool ok, uint32_t flip,
                                         int g) {
#pragma unroll
    for (int c = 0; c < kKc; ++c) {
      const int d0 = KChunks<kFp8, D>::dims(c, g);
      uint4 v = ok ? *reinterpret_cast<const uint4*>(qp + d0) : make_uint4(0, 0, 0, 0);
      v = make_uint4(v.x ^ flip, v.y ^ flip, v.z ^ flip, v.w ^ flip);
      qb[cb][c] = __builtin_bit_cast(bf16x8_t, v);
    }
  }

  // Scores of two tiles, whose K rows are in the wave's LDS kx (KChunks).
  __device__ __forceinline__ void scores(const uint8_t* kx, int lane, floatx4_t (&sa)[kCB],
                                         floatx4_t (&sb)[kCB]) const {
    uint4 ka[kKc], kb[kKc];
    KChunks<kFp8, D>::get(kx, lane, ka);
    KChunks<kFp8, D>::get(kx + KChunks<kFp8, D>::kBytes, lane, kb);
#pragma unroll
    for (int cb = 0; cb < kCB; ++cb) {
      sa[cb] = qk_scores_n(ka, qb[cb]);
      sb[cb] = qk_scores_n(kb, qb[cb]);
    }
  }
  // Scores to weights (in place; the weights are 2^(s2 score - m), s2 = scale log2(e)
  // [k_scale] >= 0), moving the maxima where they have to.  Key i of tile a is visible to this
  // lane's column of block cb where ra + i < lim[cb] (unsigned), likewise b; `full`: all are,
  // to every column.
  __device__ __forceinline__ void softmax(floatx4_t (&sa)[kCB], floatx4_t (&sb)[kCB], float s2,
                                          uint32_t ra, uint32_t rb, const uint32_t (&lim)[kCB],
                                          bool full) {
    // (Scaled first: the products are rounded alike here and in the maximum, so that no weight
    // exceeds 2^kLazyMax however great the scores; and a scale of 0 meets no infinity.)
#pragma unroll
    for (int cb = 0; cb < kCB; ++cb) {
      sa[cb] *= s2;
      sb[cb] *= s2;
    }
    if (!full) {
#pragma unroll
      for (int cb = 0; cb < kCB; ++cb)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (!(ra + i < lim[cb])) sa[cb][i] = kNegInf;
          if (!(rb + i < lim[cb])) sb[cb][i] = kNegInf;
        }
    }
    float top[kCB];
    bool move = false;
#pragma unroll
    for (int cb = 0; cb < kCB; ++cb) {
      top[cb] = fmaxf(fmaxf(fmaxf(sa[cb][0], sa[cb][1]), fmaxf(sa[cb][2], sa[cb][3])),
                      fmaxf(fmaxf(sb[cb][0], sb[cb][1]), fmaxf(sb[cb][2], sb[cb][3])));
      move |= top[cb] > m[cb] + kLazyMax;
    }
    if (__ballot(move) != 0) {
#pragma unroll
      for (int cb = 0; cb < kCB; ++cb) {
        const float m_new = fmaxf(m[cb], pair_max(top[cb]));
        const float alpha = __builtin_amdgcn_exp2f(m[cb] - m_new);
        m[cb] = m_new;
        l[cb] *= alpha;
#pragma unroll
        for (int d = 0; d < kSl; ++d) o[cb][d] *= alpha;
      }
    }
#pragma unroll
    for (int cb = 0; cb < kCB; ++cb) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        sa[cb][i] = __builtin_amdgcn_exp2f(sa[cb][i] - m[cb]);
        sb[cb][i] = __builtin_amdgcn_exp2f(sb[cb][i] - m[cb]);
      }
    }
#pragma unroll
    for (int cb = 0; cb < kCB; ++cb)
      l[cb] += (sa[cb][0] + sa[cb][1]) + (sa[cb][2] + sa[cb][3]) +
               ((sb[cb][0] + sb[cb][1]) + (sb[cb][2] + sb[cb][3]));
  }
  // O += P V.  V rows that no column sees (ra + i >= span) may hold anything: zeroed, so that
  // a zero weight never meets a NaN.  The weights are rounded to bf16 (2^-9 relative on
  // average, of either sign), as in the decode kernel; the sum is of the unrounded ones.
  __device__ __forceinline__ void values(DTile<kFp8, D>& a, DTile<kFp8, D>& b,
                                         const floatx4_t (&pa)[kCB], const floatx4_t (&pb)[kCB],
                                         uint32_t ra, uint32_t rb, uint32_t span, bool full) {
    if (!full) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int q = 0; q < DTile<kFp8, D>::kVWords; ++q) {
          a.v[i][q] = ra + i < span ? a.v[i][q] : 0u;
          b.v[i][q] = rb + i < span ? b.v[i][q] : 0u;
        }
    }
    short4_t va[kSl], vb[kSl];
    if constexpr (kFp8) {
      const bool all[4] = {true, true, true, true};
      v_operands_fp8(a, true, all, va);
      v_operands_fp8(b, true, all, vb);
    } else {
      v_operands_w(a.v, va);
      v_operands_w(b.v, vb);
    }
#pragma unroll
    for (int cb = 0; cb < kCB; ++cb) {
      const float fa[4] = {pa[cb][0], pa[cb][1], pa[cb][2], pa[cb][3]};
      const float fb[4] = {pb[cb][0], pb[cb][1], pb[cb][2], pb[cb][3]};
      const uint2 x = __builtin_bit_cast(uint2, p_operand(fa));
      const uint2 y = __builtin_bit_cast(uint2, p_operand(fb));
      const bf16x8_t p = __builtin_bit_cast(bf16x8_t, make_uint4(x.x, x.y, y.x, y.y));
#pragma unroll
      for (int d = 0; d < kSl; ++d) {
        const uint2 v = __builtin_bit_cast(uint2, va[d]), w = __builtin_bit_cast(uint2, vb[d]);
        o[cb][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            __builtin_bit_cast(bf16x8_t, make_uint4(v.x, v.y, w.x, w.y)), p, o[cb][d], 0, 0, 0);
      }
    }
  }
};

// Where a wave's lanes read a tile: byte offsets from the tile's first row of the kv head.
template <bool kFp8, int D>
struct TileLanes {
  uint32_t k, k_step, v[4];
  __device__ __forceinline__ TileLanes(int num_kv_heads, int lane) {
    constexpr int kElt = kFp8 ? 1 : 2;
    using K = KChunks<kFp8, D>;
    const int r = lane & 15, g = lane >> 4;
    const uint32_t row = static_cast<uint32_t>(num_kv_heads) * D * kElt;
    k = lane / K::kPieces * row + 16 * (lane % K::kPieces);
    k_step = K::kRows * row;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (4 * g + i) * row + (D / 16) * r * kElt;
  }
};
// Issue a tile's K or V loads; row: its first row of the kv head (wave-uniform).
template <bool kFp8, int D>
__device__ __forceinline__ void load_tile_k(const uint8_t* row, const TileLanes<kFp8, D>& at,
                                            DTile<kFp8, D>& t) {
#pragma unroll
  for (int i = 0; i < DTile<kFp8, D>::kKLoads; ++i)
    t.k[i] = ld16(row + static_cast<int64_t>(i) * at.k_step + at.k);
}
template <bool kFp8, int D>
__device__ __forceinline__ void load_tile_v(const uint8_t* row, const TileLanes<kFp8, D>& at,
                                            DTile<kFp8, D>& t) {
#pragma unroll
  for (int i = 0; i < 4; ++i) ld_words(row + at.v[i], t.v[i]);
}

// What a wave's columns see of positions [from, to): lim[cb] keys from `from` on for this lane's
// column of block cb, at most `span` for any column of the wave and at least `least`.
template <int kCB>
struct Limits {
  uint32_t lim[kCB];
  uint32_t span, least;
};

// Streams units first, first + step, ... (< units) of a list into st, of each the positions in
// [from, to).  unit_at(u, page, tok) gives unit u's page (-1: nothing to read) and its first
// token's position; a unit is 1 << unit_tiles_log2 tiles of its page.  Lane k looks up the
// wave's unit k, 64 at a time, and the units with something to read are packed to the front, so
// that the tile loop only meets those.  The K rows of the next two tiles are requested when this
// step's are in LDS (kx: two tiles of the wave's own), the V rows when P V has used this step's.
// limits() is asked once, when the first rows are on their way.
template <int kCB, int D, bool kFp8, class UnitAt, class LimitsOf>
__device__ __forceinline__ void stream_units(const PageAttnParams& P,
                                             ColumnState<kCB, D, kFp8>& st, UnitAt unit_at,
                                             int units, int first, int step, int unit_tiles_log2,
                                             int from, int to, LimitsOf limits, int kvh, float s2,
                                             uint8_t* kx, int lane) {
  constexpr int kElt = kFp8 ? 1 : 2;
  const int g = lane >> 4;
  const int page_mask = (1 << P.block_size_log2) - 1;
  const TileLanes<kFp8, D> at(P.num_kv_heads, lane);
  const int64_t row_bytes = static_cast<int64_t>(P.num_kv_heads) * D * kElt;
  const uint8_t* const kh = P.k_cache + static_cast<int64_t>(kvh) * D * kElt;
  const uint8_t* const vh = P.v_cache + static_cast<int64_t>(kvh) * D * kElt;
  Limits<kCB> lm;
  bool asked = false;
  for (int64_t u0 = first; u0 < units; u0 += static_cast<int64_t>(64) * step) {
    const int64_t u = u0 + static_cast<int64_t>(lane) * step;
    int page = -1, tok = 0;
    if (u < units) unit_at(static_cast<int>(u), page, tok);
    const bool ok = page >= 0 && page < P.num_blocks && tok < to &&
                    static_cast<int64_t>(tok) + (kTile << unit_tiles_log2) > from;
    const uint64_t oks = __ballot(ok);
    const int n = __builtin_popcountll(oks);
    if (n == 0) continue;
    // lane k <- the k-th lane with ok set
    const int rank = __builtin_popcountll(oks & ((uint64_t{1} << lane) - 1));
    const int dst = ok ? rank : n + (lane - rank);
    page = __builtin_amdgcn_ds_permute(dst << 2, page);
    tok = __builtin_amdgcn_ds_permute(dst << 2, tok);
    const int tiles = n << unit_tiles_log2;
    const int sub_mask = (1 << unit_tiles_log2) - 1;
    // First row and position (less from; unsigned, so one before it wraps past span) of tile x.
    auto row_of = [&](int x, uint32_t& rel) -> int64_t {
      const int pg = __builtin_amdgcn_readlane(page, x >> unit_tiles_log2);
      const int t0 = __builtin_amdgcn_readlane(tok, x >> unit_tiles_log2) +
                     kTile * (x & sub_mask);
      rel = static_cast<uint32_t>(t0) - static_cast<uint32_t>(from);
      return ((static_cast<int64_t>(pg) << P.block_size_log2) + (t0 & page_mask)) * row_bytes;
    };
    DTile<kFp8, D> a, b;
    uint32_t ra, rb;
    int64_t at_a = row_of(0, ra), at_b = row_of(min(1, tiles - 1), rb);
    load_tile_k(kh + at_a, at, a);
    load_tile_k(kh + at_b, at, b);
    load_tile_v(vh + at_a, at, a);
    load_tile_v(vh + at_b, at, b);
    loads_issued();
    if (!asked) {
      lm = limits();
      asked = true;
    }
    for (int x = 0; x < tiles; x += 2) {
      floatx4_t sa[kCB], sb[kCB];
      KChunks<kFp8, D>::put(a, kx, lane);
      KChunks<kFp8, D>::put(b, kx + KChunks<kFp8, D>::kBytes, lane);
      // (past the last tiles, these are read once more: the number of loads in flight stays
      // known to the compiler's wait counts)
      uint32_t na, nb;
      at_a = row_of(min(x + 2, tiles - 1), na);
      at_b = row_of(min(x + 3, tiles - 1), nb);
      load_tile_k(kh + at_a, at, a);
      load_tile_k(kh + at_b, at, b);
      loads_issued();
      st.scores(kx, lane, sa, sb);
      loads_issued();
      if (x + 1 >= tiles) rb = lm.span;  // no second tile: masked
      const bool full = ra < lm.least && lm.least - ra >= kTile && rb < lm.least &&
                        lm.least - rb >= kTile;
      st.softmax(sa, sb, s2, ra + 4 * g, rb + 4 * g, lm.lim, full);
      st.values(a, b, sa, sb, ra + 4 * g, rb + 4 * g, lm.span, full);
      load_tile_v(vh + at_a, at, a);
      load_tile_v(vh + at_b, at, b);
      loads_issued();
      ra = na;
      rb = nb;
    }
  }
}

// Merges the waves' states of all column blocks and hands each quad of adjacent dims of each
// of the ncols columns to emit(column, dim, o, M, L): o = O[dim .. dim + 3] before the division.
// lds: merge_lds_floats(16 kCB columns at most), of the waves' K rows until all have come here;
// every thread of the work-group calls it, and may write to lds again only after a barrier.
template <int kWaves, int D>
constexpr int merge_lds_floats(int cols) { return kWaves * cols * (D + 4 + 2); }
template <int kWaves, int kCB, int D, bool kFp8, class Emit>
__device__ __forceinline__ void merge_waves(const ColumnState<kCB, D, kFp8>& st, float* lds,
                                            int wave, int lane, int ncols, Emit emit) {
  constexpr int kRow = D + 4;  // (rows 16 bytes apart modulo the banks)
  constexpr int kSl = D / 16;
  const int r = lane & 15, g = lane >> 4;
  float2* const xm = reinterpret_cast<float2*>(lds + kWaves * ncols * kRow);  // (m, l)
  __syncthreads();  // lds was the waves' K rows
#pragma unroll
  for (int cb = 0; cb < kCB; ++cb) {
    const float l = pair_sum(st.l[cb]);
    const int j = 16 * cb + r;
    if (j < ncols) {
      if (g == 0) xm[wave * ncols + j] = make_float2(st.m[cb], l);
      float* dst = lds + (wave * ncols + j) * kRow + (D / 4) * g;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int d = 0; d < kSl; d += 4)
          *reinterpret_cast<float4*>(dst + kSl * i + d) =
              make_float4(st.o[cb][d][i], st.o[cb][d + 1][i], st.o[cb][d + 2][i],
                          st.o[cb][d + 3][i]);
    }
  }
  __syncthreads();
#pragma unroll 2
  for (int x = threadIdx.x; x < ncols * (D / 4); x += kWaves * 64) {
    const int j = x / (D / 4), dim = 4 * (x % (D / 4));
    float2 s[kWaves];
    float4 o[kWaves];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      s[w] = xm[w * ncols + j];
      o[w] = *reinterpret_cast<const float4*>(lds + (w * ncols + j) * kRow + dim);
    }
    float M = s[0].x;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) M = fmaxf(M, s[w].x);
    float L = 0.f;
    float4 u = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float f = __builtin_amdgcn_exp2f(s[w].x - M);
      L = __builtin_fmaf(s[w].y, f, L);
      u.x = __builtin_fmaf(o[w].x, f, u.x);
      u.y = __builtin_fmaf(o[w].y, f, u.y);
      u.z = __builtin_fmaf(o[w].z, f, u.z);
      u.w = __builtin_fmaf(o[w].w, f, u.w);
    }
    emit(j, dim, u, M, L);
  }
}

// A wave's state of its first column block as a partial: O [columns][D] and (m, l) per column.
template <int kCB, int D, bool kFp8>
__device__ __forceinline__ void write_partial(const ColumnState<kCB, D, kFp8>& st, float* o,
                                              float* ml, int lane, int ncols) {
  constexpr int kSl = D / 16;
  const int r = lane & 15, g = lane >> 4;
  const float l = pair_sum(st.l[0]);
  if (r >= ncols) return;
  if (g == 0) *reinterpret_cast<float2*>(ml + 2 * r) = make_float2(st.m[0], l);
  float* dst = o + r * D + (D / 4) * g;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int d = 0; d < kSl; d += 4)
      *reinterpret_cast<float4*>(dst + kSl * i + d) =
          make_float4(st.o[0][d][i], st.o[0][d + 1][i], st.o[0][d + 2][i], st.o[0][d + 3][i]);
}

// Running log-sum-exp state of four dims of a column over partials.
struct Folded {
  float M, L;
  float4 o;
  __device__ __forceinline__ void reset() {
    M = kNoMax;
    L = 0.f;
    o = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  __device__ __forceinline__ void add(float m, float l, const float4& x) {
    const float top = fmaxf(M, m);
    const float fa = __builtin_amdgcn_exp2f(M - top), fb = __builtin_amdgcn_exp2f(m - top);
    M = top;
    L = L * fa + l * fb;
    o.x = o.x * fa + x.x * fb;
    o.y = o.y * fa + x.y * fb;
    o.z = o.z * fa + x.z * fb;
    o.w = o.w * fa + x.w * fb;
  }
};

// Merges the partials of columns j0 .. j0 + nc - 1, kMergeThreads threads.  A thread folds four dims of a
// column; where the columns leave threads over, the pieces are dealt out among them and the
// threads' states folded through LDS (`folded`, one per thread).  pieces(j) is the number of
// column j's pieces, at(k, j, ml, o) where piece k's (m, l) and O are; emit(j, dim, o, M, L)
// gets the merged state.
constexpr int kMergeThreads = 256;
// Columns of a merge's work-group: all `cols` of a row and block of heads where there are many
// of those, fewer where the work-groups would not make two a CU, so that more threads share a
// column's pieces.  (4 rows of two prefixes of 17000 and 21000 tokens: a call of 40 us instead
// of 51.  With twice the work-groups 64 rows take 6.5 us instead of 5.5.)
inline int merge_cols(int64_t rows, int vheads, int cols) {
  const int64_t per = (rows * vheads * cols + 2 * num_cus() - 1) / (2 * num_cus());
  return static_cast<int>(per < 1 ? 1 : per < cols ? per : cols);
}
constexpr int kMergeAhead = 8;  // pieces whose loads are in flight
template <int D, class Pieces, class At, class Emit>
__device__ __forceinline__ void merge_pieces(int j0, int nc, Folded* folded, Pieces pieces, At at,
                                             Emit emit) {
  const int tid = threadIdx.x;
  const int items = nc * (D / 4);
  if (items <= 0) return;  // (a work-group behind the last column)
  const int slices = max(1, kMergeThreads / items);
  for (int x0 = 0; x0 < items; x0 += kMergeThreads) {
    const int x = x0 + (slices > 1 ? tid % items : tid);
    const int slice = slices > 1 ? tid / items : 0;
    const bool ok = x < items && slice < slices;
    const int j = j0 + x / (D / 4), dim = 4 * (x % (D / 4));
    Folded f;
    f.reset();
    const int n = ok ? pieces(j) : 0;
    for (int k0 = slice; k0 < n; k0 += kMergeAhead * slices) {
      float2 s[kMergeAhead];
      float4 o[kMergeAhead];
#pragma unroll
      for (int u = 0; u < kMergeAhead; ++u) {
        const float *ml, *row;
        at(min(k0 + u * slices, n - 1), j, ml, row);
        s[u] = *reinterpret_cast<const float2*>(ml);
        o[u] = *reinterpret_cast<const float4*>(row + dim);
      }
#pragma unroll
      for (int u = 0; u < kMergeAhead; ++u)
        if (k0 + u * slices < n) f.add(s[u].x, s[u].y, o[u]);
    }
    if (slices > 1) {
      folded[tid] = f;
      __syncthreads();
      if (slice == 0)
        for (int u = 1; u < slices; ++u) {
          const Folded& y = folded[x + u * items];
          f.add(y.M, y.L, y.o);
        }
    }
    if (ok && slice == 0) emit(j, dim, f.o, f.M, f.L);
  }
}

// Output of a finished row: O (scaled by the V scale of fp8 pages) over the sum, which the
// head's sink joins; a row that saw no key is zero.
__device__ __forceinline__ void write_quad(const PageAttnParams& P, int64_t row, int hq, int D,
                                           int dim, const float4& o, float M, float L,
                                           float vsc) {
  const float sink = P.sinks ? P.sinks[hq] * kLog2e : kNegInf;
  const float l = with_sink(L, M, sink);
  const float f = l > 0.f ? vsc / l : 0.f;
  const bf16x2_t a = {static_cast<__bf16>(o.x * f), static_cast<__bf16>(o.y * f)};
  const bf16x2_t b = {static_cast<__bf16>(o.z * f), static_cast<__bf16>(o.w * f)};
  *reinterpret_cast<uint2*>(P.out + row * P.out_row_stride + static_cast<int64_t>(hq) * D + dim) =
      make_uint2(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b));
}

// Checks the arguments the entry points share and fills A from them.
inline int fill_page_attn(const char* what, PageAttnParams& A, void* out, int64_t out_row_stride,
                          const void* q, int64_t q_row_stride, const void* k_cache,
                          const void* v_cache, int kv_dtype, const float* k_scale,
                          const float* v_scale, int64_t bt_row_stride, int64_t bt_width,
                          int64_t batch, int num_heads, int num_kv_heads, int head_size,
                          int block_size, int64_t num_blocks, float scale, const float* sinks) {
  FK_REQUIRE(batch >= 0 && batch <= 65535, "%s: batch %lld outside [0, 65535]", what,
             static_cast<long long>(batch));
  FK_REQUIRE(num_kv_heads > 0 && num_heads > 0 && num_heads % num_kv_heads == 0 &&
                 num_heads <= 65535,
             "%s: %d query heads over %d kv heads", what, num_heads, num_kv_heads);
  FK_REQUIRE(kv_dtype == FK_DTYPE_BF16 || kv_dtype == FK_DTYPE_FP8_E4M3FN,
             "%s: the caches must be bf16 or fp8 e4m3fn", what);
  FK_REQUIRE(block_size >= 16 && block_size <= (1 << 30) && (block_size & (block_size - 1)) == 0,
             "%s: block_size %d must be a power of two >= 16", what, block_size);
  FK_REQUIRE(num_blocks > 0 && num_blocks <= 0x7fffffff, "%s: num_blocks %lld", what,
             static_cast<long long>(num_blocks));
  FK_REQUIRE(bt_width >= 0 && bt_width <= 0x7fffffff && bt_row_stride >= 0,
             "%s: block table of %lld columns", what, static_cast<long long>(bt_width));
  if (head_size != 64 && head_size != 128 && head_size != 256)
    return set_error(FK_ERR_UNSUPPORTED, "%s: head_size %d unsupported (64, 128 or 256)", what,
                     head_size);
  FK_REQUIRE(aligned16(q) && aligned16(out) && aligned16(k_cache) && aligned16(v_cache) &&
                 q_row_stride % 8 == 0 && out_row_stride % 8 == 0,
             "%s: q, out and the caches must have 16-byte aligned rows", what);
  A.out = static_cast<uint16_t*>(out);
  A.out_row_stride = out_row_stride;
  A.q = static_cast<const uint16_t*>(q);
  A.q_row_stride = q_row_stride;
  A.k_cache = static_cast<const uint8_t*>(k_cache);
  A.v_cache = static_cast<const uint8_t*>(v_cache);
  A.k_scale = k_scale;
  A.v_scale = v_scale;
  A.num_heads = num_heads;
  A.num_kv_heads = num_kv_heads;
  A.gqa = num_heads / num_kv_heads;
  A.col_blocks = (A.gqa + 15) / 16;
  A.block_size_log2 = 31 - __builtin_clz(static_cast<unsigned>(block_size));
  A.num_blocks = num_blocks;
  A.scale_log2 = scale * kLog2e;
  A.sinks = sinks;
  A.bt_row_stride = bt_row_stride;
  A.bt_width = static_cast<int>(bt_width);
  A.batch = static_cast<int>(batch);
  return FK_OK;
}

}  // namespace fk
