// Decode attention over the 4-bit cache (fk_mxfp4.h): one query row per sequence, or a few (a
// step that checks drafted tokens).
//
// The query rows of a sequence times the query heads of one kv head are the columns of matrix
// products with the keys: S = K Q^T, then O^T += V^T P^T, 16 columns at a time.  Codes become
// bf16 operands in registers, exactly (fk_mxfp4.h), with their scales, so that the products,
// the softmax and the sums are those of a bf16 cache of the same values.
//
// Work.  Items (sequence, kv head, kCB blocks of 16 columns) of 32-key steps lie on one line, cut
// into equal ranges (fk_lines.h); the four waves of a work-group take the steps of a part in
// turn and merge their states through LDS.  An item inside one range is finished there; of the
// others each part leaves a partial state, which a second launch merges.
//
// Measured (a call, captured): 64 rows over 512 .. 8192 tokens, 32 / 8 heads of 128, pages of 16:
// 69 us, 4.7 TB/s (bf16 pages 212, fp8 116); 8 rows over up to 65536, 64 / 8 heads 75 us; 32
// sequences with up to 4 rows 99 us, 3.5 TB/s.  What bounds it: memory with one column block;
// with two, the vector instructions between the loads (48% of the time; a step's 300, of which 64
// are conversions), as with 20 / 20 heads of 64 (112 us), where one column of 16 is used.  (What the
// kernels of two column blocks and of head size 256 spill, 132 and 176 bytes a lane, is touched once
// a part.)  A third set of codes in registers costs 5% (more spills, code), codes through LDS three
// steps ahead 3 to 20%.
//
// Lanes.  Lane (r, g), r = lane % 16, g = lane / 16.  A step's keys 8 j + i are row 4 j + i of
// tile A and keys 8 j + 4 + i row 4 j + i of tile B, so that column r's scores of tile A and B
// in lane (r, g) are keys 8 g .. 8 g + 7: P's operand.  K: lane (r, g) holds the quarter g of
// the dims of a row, V: the sixteenth r of the dims of keys 8 g .. 8 g + 7.
#include "fk_lines.h"
#include "fk_mxfp4.h"
#include "fk_page_attn.h"
#include "fk_query_rows.h"

namespace fk {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * 64;
constexpr int kStep = 32;  // keys
// What a part costs besides its steps, in steps: queries, first loads, the waves' merge.  (64 rows:
// 72 us, 86 with none.)
constexpr int kPad = 8;

struct Mxfp4Params {
  PageAttnParams A;
  const uint8_t* k_scales;
  const uint8_t* v_scales;
  int rows;         // rows of q and out
  int most;         // rows of a sequence at most
  int window_left;
  int wgs;
  int merge_cols;
  float* o;         // [2 wgs][columns][D]
  float* ml;        // [2 wgs][columns] (maximum, sum)
  LineRecord* records;
};

template <int D>
struct Codes {
  static constexpr int kWords = D / 32;  // 32-bit words of K per tile, of V per four keys
  static constexpr int kScales = D == 256 ? 2 : 1;
  uint32_t k[2][kWords];
  uint2 ks[kScales];  // scales of keys 8 j .. 8 j + 7 of this lane's blocks
  uint32_t v[2][kWords];
  uint2 vs;
};

// Loads a step whose halves of 16 keys are in pages page0 and page1 (of a kv head), at places tok
// and tok + 16 modulo a page.  kOne: pages hold whole steps.  Then what differs between lanes is
// the same in every step, and a load is a scalar base and a lane's own 32 bits; in pages of 16 keys
// the halves lie anywhere, and lanes select between them.
template <int D, bool kOne>
__device__ __forceinline__ void load_step(const Mxfp4Params& P, uint32_t page0, uint32_t page1,
                                          uint32_t tok, int r, int g, Codes<D>& c) {
  constexpr int kRow = D / 2, kBlocks = D / 32;
  const int log2 = kOne ? P.A.block_size_log2 : 4;
  const uint32_t k_row = 8 * ((r >> 2) & 1) + (r & 3), v_row = 8 * (g & 1);
  const uint8_t *k, *v, *ks, *vs;
  if constexpr (kOne) {
    const uint64_t row = (static_cast<uint64_t>(page0) << log2) + tok;
    const uint64_t s_row = (static_cast<uint64_t>(page0) * kBlocks << log2) + tok;
    k = P.A.k_cache + row * kRow + ((16 * (r >> 3) + k_row) * kRow + g * (D / 8));
    v = P.A.v_cache + row * kRow + ((16 * (g >> 1) + v_row) * kRow + r * (D / 8));
    ks = P.k_scales + s_row +
         ((static_cast<uint32_t>(g * D / 128) << log2) + 16 * (r >> 3) + (k_row & 8));
    vs = P.v_scales + s_row + ((static_cast<uint32_t>(r * D / 512) << log2) + 16 * (g >> 1) + v_row);
  } else {
    const uint64_t pk = r >> 3 ? page1 : page0, pv = g >> 1 ? page1 : page0;
    k = P.A.k_cache + pk * (16 * kRow) + (k_row * kRow + g * (D / 8));
    v = P.A.v_cache + pv * (16 * kRow) + (v_row * kRow + r * (D / 8));
    ks = P.k_scales + pk * (16 * kBlocks) +
         ((static_cast<uint32_t>(g * D / 128) << log2) + (k_row & 8));
    vs = P.v_scales + pv * (16 * kBlocks) +
         ((static_cast<uint32_t>(r * D / 512) << log2) + v_row);
  }
  ld_words(k, c.k[0]);
  ld_words(k + 4 * kRow, c.k[1]);
#pragma unroll
  for (int i = 0; i < Codes<D>::kScales; ++i)
    c.ks[i] = ld8(ks + (static_cast<uint32_t>(i) << log2));
  ld_words(v, c.v[0]);
  ld_words(v + 4 * kRow, c.v[1]);
  c.vs = ld8(vs);
}

// K operands of tile t: chunk c is dims (D/4) g + 8 c .. + 7 of this lane's row.
template <int D>
__device__ __forceinline__ void k_operands(const Codes<D>& c, int t, int r, uint4 (&k)[D / 32]) {
#pragma unroll
  for (int x = 0; x < D / 32; ++x) {
    const uint2 s = c.ks[D == 256 ? x >> 2 : 0];
    const float scale = __uint_as_float(((t ? s.y : s.x) >> (8 * (r & 3))) << 23);
    k[x] = fp4x8_to_bf16x8(c.k[t][x], scale);
  }
}

// Codes of byte `b` (of D / 32) of key i (of four) as two bf16.
template <int D>
__device__ __forceinline__ uint32_t v_pair(const uint32_t (&w)[D / 32], int i, int b,
                                           const float (&s)[4]) {
  const int byte = i * (D / 32) + b;  // of the lane's 16ths of four keys
  const uint32_t x = w[byte >> 2];
  switch (byte & 3) {
    case 0: return fp4x2_to_bf16x2<0>(x, s[i]);
    case 1: return fp4x2_to_bf16x2<1>(x, s[i]);
    case 2: return fp4x2_to_bf16x2<2>(x, s[i]);
    default: return fp4x2_to_bf16x2<3>(x, s[i]);
  }
}

// O += P V of one step.  Keys whose bit in `keep` is clear (of this lane's eight) count as zero:
// their weights are, and what is there may be NaN.  kSome: only the columns of blocks whose bit in
// `columns` is set change.
template <int kCB, int D, bool kSome>
__device__ __forceinline__ void values(ColumnState<kCB, D, false>& st, const Codes<D>& c,
                                       const floatx4_t (&pa)[kCB], const floatx4_t (&pb)[kCB],
                                       uint32_t keep, uint32_t columns) {
  bf16x8_t p[kCB];
#pragma unroll
  for (int cb = 0; cb < kCB; ++cb) {
    const float fa[4] = {pa[cb][0], pa[cb][1], pa[cb][2], pa[cb][3]};
    const float fb[4] = {pb[cb][0], pb[cb][1], pb[cb][2], pb[cb][3]};
    const uint2 x = __builtin_bit_cast(uint2, p_operand(fa));
    const uint2 y = __builtin_bit_cast(uint2, p_operand(fb));
    p[cb] = __builtin_bit_cast(bf16x8_t, make_uint4(x.x, x.y, y.x, y.y));
  }
  // (a scale of 2^-127 in place of one that does not count: no code then makes a NaN)
  uint2 vs = c.vs;
  if (keep != 0xffu) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      vs.x = keep >> i & 1 ? vs.x : vs.x & ~(0xffu << (8 * i));
      vs.y = keep >> (4 + i) & 1 ? vs.y : vs.y & ~(0xffu << (8 * i));
    }
  }
  const float sa[4] = {scale_of<0>(vs.x), scale_of<1>(vs.x), scale_of<2>(vs.x),
                       scale_of<3>(vs.x)};
  const float sb[4] = {scale_of<0>(vs.y), scale_of<1>(vs.y), scale_of<2>(vs.y),
                       scale_of<3>(vs.y)};
#pragma unroll
  for (int b = 0; b < D / 32; ++b) {
    uint32_t a[4], x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a[i] = v_pair<D>(c.v[0], i, b, sa);
      x[i] = v_pair<D>(c.v[1], i, b, sb);
    }
    const uint4 even = make_uint4(lo_pair(a[0], a[1]), lo_pair(a[2], a[3]), lo_pair(x[0], x[1]),
                                  lo_pair(x[2], x[3]));
    const uint4 odd = make_uint4(hi_pair(a[0], a[1]), hi_pair(a[2], a[3]), hi_pair(x[0], x[1]),
                                 hi_pair(x[2], x[3]));
#pragma unroll
    for (int cb = 0; cb < kCB; ++cb) {
      const floatx4_t e = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
          __builtin_bit_cast(bf16x8_t, even), p[cb], st.o[cb][2 * b], 0, 0, 0);
      const floatx4_t f = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
          __builtin_bit_cast(bf16x8_t, odd), p[cb], st.o[cb][2 * b + 1], 0, 0, 0);
      if constexpr (kSome) {
        const bool mine = columns >> cb & 1;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          st.o[cb][2 * b][i] = mine ? e[i] : st.o[cb][2 * b][i];
          st.o[cb][2 * b + 1][i] = mine ? f[i] : st.o[cb][2 * b + 1][i];
        }
      } else {
        st.o[cb][2 * b] = e;
        st.o[cb][2 * b + 1] = f;
      }
    }
  }
}

template <int kCB, int D, bool kOne>
__global__ __launch_bounds__(kThreads)
__attribute__((amdgpu_waves_per_eu(2))) void mxfp4_decode_kernel(
    Mxfp4Params P, const int32_t* __restrict__ bt, const int32_t* __restrict__ ctx_lens,
    const int32_t* __restrict__ cu) {
  constexpr int kCols = 16 * kCB;
  __shared__ LineLds<kThreads> line;
  extern __shared__ __align__(16) float lds[];
  // The queries' operands, where they are 32 registers or more: of those that then have no
  // register, a step's reload comes after the next step's loads, and waits for them.
  constexpr bool kQLds = kCB * D >= 256;
  uint4* const q_lds = reinterpret_cast<uint4*>(lds);  // (the merge's, until the part's last step)
  const PageAttnParams& A = P.A;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int r = lane & 15, g = lane >> 4;
  const float s2 = A.scale_log2;
  const int page_mask = (1 << A.block_size_log2) - 1;

  auto items_of = [&](const SeqRows& s) {
    LineItems x;
    int none;
    row_keys(s, 0, P.window_left, x.from, none);
    row_keys(s, s.rows - 1, P.window_left, none, x.to);
    // (past the table's end there is nothing to see)
    x.to = static_cast<int>(min(min(static_cast<int64_t>(x.to), int64_t{0x7fffff00}),
                                static_cast<int64_t>(A.bt_width) << A.block_size_log2));
    x.from &= -kStep;
    x.steps = x.to > x.from ? (x.to - x.from - 1) / kStep + 1 : 1;
    x.items = A.num_kv_heads * ((s.rows * A.gqa + kCols - 1) / kCols);
    return x;
  };
  auto body = [&](int b, const SeqRows& sr, const LineItems& x, int it, int s_lo, int s_hi,
                  int64_t slot, int64_t) {
    const int col_items = x.items / A.num_kv_heads;
    const int kvh = it / col_items;
    const int col0 = (it - kvh * col_items) * kCols;
    const int n_cols = min(kCols, sr.rows * A.gqa - col0);
    ColumnState<kCB, D, false> st;
    st.reset();
    int lo[kCB], hi[kCB];  // keys that this lane's column sees
    int all_lo = 0, all_hi = 0x7fffffff;  // that every column sees
#pragma unroll
    for (int cb = 0; cb < kCB; ++cb) {
      const int c = 16 * cb + r;
      const bool ok = c < n_cols;
      const int i = ok ? (col0 + c) / A.gqa : 0, hq = kvh * A.gqa + (ok ? (col0 + c) % A.gqa : 0);
      row_keys(sr, i, P.window_left, lo[cb], hi[cb]);
      const uint16_t* const qp =
          A.q + (sr.row0 + i) * A.q_row_stride + static_cast<int64_t>(hq) * D + g * (D / 4);
#pragma unroll
      for (int k = 0; k < D / 32; ++k) {
        if (kQLds && (cb * (D / 32) + k) % kWaves != wave) continue;
        const uint32_t flip = s2 < 0.f ? 0x80008000u : 0u;
        uint4 v = ok ? *reinterpret_cast<const uint4*>(qp + 8 * k) : make_uint4(0, 0, 0, 0);
        v = make_uint4(v.x ^ flip, v.y ^ flip, v.z ^ flip, v.w ^ flip);
        if constexpr (kQLds)
          q_lds[(cb * (D / 32) + k) * 64 + lane] = v;
        else
          st.qb[cb][k] = __builtin_bit_cast(bf16x8_t, v);
      }
      if (!ok) hi[cb] = lo[cb] = 0;
    }
    if constexpr (kQLds) __syncthreads();
    auto score = [&](int cb, const uint4 (&k)[D / 32]) {
      if constexpr (!kQLds) {
        return qk_scores_n(k, st.qb[cb]);
      } else {
        bf16x8_t q[D / 32];
#pragma unroll
        for (int x = 0; x < D / 32; ++x)
          q[x] = __builtin_bit_cast(bf16x8_t, q_lds[(cb * (D / 32) + x) * 64 + lane]);
        return qk_scores_n(k, q);
      }
    };
    const int row_a = col0 / A.gqa, row_z = (col0 + n_cols - 1) / A.gqa;
    int none;
    row_keys(sr, row_z, P.window_left, all_lo, none);
    row_keys(sr, row_a, P.window_left, none, all_hi);
    const float abs_s2 = __builtin_fabsf(s2);

    const int32_t* const table = bt + b * A.bt_row_stride;
    // The wave's steps, 32 at a time: lane 2 m + h looks up half h of the m-th.
    for (int s0 = s_lo + wave; s0 < s_hi; s0 += 32 * kWaves) {
      const int64_t key = x.from + static_cast<int64_t>(s0 + (lane >> 1) * kWaves) * kStep +
                          16 * (lane & 1);
      int page = -1;
      if (key < x.to) {
        const int64_t j = key >> A.block_size_log2;
        page = j < A.bt_width ? table[j] : -1;
        if (page >= A.num_blocks) page = -1;
      }
      const uint64_t there = __ballot(page >= 0);
      page = max(page, 0) * A.num_kv_heads + kvh;  // (below: a head's page)
      const int n = min(32, (s_hi - s0 + kWaves - 1) / kWaves);
      auto load = [&](int m, Codes<D>& c) {
        const int t0 = x.from + (s0 + m * kWaves) * kStep;
        load_step<D, kOne>(P, __builtin_amdgcn_readlane(page, 2 * m),
                           __builtin_amdgcn_readlane(page, 2 * m + 1), t0 & page_mask, r, g, c);
      };
      auto attend = [&](int m, const Codes<D>& c) {
        const int t0 = x.from + (s0 + m * kWaves) * kStep;
        const uint32_t halves = there >> (2 * m) & 3;
        floatx4_t sa[kCB], sb[kCB];
        {
          uint4 k[D / 32];
          k_operands<D>(c, 0, r, k);
#pragma unroll
          for (int cb = 0; cb < kCB; ++cb) sa[cb] = score(cb, k);
          k_operands<D>(c, 1, r, k);
#pragma unroll
          for (int cb = 0; cb < kCB; ++cb) sb[cb] = score(cb, k);
        }
#pragma unroll
        for (int cb = 0; cb < kCB; ++cb) {
          sa[cb] *= abs_s2;
          sb[cb] *= abs_s2;
        }
        const bool full = halves == 3 && t0 >= all_lo && all_hi - t0 >= kStep;
        const bool half = halves >> (g >> 1) & 1;
        uint32_t keep = 0xff;
        if (!full) {
          keep = 0;
#pragma unroll
          for (int cb = 0; cb < kCB; ++cb)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int t = t0 + 8 * g + i;
              const bool see = half && t >= lo[cb] && t < hi[cb];
              if (!see) (i < 4 ? sa : sb)[cb][i & 3] = kNegInf;
              keep |= see ? 1u << i : 0u;
            }
        }
        const uint32_t none[kCB] = {};
        st.softmax(sa, sb, 1.f, 0, 0, none, true);
        if (full) {
          values<kCB, D, false>(st, c, sa, sb, 0xff, 0);
          return;
        }
        // Any column's keys: the lanes of a group of 16 hold the same ones.
#pragma unroll
        for (int off = 8; off; off >>= 1) keep |= __shfl_xor(keep, off, 64);
        // A NaN or an infinity among them that some of the columns do not see stays with the
        // others: row by row.
        bool odd = false;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          odd |= (keep >> i & 1) &&
                 !all_finite((i < 4 ? c.vs.x : c.vs.y) >> (8 * (i & 3)) & 0xff);
        if (row_a == row_z || __ballot(odd) == 0) {
          values<kCB, D, false>(st, c, sa, sb, keep, 0);
          return;
        }
#pragma unroll 1
        for (int i = row_a; i <= row_z; ++i) {
          int row_lo, row_hi;
          row_keys(sr, i, P.window_left, row_lo, row_hi);
          uint32_t see = 0, mine = 0;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int t = t0 + 8 * g + k;
            see |= half && t >= row_lo && t < row_hi ? 1u << k : 0u;
          }
#pragma unroll
          for (int cb = 0; cb < kCB; ++cb)
            mine |= (col0 + 16 * cb + r) / A.gqa == i ? 1u << cb : 0u;
          values<kCB, D, true>(st, c, sa, sb, see, mine);
        }
      };
      Codes<D> c0, c1;
      load(0, c0);
      for (int m = 0; m < n; m += 2) {
        load(min(m + 1, n - 1), c1);
        loads_issued();
        attend(m, c0);
        load(min(m + 2, n - 1), c0);
        loads_issued();
        if (m + 1 < n) attend(m + 1, c1);
      }
    }
    float* const po = P.o + slot * kCols * D;
    float* const pm = P.ml + slot * kCols * 2;
    merge_waves<kWaves>(st, lds, wave, lane, n_cols,
                        [&](int j, int dim, const float4& o, float M, float L) {
                          if (slot < 0) {
                            write_quad(A, sr.row0 + (col0 + j) / A.gqa,
                                       kvh * A.gqa + (col0 + j) % A.gqa, D, dim, o, M, L, 1.f);
                            return;
                          }
                          *reinterpret_cast<float4*>(po + j * D + dim) = o;
                          if (dim == 0)
                            *reinterpret_cast<float2*>(pm + 2 * j) = make_float2(M, L);
                        });
    __syncthreads();
  };
  walk_line(line, A.batch, P.wgs, blockIdx.x, kWaves, kPad, P.records,
            [&](int b) { return seq_rows(cu, ctx_lens, b, P.rows, P.most); }, items_of, body);
}

// One work-group per (query row, kv head, some of its columns): merges the pieces of an item that
// ranges cut.
template <int kCB, int D>
__global__ __launch_bounds__(kMergeThreads) void mxfp4_merge_kernel(
    Mxfp4Params P, const int32_t* __restrict__ ctx_lens, const int32_t* __restrict__ cu) {
  constexpr int kCols = 16 * kCB;
  __shared__ Folded folded[kMergeThreads];
  const PageAttnParams& A = P.A;
  const int t = blockIdx.y, kvh = blockIdx.x;
  int b, vis;
  if (!query_row(cu, ctx_lens, A.batch, t, b, vis)) return;
  const SeqRows s = seq_rows(cu, ctx_lens, b, P.rows, P.most);
  const int i = t - s.row0;
  if (i < 0 || i >= s.rows) return;
  const LineRecord rec = P.records[b];
  const int col_items = (s.rows * A.gqa + kCols - 1) / kCols;
  const int j0 = blockIdx.z * P.merge_cols;
  const int j1 = min(j0 + P.merge_cols, A.gqa);
  // The row's columns, item by item.
  for (int j = j0; j < j1;) {
    const int c = i * A.gqa + j;
    const int it = kvh * col_items + c / kCols;
    const int in = c % kCols, nc = min(j1 - j, kCols - in);
    const LinePieces pieces(rec, it, kPad);
    if (pieces.n > 1) {
      merge_pieces<D>(
          0, nc, folded, [&](int) { return pieces.n; },
          [&](int k, int x, const float*& ml, const float*& o) {
            const int64_t at = pieces.slot(k) * kCols + in + x;
            ml = P.ml + 2 * at;
            o = P.o + at * D;
          },
          [&](int x, int dim, const float4& o, float M, float L) {
            write_quad(A, t, kvh * A.gqa + j + x, D, dim, o, M, L, 1.f);
          });
      __syncthreads();
    }
    j += nc;
  }
}

struct Mxfp4Plan {
  int wgs, blocks;  // work-groups, column blocks of an item
  int64_t o, ml, records, bytes;
};
Mxfp4Plan plan_of(int64_t batch, int64_t max_seqlen_q, int num_heads, int num_kv_heads,
                  int head_size) {
  Mxfp4Plan p{};
  const int64_t cols = max_seqlen_q * (num_heads / num_kv_heads);
  p.blocks = cols > 16 && head_size < 256 ? 2 : 1;
  p.wgs = num_cus() * 2;
  auto take = [&](int64_t bytes) {
    const int64_t at = p.bytes;
    p.bytes += (bytes + 255) / 256 * 256;
    return at;
  };
  p.o = take(int64_t{2} * p.wgs * p.blocks * 16 * head_size * 4);
  p.ml = take(int64_t{2} * p.wgs * p.blocks * 16 * 8);
  p.records = take(batch * static_cast<int64_t>(sizeof(LineRecord)));
  return p;
}

template <int kCB, int D>
void launch(const Mxfp4Params& P, hipStream_t s, const int32_t* bt, const int32_t* ctx,
            const int32_t* cu) {
  const unsigned lds = 4 * merge_lds_floats<kWaves, D>(16 * kCB);
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(P.wgs + 1), dim3(kThreads), lds, s, P, bt, ctx, cu);
  };
  P.A.block_size_log2 >= 5 ? go(mxfp4_decode_kernel<kCB, D, true>)
                           : go(mxfp4_decode_kernel<kCB, D, false>);
  hipLaunchKernelGGL((mxfp4_merge_kernel<kCB, D>),
                     dim3(P.A.num_kv_heads, P.rows,
                          (P.A.gqa + P.merge_cols - 1) / P.merge_cols),
                     dim3(kMergeThreads), 0, s, P, ctx, cu);
}

}  // namespace
}  // namespace fk

using namespace fk;

extern "C" int fk_mxfp4_paged_decode(
    void* out, int64_t out_row_stride, const void* q, int64_t q_row_stride, const void* k_cache,
    const void* v_cache, const void* k_scales, const void* v_scales, const int32_t* block_tables,
    int64_t bt_row_stride, int64_t bt_width, const int32_t* cache_seqlens,
    const int32_t* cu_seqlens_q, int64_t batch, int64_t rows, int64_t max_seqlen_q, int num_heads,
    int num_kv_heads, int head_size, int block_size, int64_t num_blocks, float scale,
    int window_left, const float* sinks, void* workspace, int64_t workspace_bytes,
    void* stream) {
  const char* what = "fk_mxfp4_paged_decode";
  PageAttnParams A{};
  if (int rc = fill_page_attn(what, A, out, out_row_stride, q, q_row_stride, k_cache, v_cache,
                              FK_DTYPE_BF16, nullptr, nullptr, bt_row_stride, bt_width, batch,
                              num_heads, num_kv_heads, head_size, block_size, num_blocks, scale,
                              sinks))
    return rc;
  FK_REQUIRE(rows >= 0 && rows <= 65535, "%s: rows %lld outside [0, 65535]", what,
             static_cast<long long>(rows));
  FK_REQUIRE(window_left >= -1, "%s: window_left %d must be -1 or >= 0", what, window_left);
  FK_REQUIRE(max_seqlen_q >= 1 && max_seqlen_q <= 65535, "%s: max_seqlen_q %lld", what,
             static_cast<long long>(max_seqlen_q));
  // (a head's page is counted in 32 bits; more are over 2 TB)
  FK_REQUIRE(num_blocks * num_kv_heads <= 0x7fffffff, "%s: %lld pages of %d heads", what,
             static_cast<long long>(num_blocks), num_kv_heads);
  // (a lane's offset to a block's scales is 32 bits)
  FK_REQUIRE(block_size <= 1 << 28, "%s: block_size %d above 2^28", what, block_size);
  if (batch == 0 || rows == 0) return FK_OK;
  FK_REQUIRE(out && q && k_cache && v_cache && k_scales && v_scales && block_tables &&
                 cache_seqlens,
             "%s: null pointer", what);
  FK_REQUIRE(aligned16(k_scales) && aligned16(v_scales), "%s: scales must be 16-byte aligned",
             what);
  if (!cu_seqlens_q) max_seqlen_q = 1;
  const Mxfp4Plan plan = plan_of(batch, max_seqlen_q, num_heads, num_kv_heads, head_size);
  if (workspace_bytes < plan.bytes || !workspace)
    return set_error(FK_ERR_WORKSPACE, "%s: workspace of %lld bytes, %lld needed", what,
                     static_cast<long long>(workspace_bytes), static_cast<long long>(plan.bytes));
  FK_REQUIRE(aligned16(workspace), "%s: workspace must be 16-byte aligned", what);
  uint8_t* const ws = static_cast<uint8_t*>(workspace);
  Mxfp4Params P{};
  P.A = A;
  P.k_scales = static_cast<const uint8_t*>(k_scales);
  P.v_scales = static_cast<const uint8_t*>(v_scales);
  P.rows = static_cast<int>(rows);
  P.most = static_cast<int>(max_seqlen_q);
  P.window_left = window_left;
  P.wgs = plan.wgs;
  P.merge_cols = merge_cols(rows, num_kv_heads, A.gqa);
  P.o = reinterpret_cast<float*>(ws + plan.o);
  P.ml = reinterpret_cast<float*>(ws + plan.ml);
  P.records = reinterpret_cast<LineRecord*>(ws + plan.records);
  hipStream_t s = as_stream(stream);
  if (head_size == 64)
    plan.blocks == 1 ? launch<1, 64>(P, s, block_tables, cache_seqlens, cu_seqlens_q)
                     : launch<2, 64>(P, s, block_tables, cache_seqlens, cu_seqlens_q);
  else if (head_size == 128)
    plan.blocks == 1 ? launch<1, 128>(P, s, block_tables, cache_seqlens, cu_seqlens_q)
                     : launch<2, 128>(P, s, block_tables, cache_seqlens, cu_seqlens_q);
  else
    launch<1, 256>(P, s, block_tables, cache_seqlens, cu_seqlens_q);
  return check_launch(what);
}

extern "C" int fk_mxfp4_paged_decode_plan(int64_t batch, int64_t max_seqlen_q, int num_heads,
                                          int num_kv_heads, int head_size,
                                          int64_t* workspace_bytes) {
  FK_REQUIRE(workspace_bytes, "fk_mxfp4_paged_decode_plan: null output pointer");
  FK_REQUIRE(batch >= 0 && batch <= 65535 && max_seqlen_q >= 1 && max_seqlen_q <= 65535 &&
                 num_kv_heads > 0 && num_heads > 0 && num_heads % num_kv_heads == 0,
             "fk_mxfp4_paged_decode_plan: invalid argument");
  *workspace_bytes =
      batch == 0 ? 0 : plan_of(batch, max_seqlen_q, num_heads, num_kv_heads, head_size).bytes;
  return FK_OK;
}
