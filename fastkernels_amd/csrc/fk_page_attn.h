// Attention of one block of up to 16 query columns over a list of page pieces, by the waves
// of one work-group: shared by the sparse and the shared-prefix decode kernels.
//
// A unit is a run of 16-token tiles inside one page.  The waves take the units in turn
// (wave w of n takes units w, w + n, ...), each keeps the softmax state of its units (running
// maximum, sum, unnormalised O, all fp32), and the states are merged through LDS with the
// log-sum-exp rule M = max m_w, L = sum l_w 2^(m_w - M), O = sum o_w 2^(m_w - M).
#pragma once

#include "fk_attn_tile.h"

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

// Waves of a work-group: their O states (columns x D floats each) take at most 64 KB of LDS.
template <int kG, int D>
constexpr int page_attn_waves() { return kG * D > 2048 ? 4 : 8; }

// Softmax state of one wave over up to 16 query columns.  Lane (r, g) holds column r's
// maximum and its share of the sum, and O[column 4g + i][dims (D/16) r ..].
template <int kG, int D, bool kFp8>
struct ColumnState {
  static constexpr int kKc = D / 32;
  static constexpr int kSl = D / 16;
  bf16x8_t qb[kKc];
  float m, l;
  floatx4_t o[kSl];

  // qp: the row of this lane's column (read where ok).
  __device__ __forceinline__ void init(const uint16_t* qp, bool ok, int g) {
#pragma unroll
    for (int c = 0; c < kKc; ++c) {
      const int d0 = kFp8 ? (D / 4) * g + 8 * c : 32 * c + 8 * g;
      const uint4 v = ok ? *reinterpret_cast<const uint4*>(qp + d0) : make_uint4(0, 0, 0, 0);
      qb[c] = __builtin_bit_cast(bf16x8_t, v);
    }
    m = kNegInf;
    l = 0.f;
#pragma unroll
    for (int d = 0; d < kSl; ++d) o[d] = floatx4_t{0.f, 0.f, 0.f, 0.f};
  }

  // One tile of 16 tokens.  This lane's rows are visible where rel0 + i < span (unsigned:
  // rel0 = position of row 4g less the first visible one); full: all 16 rows are.
  __device__ __forceinline__ void tile(const DTile<kFp8, D>& cur, float ks, float s2,
                                       uint32_t rel0, uint32_t span, bool full, int g) {
    uint4 kc[kKc];
    k_chunks_d(cur, kc);
    const floatx4_t acc = qk_scores_n(kc, qb);
    float s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = kFp8 ? acc[i] * ks * s2 : acc[i] * s2;
    if (!full) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (!(rel0 + i < span)) s[i] = kNegInf;
    }
    const float m_new = fmaxf(m, pair_max(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]))));
    const float m_use = m_new == kNegInf ? 0.f : m_new;
    const float alpha = m_new == kNegInf ? 1.f : __builtin_amdgcn_exp2f(m - m_use);
    float pr[4];
    float psum = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      pr[i] = __builtin_amdgcn_exp2f(s[i] - m_use);
      psum += pr[i];
    }
    l = l * alpha + psum;
    m = m_new;
    if (__ballot(alpha != 1.f) != 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float a = row_value<kG>(alpha, g, i);
#pragma unroll
        for (int d = 0; d < kSl; ++d) o[d][i] *= a;
      }
    }
    // The weights enter P V as bf16 (half a step, 2^-9 relative, each; their signs differ
    // from key to key), as in the decode kernel.
    const short4_t pa = p_operand(pr);
    // V rows that are masked may hold anything: zeroed, so that 0 never meets a NaN.
    short4_t vb[kSl];
    if constexpr (kFp8) {
      bool keep[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) keep[i] = rel0 + i < span;
      v_operands_fp8(cur, full, keep, vb);
    } else {
      uint32_t vw[4][D / 32];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v_words(cur, i, full || rel0 + i < span, vw[i]);
      v_operands_w(vw, vb);
    }
    pv_accumulate_n(o, pa, vb);
  }
};

// Issues the loads of the tile whose first token is slot0 (of the cache's slots), kv head
// kvh.
template <bool kFp8, int D>
__device__ __forceinline__ void load_page_tile(const PageAttnParams& P, int64_t slot0, int kvh,
                                               int r, int g, DTile<kFp8, D>& t) {
  constexpr int kElt = kFp8 ? 1 : 2;
  const int64_t row_bytes = static_cast<int64_t>(P.num_kv_heads) * D * kElt;
  const int64_t at = slot0 * row_bytes + static_cast<int64_t>(kvh) * D * kElt;
  const uint8_t* krow = P.k_cache + at + r * row_bytes;
  const uint8_t* vrow = P.v_cache + at + 4 * g * row_bytes + (D / 16) * r * kElt;
#pragma unroll
  for (int c = 0; c < DTile<kFp8, D>::kKLoads; ++c)
    t.k[c] = ld16(kFp8 ? krow + (D / 4) * g + 16 * c : krow + (32 * c + 8 * g) * 2);
#pragma unroll
  for (int i = 0; i < 4; ++i) ld_words(vrow + i * row_bytes, t.v[i]);
}

// Streams units first, first + step, ... (< units) of the list into st.  unit_at(u, page,
// tok0) gives unit u's page (-1: nothing to read) and its first token's position; a unit has
// unit_tiles tiles of its page, of which those from position `hi` on, or wholly before `lo`,
// are skipped.  Lane k looks up the wave's unit k, 64 at a time, and the units with something
// to read are packed to the front, so that the tile loop only meets those.
template <int kG, int D, bool kFp8, int U, class UnitAt>
__device__ __forceinline__ void stream_units(const PageAttnParams& P, ColumnState<kG, D, kFp8>& st,
                                             UnitAt unit_at, int units, int first, int step,
                                             int unit_tiles_log2, int lo, int hi, int kvh,
                                             float ks, int lane) {
  const int r = lane & 15, g = lane >> 4;
  const uint32_t span = static_cast<uint32_t>(max(hi - lo, 0));
  const int page_mask = (1 << P.block_size_log2) - 1;
  for (int64_t u0 = first; u0 < units; u0 += static_cast<int64_t>(64) * step) {
    const int64_t u = u0 + static_cast<int64_t>(lane) * step;
    int page = -1, tok = 0;
    if (u < units) unit_at(static_cast<int>(u), page, tok);
    const bool ok = page >= 0 && page < P.num_blocks && tok < hi &&
                    static_cast<int64_t>(tok) + (kTile << unit_tiles_log2) > lo;
    const uint64_t oks = __ballot(ok);
    const int n = __builtin_popcountll(oks);
    // lane k <- the k-th lane with ok set
    const int rank = __builtin_popcountll(oks & ((uint64_t{1} << lane) - 1));
    const int to = ok ? rank : n + (lane - rank);
    page = __builtin_amdgcn_ds_permute(to << 2, page);
    tok = __builtin_amdgcn_ds_permute(to << 2, tok);
    const int tiles = n << unit_tiles_log2;
    const int sub_mask = (1 << unit_tiles_log2) - 1;
    for (int x0 = 0; x0 < tiles; x0 += U) {
      DTile<kFp8, D> buf[U];
      int t0[U];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int x = min(x0 + k, tiles - 1);
        const int pg = __builtin_amdgcn_readlane(page, x >> unit_tiles_log2);
        t0[k] = __builtin_amdgcn_readlane(tok, x >> unit_tiles_log2) + kTile * (x & sub_mask);
        const int64_t slot = (static_cast<int64_t>(pg) << P.block_size_log2) +
                             (t0[k] & page_mask);
        load_page_tile<kFp8, D>(P, slot, kvh, r, g, buf[k]);
      }
#pragma unroll
      for (int k = 0; k < U; ++k) {
        // (unsigned: a tile that begins before lo wraps past span)
        const uint32_t rel = static_cast<uint32_t>(t0[k]) - static_cast<uint32_t>(lo);
        if (x0 + k < tiles)
          st.tile(buf[k], ks, P.scale_log2, rel + 4 * g, span,
                  rel < span && span - rel >= kTile, g);
      }
    }
  }
}

// Merges the waves' states and hands each pair of adjacent dims of each of the ncols columns
// to emit(column, dim, x, y, M, L): x and y are O[dim], O[dim + 1] before the division.
template <int kG, int D, bool kFp8, class Emit>
__device__ __forceinline__ void merge_waves(ColumnState<kG, D, kFp8>& st, float* lds, int wave,
                                            int lane, int ncols, Emit emit) {
  constexpr int kWaves = page_attn_waves<kG, D>();
  constexpr int kSl = D / 16;
  const int r = lane & 15, g = lane >> 4;
  float* const xo = lds;                         // [wave][column][D]
  float* const xm = lds + kWaves * kG * D;       // [wave][column] maximum
  float* const xl = xm + kWaves * kG;            // [wave][column] sum
  st.l = pair_sum(st.l);
  if (g == 0 && r < kG) {
    xm[wave * kG + r] = st.m;
    xl[wave * kG + r] = st.l;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int j = 4 * g + i;
    if (j < kG) {
      float* dst = xo + (wave * kG + j) * D + kSl * r;
#pragma unroll
      for (int d = 0; d < kSl; d += 4)
        *reinterpret_cast<float4*>(dst + d) =
            make_float4(st.o[d][i], st.o[d + 1][i], st.o[d + 2][i], st.o[d + 3][i]);
    }
  }
  __syncthreads();
  for (int x = threadIdx.x; x < ncols * (D / 2); x += kWaves * 64) {
    const int j = x / (D / 2), dim = 2 * (x % (D / 2));
    float M = kNegInf;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) M = fmaxf(M, xm[w * kG + j]);
    float L = 0.f, a = 0.f, b = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float mw = xm[w * kG + j];
      const float f = mw == kNegInf ? 0.f : __builtin_amdgcn_exp2f(mw - M);
      const float2 v = *reinterpret_cast<const float2*>(xo + (w * kG + j) * D + dim);
      L = __builtin_fmaf(xl[w * kG + j], f, L);
      a = __builtin_fmaf(v.x, f, a);
      b = __builtin_fmaf(v.y, f, b);
    }
    emit(j, dim, a, b, M, L);
  }
}
template <int kG, int D>
constexpr int merge_lds_floats() { return page_attn_waves<kG, D>() * kG * (D + 2); }

// Output of a finished row: O (scaled by the V scale of fp8 pages) over the sum, which the
// head's sink joins; a row that saw no key is zero.
__device__ __forceinline__ void write_pair(const PageAttnParams& P, int64_t row, int hq, int D,
                                           int dim, float x, float y, float M, float L,
                                           float vsc) {
  const float sink = P.sinks ? P.sinks[hq] * kLog2e : kNegInf;
  const float l = with_sink(L, M, sink);
  const float f = l > 0.f ? vsc / l : 0.f;
  const bf16x2_t pk = {static_cast<__bf16>(x * f), static_cast<__bf16>(y * f)};
  *reinterpret_cast<uint32_t*>(P.out + row * P.out_row_stride + static_cast<int64_t>(hq) * D +
                               dim) = __builtin_bit_cast(uint32_t, pk);
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
