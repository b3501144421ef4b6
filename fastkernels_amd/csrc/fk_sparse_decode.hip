// Decode attention over the pages selected for each query row and kv head.
//
//   out[t, hq] = sum_k softmax_k(scale q[t, hq] . K[k]) V[k]   over the keys k < vis(t) of the
//   pages block_indices[t, kv head of hq, :] of the row's sequence (entries outside the
//   table, or at pages that hold no visible key, are skipped; a page listed twice counts
//   twice).  Sinks join the denominator; a row without a visible key is zero.
//
// A work-group takes a share of the list of one (query row, kv head, block of 16 query heads),
// its waves every fourth unit of the share (fk_page_attn.h).  Where the rows are too few to fill
// the chip, the list is shared among up to kMaxParts work-groups and a second launch merges
// their partials.  The kv head varies fastest in the grid: the rows of a sequence that check
// drafted tokens, which mostly select the same pages, run side by side on one XCD's L2.
//
// Bound by memory where the lists are many: 64 rows of 32 / 8 heads, 2048 bf16 keys a list, take
// 96.9 us (538 MB, 5.6 TB/s); bound by the latency of its steps, partly of L2 hits, where rows
// share pages: 85 rows that check drafted tokens over fp8 pages 53.1 us (137 MB that differ, 370
// read).  One row takes 5.8 us and its merge 4.0.  Two or more steps of loads ahead gain nothing
// (96 and 60 us, more 148 and 63), nor does another order of the lists over the XCDs.
#include <limits.h>

#include "fk_page_attn.h"
#include "fk_query_rows.h"

namespace fk {
namespace {

struct SparseParams {
  PageAttnParams A;
  const int32_t* indices;
  int64_t idx_row_stride, idx_head_stride;
  int keep;
  int unit_tiles_log2;
  int parts;     // work-groups per list
  int cols;      // columns of a partial: min(16, gqa)
  int merge_cols;  // of which a work-group of the merge takes so many
  float* part_o; // [(row, virtual head), part][cols][D], then (maximum, sum) per column
  float* part_ml;
};

// Registers: two waves a SIMD, or one at head size 256 (the query, a step's K and V rows and O
// take more than 256 there).
constexpr int kWaves = 4;
constexpr int kMaxParts = 64;

template <int D, bool kFp8>
__global__ __launch_bounds__(kWaves * 64)
__attribute__((amdgpu_waves_per_eu(D == 256 ? 1 : 2))) void sparse_decode_kernel(
    SparseParams P, const int32_t* __restrict__ bt, const int32_t* __restrict__ ctx,
    const int32_t* __restrict__ cu) {
  extern __shared__ __align__(16) float lds[];  // merge_lds_floats of the group's columns
  const PageAttnParams& A = P.A;
  const int t = blockIdx.y, part = blockIdx.z;
  int b, vis;
  if (!query_row(cu, ctx, A.batch, t, b, vis)) return;
  const int kvh = blockIdx.x / A.col_blocks;
  const int qbase = kvh * A.gqa + 16 * (blockIdx.x - kvh * A.col_blocks);
  const int ncols = min(16, (kvh + 1) * A.gqa - qbase);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int r = lane & 15, g = lane >> 4;
  ColumnState<1, D, kFp8> st;
  st.reset();
  const float s2 = kFp8 && A.k_scale ? A.scale_log2 * A.k_scale[kvh] : A.scale_log2;
  st.load_q(0, A.q + t * A.q_row_stride + static_cast<int64_t>(qbase + r) * D, r < ncols,
            s2 < 0.f ? 0x80008000u : 0u, g);
  const float vsc = kFp8 && A.v_scale ? A.v_scale[kvh] : 1.f;
  const int32_t* list = P.indices + t * P.idx_row_stride + kvh * P.idx_head_stride;
  const int32_t* bt_row = bt + b * A.bt_row_stride;
  // units of a page: its tiles in runs of 1 << unit_tiles_log2
  const int per_log2 = A.block_size_log2 - 4 - P.unit_tiles_log2;
  auto unit_at = [&](int u, int& page, int& tok) {
    const int j = list[u >> per_log2];
    if (j < 0 || j >= A.bt_width) return;
    const int64_t pos = (static_cast<int64_t>(j) << A.block_size_log2) +
                        ((u & ((1 << per_log2) - 1)) << (4 + P.unit_tiles_log2));
    if (pos >= vis) return;
    page = bt_row[j];
    tok = static_cast<int>(pos);
  };
  const uint32_t span = static_cast<uint32_t>(max(vis, 0));
  stream_units(A, st, unit_at, P.keep << per_log2, kWaves * part + wave, kWaves * P.parts,
               P.unit_tiles_log2, 0,
               max(vis, 0), [&] { return Limits<1>{{span}, span, span}; }, kvh,
               __builtin_fabsf(s2),
               reinterpret_cast<uint8_t*>(lds) + wave * 2 * KChunks<kFp8, D>::kBytes, lane);
  if (P.parts == 1) {
    merge_waves<kWaves>(st, lds, wave, lane, ncols,
                        [&](int j, int dim, const float4& o, float M, float L) {
                          write_quad(A, t, qbase + j, D, dim, o, M, L, vsc);
                        });
  } else {
    const int64_t col =
        ((static_cast<int64_t>(t) * gridDim.x + blockIdx.x) * P.parts + part) * P.cols;
    merge_waves<kWaves>(st, lds, wave, lane, ncols,
                        [&](int j, int dim, const float4& o, float M, float L) {
                          *reinterpret_cast<float4*>(P.part_o + (col + j) * D + dim) = o;
                          if (dim == 0)
                            *reinterpret_cast<float2*>(P.part_ml + 2 * (col + j)) =
                                make_float2(M, L);
                        });
  }
}

// One work-group per (query row, virtual head) merges the list's parts.
template <int D>
__global__ __launch_bounds__(kMergeThreads) void sparse_merge_kernel(
    SparseParams P, const int32_t* __restrict__ ctx, const int32_t* __restrict__ cu, int fp8) {
  __shared__ Folded folded[kMergeThreads];
  const PageAttnParams& A = P.A;
  const int t = blockIdx.y;
  int b, vis;
  if (!query_row(cu, ctx, A.batch, t, b, vis)) return;
  const int kvh = blockIdx.x / A.col_blocks;
  const int qbase = kvh * A.gqa + 16 * (blockIdx.x - kvh * A.col_blocks);
  const float vsc = fp8 && A.v_scale ? A.v_scale[kvh] : 1.f;
  const int64_t col0 = (static_cast<int64_t>(t) * gridDim.x + blockIdx.x) * P.parts * P.cols;
  const int j0 = blockIdx.z * P.merge_cols;
  merge_pieces<D>(
      j0, min(P.merge_cols, min(16, (kvh + 1) * A.gqa - qbase) - j0), folded, [&](int) { return P.parts; },
      [&](int k, int j, const float*& ml, const float*& o) {
        const int64_t col = col0 + static_cast<int64_t>(k) * P.cols + j;
        ml = P.part_ml + 2 * col;
        o = P.part_o + col * D;
      },
      [&](int j, int dim, const float4& o, float M, float L) {
        write_quad(A, t, qbase + j, D, dim, o, M, L, vsc);
      });
}

// Work-groups per list: where the lists are fewer than the CUs, as many as make two per CU, each
// with eight tiles at the least: two per wave in pages of 16, one or two units of a wave's own in
// larger pages, where a unit is up to four tiles (with pages of 64 and more two of the four waves
// then have none).  (With a list for each CU, parts only add their merge: 512 lists of 2048 keys
// 98 us in one part, 109 in two.)
int parts_of(int64_t rows, int64_t keep, int vheads, int block_size) {
  const int64_t lists = rows * vheads;
  const int64_t tiles = keep * (block_size / kTile);
  const int64_t cus = num_cus();
  int64_t parts = lists > 0 && lists < cus ? (2 * cus + lists - 1) / lists : 1;
  if (parts > tiles / (2 * kWaves)) parts = tiles / (2 * kWaves);
  return static_cast<int>(parts < 1 ? 1 : parts > kMaxParts ? kMaxParts : parts);
}
int64_t part_bytes(int64_t rows, int vheads, int parts, int cols, int head_size) {
  return parts > 1 ? rows * vheads * parts * cols * (head_size + 2) * 4 : 0;
}

template <int D>
void launch_d(bool fp8, const SparseParams& P, int64_t rows, hipStream_t s, const int32_t* bt,
              const int32_t* ctx, const int32_t* cu) {
  const unsigned vheads = P.A.num_kv_heads * P.A.col_blocks;
  const dim3 grid(vheads, static_cast<unsigned>(rows), static_cast<unsigned>(P.parts));
  const int rows_lds = kWaves * 2 * (fp8 ? KChunks<true, D>::kBytes : KChunks<false, D>::kBytes);
  const int merge_lds = 4 * merge_lds_floats<kWaves, D>(P.cols);
  const unsigned lds = merge_lds > rows_lds ? merge_lds : rows_lds;
  if (fp8)
    hipLaunchKernelGGL((sparse_decode_kernel<D, true>), grid, dim3(kWaves * 64), lds, s, P, bt,
                       ctx, cu);
  else
    hipLaunchKernelGGL((sparse_decode_kernel<D, false>), grid, dim3(kWaves * 64), lds, s, P, bt,
                       ctx, cu);
  if (P.parts > 1)
    hipLaunchKernelGGL((sparse_merge_kernel<D>),
                       dim3(vheads, static_cast<unsigned>(rows),
                            (P.cols + P.merge_cols - 1) / P.merge_cols),
                       dim3(kMergeThreads), 0, s, P, ctx, cu, fp8 ? 1 : 0);
}

}  // namespace
}  // namespace fk

using namespace fk;

extern "C" int fk_sparse_paged_decode(
    void* out, int64_t out_row_stride, const void* q, int64_t q_row_stride, const void* k_cache,
    const void* v_cache, int kv_dtype, const float* k_scale, const float* v_scale,
    const int32_t* block_tables, int64_t bt_row_stride, int64_t bt_width,
    const int32_t* cache_seqlens, const int32_t* cu_seqlens_q, int64_t batch, int64_t rows,
    const int32_t* block_indices, int64_t idx_row_stride, int64_t idx_head_stride, int64_t keep,
    int num_heads, int num_kv_heads, int head_size, int block_size, int64_t num_blocks,
    float scale, const float* sinks, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "fk_sparse_paged_decode";
  PageAttnParams A{};
  if (int rc = fill_page_attn(what, A, out, out_row_stride, q, q_row_stride, k_cache, v_cache,
                              kv_dtype, k_scale, v_scale, bt_row_stride, bt_width, batch,
                              num_heads, num_kv_heads, head_size, block_size, num_blocks, scale,
                              sinks))
    return rc;
  FK_REQUIRE(rows >= 0 && rows <= 65535, "%s: %lld query rows outside [0, 65535]", what,
             static_cast<long long>(rows));
  FK_REQUIRE(cu_seqlens_q || rows <= batch, "%s: %lld query rows for %lld sequences", what,
             static_cast<long long>(rows), static_cast<long long>(batch));
  FK_REQUIRE(keep >= 0 && keep <= (INT_MAX >> 1) / (block_size / 16),
             "%s: %lld selected blocks", what, static_cast<long long>(keep));
  if (rows == 0 || batch == 0) return FK_OK;
  FK_REQUIRE(out && q && k_cache && v_cache && block_tables && cache_seqlens &&
                 (block_indices || keep == 0),
             "%s: null pointer", what);
  SparseParams P{};
  P.A = A;
  P.indices = block_indices;
  P.idx_row_stride = idx_row_stride;
  P.idx_head_stride = idx_head_stride;
  P.keep = static_cast<int>(keep);
  P.unit_tiles_log2 = A.block_size_log2 - 4 < 2 ? A.block_size_log2 - 4 : 2;
  const int vheads = num_kv_heads * A.col_blocks;
  P.cols = A.gqa < 16 ? A.gqa : 16;
  P.merge_cols = merge_cols(rows, vheads, P.cols);
  P.parts = parts_of(rows, keep, vheads, block_size);
  const int64_t need = part_bytes(rows, vheads, P.parts, P.cols, head_size);
  if (need > 0) {
    if (!workspace || workspace_bytes < need)
      return set_error(FK_ERR_WORKSPACE, "%s: workspace of %lld bytes, %lld needed", what,
                       static_cast<long long>(workspace_bytes), static_cast<long long>(need));
    FK_REQUIRE(aligned16(workspace), "%s: workspace must be 16-byte aligned", what);
    P.part_o = static_cast<float*>(workspace);
    P.part_ml = P.part_o + rows * vheads * P.parts * P.cols * head_size;
  }
  const bool fp8 = kv_dtype == FK_DTYPE_FP8_E4M3FN;
  hipStream_t s = as_stream(stream);
  if (head_size == 64)
    launch_d<64>(fp8, P, rows, s, block_tables, cache_seqlens, cu_seqlens_q);
  else if (head_size == 128)
    launch_d<128>(fp8, P, rows, s, block_tables, cache_seqlens, cu_seqlens_q);
  else
    launch_d<256>(fp8, P, rows, s, block_tables, cache_seqlens, cu_seqlens_q);
  return check_launch(what);
}

extern "C" int fk_sparse_paged_decode_plan(int64_t rows, int64_t keep, int num_heads,
                                           int num_kv_heads, int head_size, int block_size,
                                           int64_t* workspace_bytes) {
  FK_REQUIRE(workspace_bytes, "fk_sparse_paged_decode_plan: null output pointer");
  FK_REQUIRE(rows >= 0 && rows <= 65535 && keep >= 0 && num_kv_heads > 0 && num_heads > 0 &&
                 num_heads % num_kv_heads == 0 && head_size > 0 && block_size >= 16 &&
                 keep <= (INT_MAX >> 1) / (block_size / 16),
             "fk_sparse_paged_decode_plan: invalid argument");
  const int gqa = num_heads / num_kv_heads;
  const int vheads = num_kv_heads * ((gqa + 15) / 16);
  *workspace_bytes = part_bytes(rows, vheads, parts_of(rows, keep, vheads, block_size),
                                gqa < 16 ? gqa : 16, head_size);
  return FK_OK;
}
