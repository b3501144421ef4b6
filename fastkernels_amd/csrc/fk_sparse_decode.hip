// Decode attention over the pages selected for each query row and kv head.
//
//   out[t, hq] = sum_k softmax_k(scale q[t, hq] . K[k]) V[k]   over the keys k < vis(t) of the
//   pages block_indices[t, kv head of hq, :] of the row's sequence (entries outside the
//   table, or at pages that hold no visible key, are skipped; a page listed twice counts
//   twice).  Sinks join the denominator; a row without a visible key is zero.
//
// One work-group per (query row, kv head, block of 16 query heads): its waves share the list
// (fk_page_attn.h).
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
};

// Waves of a work-group.  At head size 256 the query, a step's K and V rows and O take more
// than the 256 registers that two waves a SIMD leave: one runs there, with as much in flight.
#ifndef XW
#define XW 4
#endif
#ifndef XEU
#define XEU 2
#endif
template <int D>
constexpr int waves_of() { return D == 256 ? 4 : XW; }

template <int D, bool kFp8>
__global__ __launch_bounds__((waves_of<D>() * 64))
__attribute__((amdgpu_waves_per_eu((D == 256 ? 1 : XEU)))) void sparse_decode_kernel(
    SparseParams P, const int32_t* __restrict__ bt, const int32_t* __restrict__ ctx,
    const int32_t* __restrict__ cu) {
  constexpr int kWaves = waves_of<D>();
  extern __shared__ __align__(16) float lds[];  // merge_lds_floats of the group's columns
  const PageAttnParams& A = P.A;
  const int t = blockIdx.y;
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
  stream_units(A, st, unit_at, P.keep << per_log2, wave, kWaves, P.unit_tiles_log2, 0,
               max(vis, 0), [&] { return Limits<1>{{span}, span, span}; }, kvh,
               __builtin_fabsf(s2), lane);
  merge_waves<kWaves>(st, lds, wave, lane, ncols,
                      [&](int j, int dim, const float4& o, float M, float L) {
                        write_quad(A, t, qbase + j, D, dim, o, M, L, vsc);
                      });
}

template <int D, bool kFp8>
void launch_t(const SparseParams& P, dim3 grid, hipStream_t s, const int32_t* bt,
              const int32_t* ctx, const int32_t* cu) {
  constexpr int kWaves = waves_of<D>();
  const int cols = P.A.gqa < 16 ? P.A.gqa : 16;
  hipLaunchKernelGGL((sparse_decode_kernel<D, kFp8>), grid, dim3(kWaves * 64),
                     (4 * merge_lds_floats<kWaves, D>(cols)), s, P, bt, ctx, cu);
}
template <int D>
void launch_d(bool fp8, const SparseParams& P, dim3 grid, hipStream_t s, const int32_t* bt,
              const int32_t* ctx, const int32_t* cu) {
  if (fp8)
    launch_t<D, true>(P, grid, s, bt, ctx, cu);
  else
    launch_t<D, false>(P, grid, s, bt, ctx, cu);
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
  const dim3 grid(static_cast<unsigned>(num_kv_heads * A.col_blocks),
                  static_cast<unsigned>(rows));
  const bool fp8 = kv_dtype == FK_DTYPE_FP8_E4M3FN;
  hipStream_t s = as_stream(stream);
  if (head_size == 64)
    launch_d<64>(fp8, P, grid, s, block_tables, cache_seqlens, cu_seqlens_q);
  else if (head_size == 128)
    launch_d<128>(fp8, P, grid, s, block_tables, cache_seqlens, cu_seqlens_q);
  else
    launch_d<256>(fp8, P, grid, s, block_tables, cache_seqlens, cu_seqlens_q);
  return check_launch(what);
}

extern "C" int fk_sparse_paged_decode_plan(int64_t rows, int64_t keep, int num_heads,
                                           int num_kv_heads, int head_size, int block_size,
                                           int64_t* workspace_bytes) {
  FK_REQUIRE(workspace_bytes, "fk_sparse_paged_decode_plan: null output pointer");
  *workspace_bytes = 0;
  return FK_OK;
}
