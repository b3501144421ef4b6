// Decode attention of a batch whose sequences come in groups that share a prefix.
//
// Rows cu_groups[g] .. cu_groups[g + 1] - 1 hold the same keys at positions below
// prefix_lens[g], which are read through the block table of the group's first row; every
// other key is read through the row's own table.  The result is that of paged decode: row b
// attends to its keys [lo, ctx_lens[b]), lo = 0 or ctx - 1 - window_left under a sliding
// window.  Rows outside every group share nothing.
#include <limits.h>

#include "fk_page_attn.h"

namespace fk {
namespace {

struct PrefixParams {
  PageAttnParams A;
  int num_groups;
  int window_left;
  int unit_tiles_log2;
};

// Group of row b (the last with cu_groups[g] <= b), or -1.
__device__ __forceinline__ int group_of(const int32_t* __restrict__ cu, int groups, int b) {
  if (groups <= 0 || b < cu[0] || b >= cu[groups]) return -1;
  int lo = 0, hi = groups;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= b) lo = mid; else hi = mid;
  }
  return lo;
}

template <int kG, int D, bool kFp8>
__global__ __launch_bounds__((page_attn_waves<kG, D>() * 64))
__attribute__((amdgpu_waves_per_eu(2))) void shared_prefix_kernel(
    PrefixParams P, const int32_t* __restrict__ bt, const int32_t* __restrict__ ctx_lens,
    const int32_t* __restrict__ cu_groups, const int32_t* __restrict__ prefix_lens) {
  constexpr int kWaves = page_attn_waves<kG, D>();
  constexpr int U = D == 64 ? 4 : D == 128 ? 2 : 1;
  __shared__ __align__(16) float lds[merge_lds_floats<kG, D>()];
  const PageAttnParams& A = P.A;
  const int b = blockIdx.y;
  const int kvh = blockIdx.x / A.col_blocks;
  const int qbase = kvh * A.gqa + 16 * (blockIdx.x - kvh * A.col_blocks);
  const int ncols = min(16, (kvh + 1) * A.gqa - qbase);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int r = lane & 15, g = lane >> 4;
  const int grp = group_of(cu_groups, P.num_groups, b);
  const int prefix = grp >= 0 ? prefix_lens[grp] : 0;
  const int64_t first_row = grp >= 0 ? max(cu_groups[grp], 0) : b;
  const int ctx = max(ctx_lens[b], 0);
  const int lo = P.window_left >= 0 ? max(0, ctx - 1 - P.window_left) : 0;
  ColumnState<kG, D, kFp8> st;
  st.init(A.q + b * A.q_row_stride + static_cast<int64_t>(qbase + r) * D, r < ncols, g);
  const float ks = kFp8 && A.k_scale ? A.k_scale[kvh] : 1.f;
  const float vsc = kFp8 && A.v_scale ? A.v_scale[kvh] : 1.f;
  const int tok_log2 = 4 + P.unit_tiles_log2;
  const int32_t* own = bt + b * A.bt_row_stride;
  const int32_t* shared = bt + first_row * A.bt_row_stride;
  // Two passes over the units: positions below the prefix through the group's table, the
  // others through the row's own (a unit across the border is masked in each).
  const int border = min(prefix > 0 ? prefix : 0, ctx);
  for (int pass = 0; pass < 2; ++pass) {
    const int from = max(lo, pass ? border : 0), to = pass ? ctx : border;
    if (from >= to) continue;
    const int u0 = from >> tok_log2;
    const int32_t* table = pass ? own : shared;
    auto unit_at = [&](int u, int& page, int& tok) {
      tok = (u0 + u) << tok_log2;
      const int j = tok >> A.block_size_log2;
      page = j < A.bt_width ? table[j] : -1;
    };
    stream_units<kG, D, kFp8, U>(A, st, unit_at, ((to - 1) >> tok_log2) + 1 - u0, wave, kWaves,
                                 P.unit_tiles_log2, from, to, kvh, ks, lane);
  }
  merge_waves(st, lds, wave, lane, ncols, [&](int j, int dim, float x, float y, float M, float L) {
    write_pair(A, b, qbase + j, D, dim, x, y, M, L, vsc);
  });
}

template <int kG, int D>
void launch_fp8(bool fp8, const PrefixParams& P, dim3 grid, hipStream_t s, const int32_t* bt,
                const int32_t* ctx, const int32_t* cu, const int32_t* pre) {
  const dim3 block(page_attn_waves<kG, D>() * 64);
  if (fp8)
    hipLaunchKernelGGL((shared_prefix_kernel<kG, D, true>), grid, block, 0, s, P, bt, ctx, cu,
                       pre);
  else
    hipLaunchKernelGGL((shared_prefix_kernel<kG, D, false>), grid, block, 0, s, P, bt, ctx, cu,
                       pre);
}
template <int D>
void launch_d(bool fp8, const PrefixParams& P, dim3 grid, hipStream_t s, const int32_t* bt,
              const int32_t* ctx, const int32_t* cu, const int32_t* pre) {
  if (P.A.gqa <= 4)
    launch_fp8<4, D>(fp8, P, grid, s, bt, ctx, cu, pre);
  else if (P.A.gqa <= 8)
    launch_fp8<8, D>(fp8, P, grid, s, bt, ctx, cu, pre);
  else
    launch_fp8<16, D>(fp8, P, grid, s, bt, ctx, cu, pre);
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
  FK_REQUIRE(num_groups >= 0 && num_groups <= INT_MAX, "%s: %lld groups", what,
             static_cast<long long>(num_groups));
  FK_REQUIRE(max_prefix_len >= 0, "%s: max_prefix_len %lld", what,
             static_cast<long long>(max_prefix_len));
  FK_REQUIRE(window_left >= -1, "%s: window_left %d must be -1 or >= 0", what, window_left);
  if (batch == 0) return FK_OK;
  FK_REQUIRE(out && q && k_cache && v_cache && block_tables && cache_seqlens &&
                 (num_groups == 0 || (cu_groups && prefix_lens)),
             "%s: null pointer", what);
  PrefixParams P{};
  P.A = A;
  P.num_groups = static_cast<int>(num_groups);
  P.window_left = window_left;
  P.unit_tiles_log2 = A.block_size_log2 - 4 < 2 ? A.block_size_log2 - 4 : 2;
  const dim3 grid(static_cast<unsigned>(num_kv_heads * A.col_blocks),
                  static_cast<unsigned>(batch));
  const bool fp8 = kv_dtype == FK_DTYPE_FP8_E4M3FN;
  hipStream_t s = as_stream(stream);
  if (head_size == 64)
    launch_d<64>(fp8, P, grid, s, block_tables, cache_seqlens, cu_groups, prefix_lens);
  else if (head_size == 128)
    launch_d<128>(fp8, P, grid, s, block_tables, cache_seqlens, cu_groups, prefix_lens);
  else
    launch_d<256>(fp8, P, grid, s, block_tables, cache_seqlens, cu_groups, prefix_lens);
  return check_launch(what);
}

extern "C" int fk_shared_prefix_decode_plan(int64_t batch, int64_t num_groups,
                                            int64_t max_prefix_len, int num_heads,
                                            int num_kv_heads, int head_size,
                                            int64_t* workspace_bytes) {
  FK_REQUIRE(workspace_bytes, "fk_shared_prefix_decode_plan: null output pointer");
  *workspace_bytes = 0;
  return FK_OK;
}
