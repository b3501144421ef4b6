// The 4-bit cache's (fk_mxfp4.h) store and its read-back as rows of bf16.
//
// Both are bound by memory: the store reads 2 D values of a token and kv head and writes
// D + D / 16 bytes, the read-back the reverse.  A thread takes 8 dims: 16 bytes of bf16, one word
// of codes.
#include "fk_mxfp4.h"
#include "fk_query_rows.h"

namespace fk {
namespace {

constexpr int kThreads = 256;

struct CacheParams {
  uint8_t* k_cache;
  uint8_t* v_cache;
  uint8_t* k_scales;
  uint8_t* v_scales;
  int num_kv_heads, head_size;
  int block_size_log2;
  int units;  // of 8 dims, of a token's K row
};

// Where the codes of dims `dim` .. `dim` + 7 of a token lie.
__device__ __forceinline__ uint8_t* k_codes(const CacheParams& P, int64_t head_page, int tok,
                                            int dim) {
  return P.k_cache + ((head_page << P.block_size_log2) + tok) * (P.head_size / 2) + dim / 2;
}
// V: the first of the codes; at head size 64 the second half of them is 4 sixteenths' bytes on.
__device__ __forceinline__ uint8_t* v_codes(const CacheParams& P, int64_t head_page, int tok,
                                            int dim) {
  const int D = P.head_size;
  const int64_t quad = ((head_page << P.block_size_log2) + (tok & ~3)) * (D / 2);
  return P.v_cache + quad + dim / (D / 16) * (D / 8) + (tok & 3) * (D / 32) + dim % (D / 16) / 2;
}
__device__ __forceinline__ int64_t scale_at(const CacheParams& P, int64_t head_page, int tok,
                                            int dim) {
  return ((head_page * (P.head_size / 32) + dim / 32) << P.block_size_log2) + tok;
}

template <typename T, bool kVec>
__device__ __forceinline__ void load8(const typename T::storage* p, float (&x)[8]) {
  using V = Vec16<T>;
  if constexpr (kVec) {
#pragma unroll
    for (int i = 0; i < 8 / V::N; ++i) {
      V v;
      v.raw = reinterpret_cast<const uint4*>(p)[i];
#pragma unroll
      for (int e = 0; e < V::N; ++e) x[V::N * i + e] = T::to_f32(v.e[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = T::to_f32(p[e]);
  }
}

// Four neighbouring lanes hold a block of 32 dims.
template <typename T, typename IdxT, bool kVec>
__global__ __launch_bounds__(kThreads) void store_mxfp4_kernel(
    CacheParams P, const typename T::storage* __restrict__ key, int64_t key_stride,
    const typename T::storage* __restrict__ value, int64_t value_stride,
    const IdxT* __restrict__ slots, int64_t num_slots, int64_t tokens) {
  const int64_t id = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t tok = id / (2 * P.units);
  if (tok >= tokens) return;  // (whole blocks of lanes: the units are a multiple of 4)
  const int u = static_cast<int>(id - tok * (2 * P.units));
  const bool is_v = u >= P.units;
  const int at = 8 * (is_v ? u - P.units : u);  // of the row
  float x[8];
  load8<T, kVec>(is_v ? value + tok * value_stride + at : key + tok * key_stride + at, x);
  const int64_t slot = slots[tok];
  float top = 0.f;
  bool bad = false;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    top = fmaxf(top, __builtin_fabsf(x[e]));
    bad |= x[e] != x[e];
  }
  if (bad) top = __builtin_huge_valf();
  top = fmaxf(top, __shfl_xor(top, 1, 64));
  top = fmaxf(top, __shfl_xor(top, 2, 64));
  if (slot < 0 || slot >= num_slots) return;
  const uint32_t e = block_scale(top);
  uint32_t codes = 0;
  if (e != 255) {
    // (a scale of 2^-127 has no exponent field of its own, and needs none: the conversion
    // takes the field 0 as that)
    const float scale = __uint_as_float(e << 23);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[0], x[1], scale, 0);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[2], x[3], scale, 1);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[4], x[5], scale, 2);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[6], x[7], scale, 3);
  }
  const int head = at / P.head_size, dim = at - head * P.head_size;
  const int in = static_cast<int>(slot & ((1 << P.block_size_log2) - 1));
  const int64_t hp = (slot >> P.block_size_log2) * P.num_kv_heads + head;
  if (!is_v) {
    *reinterpret_cast<uint32_t*>(k_codes(P, hp, in, dim)) = codes;
  } else if (P.head_size == 64) {
    *reinterpret_cast<uint16_t*>(v_codes(P, hp, in, dim)) = static_cast<uint16_t>(codes);
    *reinterpret_cast<uint16_t*>(v_codes(P, hp, in, dim + 4)) = static_cast<uint16_t>(codes >> 16);
  } else {
    *reinterpret_cast<uint32_t*>(v_codes(P, hp, in, dim)) = codes;
  }
  if (dim % 32 == 0)
    (is_v ? P.v_scales : P.k_scales)[scale_at(P, hp, in, dim)] = static_cast<uint8_t>(e);
}

// Rows of a work-group at most: their slots are looked up side by side.  Fewer where that leaves
// CUs idle (117 rows of 8 heads of 128: 3.5 us, 14.7 with 32 each).
constexpr int kGatherRows = 32;

// The rows of four tokens that lie side by side in the cache go together: a thread takes 8 dims of
// them, whose V codes and scales are then one load each.  50 thousand tokens of 8 heads of 128:
// 51 us, 5.1 TB/s, and 70 where no cache holds any of it (86 with a row at a time; 84 and 88 with
// stores through the caches).
__global__ __launch_bounds__(kThreads) void gather_mxfp4_kernel(
    CacheParams P, uint16_t* __restrict__ key, int64_t key_stride, uint16_t* __restrict__ value,
    int64_t value_stride, const int32_t* __restrict__ bt, int64_t bt_row_stride, int bt_width,
    int64_t num_blocks, const int32_t* __restrict__ cu, int batch, int rows, int rows_of_wg) {
  __shared__ int64_t slots[kGatherRows];
  __shared__ int first_row[kGatherRows + 1];  // of each group
  __shared__ int groups_of_wg;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * rows_of_wg;
  dense_slots(cu, batch, t0, rows_of_wg, rows, bt, bt_row_stride, bt_width, P.block_size_log2,
              num_blocks, slots);
  const int n = static_cast<int>(min(static_cast<int64_t>(rows_of_wg), rows - t0));
  // A row begins a group unless it is the next token of the row before and in the same four.
  bool begins = false;
  if (threadIdx.x < n) {
    const int64_t s = slots[threadIdx.x];
    begins = threadIdx.x == 0 || s < 0 || s % 4 == 0 || slots[threadIdx.x - 1] != s - 1;
  }
  const uint64_t all = __ballot(begins);  // (the first wave has all of them)
  if (threadIdx.x < 64) {
    const int before = __builtin_popcountll(all & ((uint64_t{1} << threadIdx.x) - 1));
    if (begins) first_row[before] = threadIdx.x;
    if (threadIdx.x == 0) {
      groups_of_wg = __builtin_popcountll(all);
      first_row[groups_of_wg] = n;
    }
  }
  __syncthreads();
  const int groups = groups_of_wg;
  // Short rows: several groups side by side.
  const int cols = 2 * P.units;
  const int per = cols < kThreads ? kThreads / cols : 1;
  const int group0 = cols < kThreads ? threadIdx.x / cols : 0;
  if (group0 >= per) return;
  for (int u = cols < kThreads ? threadIdx.x % cols : threadIdx.x; u < cols; u += kThreads) {
    const bool is_v = u >= P.units;
    const int at = 8 * (is_v ? u - P.units : u);
    const int head = at / P.head_size, dim = at - head * P.head_size;
    const uint8_t* const scales = is_v ? P.v_scales : P.k_scales;
    uint16_t* const out = (is_v ? value + t0 * value_stride : key + t0 * key_stride) + at;
    const int64_t stride = is_v ? value_stride : key_stride;
#pragma unroll 4
    for (int k = group0; k < groups; k += per) {
      const int row = first_row[k], end = first_row[k + 1];
      const int64_t slot = slots[row], from = max(slot, int64_t{0}) & ~int64_t{3};
      const int in = static_cast<int>(from & ((1 << P.block_size_log2) - 1));
      const int64_t hp = (from >> P.block_size_log2) * P.num_kv_heads + head;
      const uint32_t e = *reinterpret_cast<const uint32_t*>(scales + scale_at(P, hp, in, dim));
      const uint8_t* const p = is_v ? v_codes(P, hp, in, dim) : k_codes(P, hp, in, dim);
      uint32_t w[4];  // codes of the four tokens
      if (is_v && P.head_size != 256) {
        const uint4 x = *reinterpret_cast<const uint4*>(p);
        if (P.head_size == 128) {
          w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
        } else {  // the four tokens' first 4 dims, then the others
          w[0] = lo_pair(x.x, x.z), w[1] = hi_pair(x.x, x.z);
          w[2] = lo_pair(x.y, x.w), w[3] = hi_pair(x.y, x.w);
        }
      } else {
        const int apart = is_v ? 8 : P.head_size / 2;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = *reinterpret_cast<const uint32_t*>(p + i * apart);
      }
      const int first = slot < 0 ? 0 : static_cast<int>(slot & 3);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (i < first || row + i - first >= end || slot == -2) continue;
        uint4 x = fp4x8_to_bf16x8(w[i], __uint_as_float((e >> (8 * i) & 0xff) << 23));
        if (slot < 0) x = make_uint4(0, 0, 0, 0);
        store_past(out + (row + i - first) * stride, x);
      }
    }
  }
}

int fill(const char* what, CacheParams& P, void* k_cache, void* v_cache, void* k_scales,
         void* v_scales, int num_kv_heads, int head_size, int block_size, int64_t num_blocks) {
  FK_REQUIRE(num_kv_heads > 0 && num_kv_heads <= 65535, "%s: %d kv heads", what, num_kv_heads);
  FK_REQUIRE(block_size >= 16 && block_size <= (1 << 30) && (block_size & (block_size - 1)) == 0,
             "%s: block_size %d must be a power of two >= 16", what, block_size);
  FK_REQUIRE(num_blocks > 0 && num_blocks <= 0x7fffffff, "%s: num_blocks %lld", what,
             static_cast<long long>(num_blocks));
  if (head_size != 64 && head_size != 128 && head_size != 256)
    return set_error(FK_ERR_UNSUPPORTED, "%s: head_size %d unsupported (64, 128 or 256)", what,
                     head_size);
  FK_REQUIRE(aligned16(k_cache) && aligned16(v_cache) && aligned16(k_scales) &&
                 aligned16(v_scales),
             "%s: caches and scales must be 16-byte aligned", what);
  P.k_cache = static_cast<uint8_t*>(k_cache);
  P.v_cache = static_cast<uint8_t*>(v_cache);
  P.k_scales = static_cast<uint8_t*>(k_scales);
  P.v_scales = static_cast<uint8_t*>(v_scales);
  P.num_kv_heads = num_kv_heads;
  P.head_size = head_size;
  P.block_size_log2 = 31 - __builtin_clz(static_cast<unsigned>(block_size));
  P.units = num_kv_heads * head_size / 8;
  return FK_OK;
}

template <typename T>
void store(const CacheParams& P, const void* key, int64_t key_stride, const void* value,
           int64_t value_stride, const void* slots, bool i64, int64_t num_slots, int64_t tokens,
           hipStream_t s) {
  using S = typename T::storage;
  const bool vec = aligned16(key) && aligned16(value) && key_stride * sizeof(S) % 16 == 0 &&
                   value_stride * sizeof(S) % 16 == 0;
  const dim3 grid(static_cast<unsigned>((tokens * 2 * P.units + kThreads - 1) / kThreads));
  auto go = [&](auto kernel, auto* slot) {
    hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, s, P, static_cast<const S*>(key),
                       key_stride, static_cast<const S*>(value), value_stride, slot, num_slots,
                       tokens);
  };
  const auto* s64 = static_cast<const int64_t*>(slots);
  const auto* s32 = static_cast<const int32_t*>(slots);
  if (i64)
    vec ? go(store_mxfp4_kernel<T, int64_t, true>, s64)
        : go(store_mxfp4_kernel<T, int64_t, false>, s64);
  else
    vec ? go(store_mxfp4_kernel<T, int32_t, true>, s32)
        : go(store_mxfp4_kernel<T, int32_t, false>, s32);
}

}  // namespace
}  // namespace fk

using namespace fk;

extern "C" int fk_store_kvcache_mxfp4(const void* key, int64_t key_row_stride, const void* value,
                                      int64_t value_row_stride, int dtype, void* k_cache,
                                      void* v_cache, void* k_scales, void* v_scales,
                                      const void* slot_mapping, int slot_is_i64, int64_t tokens,
                                      int num_kv_heads, int head_size, int block_size,
                                      int64_t num_blocks, void* stream) {
  const char* what = "fk_store_kvcache_mxfp4";
  CacheParams P{};
  if (int rc = fill(what, P, k_cache, v_cache, k_scales, v_scales, num_kv_heads, head_size,
                    block_size, num_blocks))
    return rc;
  FK_REQUIRE(tokens >= 0 && tokens <= most_groups(kThreads) * kThreads / (2 * P.units),
             "%s: %lld tokens, more than a launch takes", what, static_cast<long long>(tokens));
  if (tokens == 0) return FK_OK;
  FK_REQUIRE(key && value && k_cache && v_cache && k_scales && v_scales && slot_mapping,
             "%s: null pointer", what);
  const int64_t num_slots = num_blocks * block_size;
  hipStream_t s = as_stream(stream);
  switch (dtype) {
    case FK_DTYPE_BF16:
      store<BF16>(P, key, key_row_stride, value, value_row_stride, slot_mapping, slot_is_i64,
                  num_slots, tokens, s);
      break;
    case FK_DTYPE_F16:
      store<F16>(P, key, key_row_stride, value, value_row_stride, slot_mapping, slot_is_i64,
                 num_slots, tokens, s);
      break;
    case FK_DTYPE_F32:
      store<F32>(P, key, key_row_stride, value, value_row_stride, slot_mapping, slot_is_i64,
                 num_slots, tokens, s);
      break;
    default:
      return set_error(FK_ERR_UNSUPPORTED, "%s: unsupported dtype %d", what, dtype);
  }
  return check_launch(what);
}

extern "C" int fk_gather_kvcache_mxfp4(void* key, int64_t key_row_stride, void* value,
                                       int64_t value_row_stride, const void* k_cache,
                                       const void* v_cache, const void* k_scales,
                                       const void* v_scales, const int32_t* block_tables,
                                       int64_t bt_row_stride, int64_t bt_width,
                                       const int32_t* cu_seqlens_k, int64_t batch, int64_t rows,
                                       int num_kv_heads, int head_size, int block_size,
                                       int64_t num_blocks, void* stream) {
  const char* what = "fk_gather_kvcache_mxfp4";
  CacheParams P{};
  if (int rc = fill(what, P, const_cast<void*>(k_cache), const_cast<void*>(v_cache),
                    const_cast<void*>(k_scales), const_cast<void*>(v_scales), num_kv_heads,
                    head_size, block_size, num_blocks))
    return rc;
  FK_REQUIRE(rows >= 0 && rows <= most_groups(kThreads) * kGatherRows && batch >= 0 &&
                 batch <= 0x7fffffff,
             "%s: %lld rows of %lld sequences", what, static_cast<long long>(rows),
             static_cast<long long>(batch));
  FK_REQUIRE(bt_width >= 0 && bt_width <= 0x7fffffff && bt_row_stride >= 0,
             "%s: block table of %lld columns", what, static_cast<long long>(bt_width));
  FK_REQUIRE(aligned16(key) && aligned16(value) && key_row_stride % 8 == 0 &&
                 value_row_stride % 8 == 0,
             "%s: key and value must have 16-byte aligned rows", what);
  if (rows == 0 || batch == 0) return FK_OK;
  FK_REQUIRE(key && value && k_cache && v_cache && k_scales && v_scales && block_tables &&
                 cu_seqlens_k,
             "%s: null pointer", what);
  const int per = dense_rows_of_wg(rows, kGatherRows);
  hipLaunchKernelGGL(gather_mxfp4_kernel, dim3(static_cast<unsigned>((rows + per - 1) / per)),
                     dim3(kThreads), 0, as_stream(stream), P, static_cast<uint16_t*>(key),
                     key_row_stride, static_cast<uint16_t*>(value), value_row_stride,
                     block_tables, bt_row_stride, static_cast<int>(bt_width), num_blocks,
                     cu_seqlens_k, static_cast<int>(batch), static_cast<int>(rows), per);
  return check_launch(what);
}
