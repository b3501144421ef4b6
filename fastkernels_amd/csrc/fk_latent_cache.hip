// The latent cache's store, with what precedes it, and its read-back as rows of bf16.
//
// A token's row is R = 512 values of the latent, normed over themselves, and the P = 64 values of
// the key's rotary part, which all heads share:
//   c = latent / sqrt(mean(latent^2) + eps) * weight,   row = [c | rotated key] (/ scale, fp8)
// and the queries' rotary parts are rotated by the same position's angles.  All of it is computed
// in fp32 and rounded once, to each of its destinations.
//
// Both are bound by memory.  A wave holds a latent (64 lanes of 8 values), or the rotary parts of
// eight heads; a work-group takes a token.  16 thousand tokens with 16 query heads into an fp8
// cache: 28 us, 3.4 TB/s.
#include "fk_attn_tile.h"
#include "fk_query_rows.h"

namespace fk {
namespace {

constexpr int kLatent = 512, kRope = 64;
constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
static_assert(kLatent == 64 * 8, "a latent is a wave's");

struct StoreParams {
  void* cache;
  const float* scale;
  const void* slots;
  int slot_is_i64;
  int64_t num_slots;
  const int64_t* positions;
  const uint16_t* latent;
  int64_t latent_stride;
  const uint16_t* key;
  int64_t key_stride;
  const uint16_t* weight;
  float eps;
  const void* cos_sin;
  int64_t max_position;
  const uint16_t* query;
  int64_t q_row_stride, q_head_stride;
  int num_heads;
  uint16_t* query_out;
  int64_t qo_row_stride, qo_head_stride;
  uint16_t* latent_out;
  int64_t lo_stride;
  uint16_t* key_out;
  int64_t ko_stride;
};

__device__ __forceinline__ void unpack8(const uint4& v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bf16x2_t p = {static_cast<__bf16>(x[2 * i]), static_cast<__bf16>(x[2 * i + 1])};
    w[i] = __builtin_bit_cast(uint32_t, p);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Values 8 i .. 8 i + 7 of a cache row.
template <bool kFp8>
__device__ __forceinline__ void store8(const StoreParams& P, int64_t slot, int dim,
                                       const float (&x)[8], float scale) {
  const int64_t at = slot * (kLatent + kRope) + dim;
  if constexpr (kFp8) {
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e)
      w[e >> 2] |= static_cast<uint32_t>(f32_to_e4m3fn_sat(x[e] / scale)) << (8 * (e & 3));
    *reinterpret_cast<uint2*>(static_cast<uint8_t*>(P.cache) + at) = make_uint2(w[0], w[1]);
  } else {
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(P.cache) + at) = pack8(x);
  }
}

template <typename CT, bool kNeox, bool kFp8>
__global__ __launch_bounds__(kThreads) void latent_store_kernel(StoreParams P) {
  const int64_t tok = blockIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int64_t slot = P.slot_is_i64 ? static_cast<const int64_t*>(P.slots)[tok]
                                     : static_cast<const int32_t*>(P.slots)[tok];
  const bool store = slot >= 0 && slot < P.num_slots;
  const float scale = kFp8 && P.scale ? *P.scale : 1.f;
  // Rotary parts: unit 0 is the key, unit 1 + h query head h; eight to a wave, a lane has eight
  // values of one.  The wave that takes the latent has one round of them less.
  const int units = 1 + P.num_heads;
  const int64_t pos = P.positions[tok];
  const bool rotate = pos >= 0 && pos < P.max_position;
  const int j = lane & 7;
  float c[8], s[8];
  if (rotate) {
    const typename CT::storage* const cs =
        static_cast<const typename CT::storage*>(P.cos_sin) + pos * kRope;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int i = kNeox ? (8 * j + e) % (kRope / 2) : 4 * j + e / 2;
      c[e] = CT::to_f32(cs[i]);
      s[e] = CT::to_f32(cs[kRope / 2 + i]);
    }
  }
  if (wave == kWaves - 1) {
    float x[8];
    unpack8(*reinterpret_cast<const uint4*>(P.latent + tok * P.latent_stride + 8 * lane), x);
    if (P.weight) {
      float w[8], ss = 0.f;
      unpack8(*reinterpret_cast<const uint4*>(P.weight + 8 * lane), w);
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = sumsq_add(ss, x[e]);
      const float inv = rms_inv(wave_sum(ss), kLatent, P.eps);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = x[e] * inv * w[e];
    }
    if (store) store8<kFp8>(P, slot, 8 * lane, x, scale);
    if (P.latent_out)
      *reinterpret_cast<uint4*>(P.latent_out + tok * P.lo_stride + 8 * lane) = pack8(x);
  }
  for (int u0 = 8 * wave; u0 < units; u0 += 8 * kWaves) {
    const int u = u0 + (lane >> 3);
    const bool ok = u < units;
    const int h = max(u - 1, 0);
    float x[8], y[8];
    const uint16_t* const from = u == 0 ? P.key + tok * P.key_stride
                                        : P.query + tok * P.q_row_stride + h * P.q_head_stride;
    unpack8(ok ? *reinterpret_cast<const uint4*>(from + 8 * j) : make_uint4(0, 0, 0, 0), x);
    if constexpr (kNeox) {
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = __shfl_xor(x[e], 4, 64);
      if (rotate) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          x[e] = j < 4 ? rope_x(x[e], y[e], c[e], s[e]) : rope_y(y[e], x[e], c[e], s[e]);
      }
    } else if (rotate) {
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const float a = x[e], b = x[e + 1];
        x[e] = rope_x(a, b, c[e], s[e]);
        x[e + 1] = rope_y(a, b, c[e], s[e]);
      }
    }
    if (!ok) continue;
    if (u == 0) {
      if (store) store8<kFp8>(P, slot, kLatent + 8 * j, x, scale);
      if (P.key_out) *reinterpret_cast<uint4*>(P.key_out + tok * P.ko_stride + 8 * j) = pack8(x);
    } else {
      *reinterpret_cast<uint4*>(P.query_out + tok * P.qo_row_stride + h * P.qo_head_stride +
                                8 * j) = pack8(x);
    }
  }
}

constexpr int kGatherRows = 32;  // of a work-group at most: their slots are looked up side by side

// 51 thousand rows from an fp8 cache: 15.8 us, 5.6 TB/s (17.9 with stores through the caches).
template <bool kFp8>
__global__ __launch_bounds__(kThreads) void latent_gather_kernel(
    uint16_t* __restrict__ out, int64_t out_stride, const uint8_t* __restrict__ cache,
    const float* __restrict__ scale, const int32_t* __restrict__ bt, int64_t bt_row_stride,
    int bt_width, const int32_t* __restrict__ cu, int batch, int rows, int block_size_log2,
    int64_t num_blocks, int rows_of_wg) {
  constexpr int kPieces = (kLatent + kRope) / 8;
  __shared__ int64_t from[kGatherRows];
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * rows_of_wg;
  dense_slots(cu, batch, t0, rows_of_wg, rows, bt, bt_row_stride, bt_width, block_size_log2, num_blocks, from);
  const float f = kFp8 && scale ? *scale : 1.f;
#pragma unroll 3
  for (int i = threadIdx.x; i < rows_of_wg * kPieces; i += kThreads) {
    const int row = i / kPieces, piece = i % kPieces;
    const int64_t at = from[row];
    if (at == -2) continue;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (at >= 0) {
      if constexpr (kFp8) {
        const uint2 x =
            *reinterpret_cast<const uint2*>(cache + at * (kLatent + kRope) + 8 * piece);
        const uint2 a = fp8x4_to_bf16x4(x.x), b = fp8x4_to_bf16x4(x.y);
        float y[8];
        unpack8(make_uint4(a.x, a.y, b.x, b.y), y);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] *= f;
        v = pack8(y);
      } else {
        v = *reinterpret_cast<const uint4*>(cache + 2 * (at * (kLatent + kRope) + 8 * piece));
      }
    }
    store_past(out + (t0 + row) * out_stride + 8 * piece, v);
  }
}

int check_cache(const char* what, int cache_dtype, const void* cache, const float* scale,
                int latent_size, int rope_size) {
  FK_REQUIRE(cache_dtype == FK_DTYPE_BF16 || cache_dtype == FK_DTYPE_FP8_E4M3FN,
             "%s: the cache must be bf16 or fp8 e4m3fn", what);
  FK_REQUIRE(!scale || cache_dtype == FK_DTYPE_FP8_E4M3FN, "%s: a bf16 cache has no scale", what);
  if (latent_size != kLatent || rope_size != kRope)
    return set_error(FK_ERR_UNSUPPORTED, "%s: rows of %d + %d unsupported (512 + 64)", what,
                     latent_size, rope_size);
  FK_REQUIRE(aligned16(cache), "%s: the cache must be 16-byte aligned", what);
  return FK_OK;
}

template <typename CT>
void store(const StoreParams& P, bool neox, bool fp8, int64_t tokens, hipStream_t s) {
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(tokens)), dim3(kThreads), 0, s, P);
  };
  if (neox)
    fp8 ? go(latent_store_kernel<CT, true, true>) : go(latent_store_kernel<CT, true, false>);
  else
    fp8 ? go(latent_store_kernel<CT, false, true>) : go(latent_store_kernel<CT, false, false>);
}

}  // namespace
}  // namespace fk

using namespace fk;

extern "C" int fk_latent_norm_rope_store(
    void* cache, int cache_dtype, const float* cache_scale, const void* slot_mapping,
    int slot_is_i64, int64_t num_slots, const int64_t* positions, const void* latent,
    int64_t latent_row_stride, const void* key_rope, int64_t key_row_stride, const void* weight,
    float eps, const void* cos_sin, int cos_sin_dtype, int64_t max_position, int is_neox,
    const void* query_rope, int64_t q_row_stride, int64_t q_head_stride, int num_heads,
    void* query_out, int64_t qo_row_stride, int64_t qo_head_stride, void* latent_out,
    int64_t latent_out_row_stride, void* key_out, int64_t key_out_row_stride, int64_t tokens,
    int latent_size, int rope_size, void* stream) {
  const char* what = "fk_latent_norm_rope_store";
  if (int rc = check_cache(what, cache_dtype, cache, cache_scale, latent_size, rope_size))
    return rc;
  FK_REQUIRE(tokens >= 0 && tokens <= most_groups(kThreads) && num_slots >= 0 && num_heads >= 0 &&
                 num_heads <= 65535 && max_position >= 0,
             "%s: %lld tokens, %lld slots, %d heads", what, static_cast<long long>(tokens),
             static_cast<long long>(num_slots), num_heads);
  FK_REQUIRE(aligned16(latent) && aligned16(key_rope) && aligned16(weight) &&
                 aligned16(query_rope) && aligned16(query_out) && aligned16(latent_out) &&
                 aligned16(key_out) &&
                 (latent_row_stride | key_row_stride | q_row_stride | q_head_stride |
                  qo_row_stride | qo_head_stride | latent_out_row_stride | key_out_row_stride) %
                         8 == 0,
             "%s: rows must be 16-byte aligned", what);
  FK_REQUIRE(cos_sin_dtype == FK_DTYPE_F32 || cos_sin_dtype == FK_DTYPE_BF16,
             "%s: cos_sin dtype %d must be f32 or bf16", what, cos_sin_dtype);
  if (tokens == 0) return FK_OK;
  FK_REQUIRE(cache && slot_mapping && positions && latent && key_rope && cos_sin &&
                 (num_heads == 0 || (query_rope && query_out)),
             "%s: null pointer", what);
  const StoreParams P{cache, cache_scale, slot_mapping, slot_is_i64 ? 1 : 0, num_slots, positions,
                      static_cast<const uint16_t*>(latent), latent_row_stride,
                      static_cast<const uint16_t*>(key_rope), key_row_stride,
                      static_cast<const uint16_t*>(weight), eps, cos_sin, max_position,
                      static_cast<const uint16_t*>(query_rope), q_row_stride, q_head_stride,
                      num_heads, static_cast<uint16_t*>(query_out), qo_row_stride, qo_head_stride,
                      static_cast<uint16_t*>(latent_out), latent_out_row_stride,
                      static_cast<uint16_t*>(key_out), key_out_row_stride};
  const bool fp8 = cache_dtype == FK_DTYPE_FP8_E4M3FN;
  if (cos_sin_dtype == FK_DTYPE_F32)
    store<F32>(P, is_neox != 0, fp8, tokens, as_stream(stream));
  else
    store<BF16>(P, is_neox != 0, fp8, tokens, as_stream(stream));
  return check_launch(what);
}

extern "C" int fk_gather_latent(void* out, int64_t out_row_stride, const void* cache,
                                int cache_dtype, const float* cache_scale,
                                const int32_t* block_tables, int64_t bt_row_stride,
                                int64_t bt_width, const int32_t* cu_seqlens_k, int64_t batch,
                                int64_t rows, int latent_size, int rope_size, int block_size,
                                int64_t num_blocks, void* stream) {
  const char* what = "fk_gather_latent";
  if (int rc = check_cache(what, cache_dtype, cache, cache_scale, latent_size, rope_size))
    return rc;
  FK_REQUIRE(block_size >= 16 && block_size <= (1 << 30) && (block_size & (block_size - 1)) == 0,
             "%s: block_size %d must be a power of two >= 16", what, block_size);
  FK_REQUIRE(num_blocks > 0 && num_blocks <= 0x7fffffff, "%s: num_blocks %lld", what,
             static_cast<long long>(num_blocks));
  FK_REQUIRE(rows >= 0 && rows <= most_groups(kThreads) * kGatherRows && batch >= 0 &&
                 batch <= 0x7fffffff,
             "%s: %lld rows of %lld sequences", what, static_cast<long long>(rows),
             static_cast<long long>(batch));
  FK_REQUIRE(bt_width >= 0 && bt_width <= 0x7fffffff && bt_row_stride >= 0,
             "%s: block table of %lld columns", what, static_cast<long long>(bt_width));
  FK_REQUIRE(aligned16(out) && out_row_stride % 8 == 0, "%s: out must have 16-byte aligned rows",
             what);
  if (rows == 0 || batch == 0) return FK_OK;
  FK_REQUIRE(out && cache && block_tables && cu_seqlens_k, "%s: null pointer", what);
  const int per = dense_rows_of_wg(rows, kGatherRows);
  const dim3 grid(static_cast<unsigned>((rows + per - 1) / per));
  const int log2 = 31 - __builtin_clz(static_cast<unsigned>(block_size));
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, as_stream(stream),
                       static_cast<uint16_t*>(out), out_row_stride,
                       static_cast<const uint8_t*>(cache), cache_scale, block_tables,
                       bt_row_stride, static_cast<int>(bt_width), cu_seqlens_k,
                       static_cast<int>(batch), static_cast<int>(rows), log2, num_blocks, per);
  };
  if (cache_dtype == FK_DTYPE_FP8_E4M3FN)
    go(latent_gather_kernel<true>);
  else
    go(latent_gather_kernel<false>);
  return check_launch(what);
}
