// Choosing which cache pages a query attends to: per-page key bounds kept beside the cache,
// each page's score for a query, and the pages with the best scores.
//
// Bounds.  For a page with keys k_0 .. k_{n-1} of one kv head, lo_d = min_i k_i[d] and
// hi_d = max_i k_i[d].  For any query q of the head's group and any key of the page
//   q . k <= sum_d max(q_d lo_d, q_d hi_d) = max(q, 0) . hi + min(q, 0) . lo,
// so the score of a page bounds every logit inside it, and takes two dot products that read
// 2 D elements instead of the page's block_size * D.  A page's score for a kv head is the
// largest over the query heads of its group, which share the pages they attend to (and so
// each K / V byte, as in decode).
//
// Bounds are elements of the cache's type: the least and greatest of values are values, so
// nothing is rounded.  A NaN key makes the page's bounds NaN, and its score NaN; NaN is taken
// as the highest score, so that such a page is attended to and shows.
#include <limits.h>

#include "fk_key_rows.h"
#include "fk_query_rows.h"

namespace fk {
namespace {

// NaN-propagating minimum and maximum.
__device__ __forceinline__ float min_nan(float a, float b) {
  return __builtin_elementwise_minimum(a, b);
}
__device__ __forceinline__ float max_nan(float a, float b) {
  return __builtin_elementwise_maximum(a, b);
}

// ---------------------------------------------------------------------------
// update_key_bounds
// ---------------------------------------------------------------------------
struct BoundsParams {
  uint8_t* bounds;
  const uint8_t* k_cache;
  int64_t bt_row_stride;
  int bt_width;
  int num_kv_heads;
  int block_size_log2;
  int64_t num_blocks;
};

// The elements of one 32-bit word (2 bf16 or 4 fp8) as floats, and back (exactly: the
// values are the type's own).
template <bool kFp8>
struct Elems {
  static constexpr int N = kFp8 ? 4 : 2;
  __device__ __forceinline__ static void unpack(uint32_t w, float (&f)[N]) {
    if constexpr (kFp8) {
      const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(w, false);
      const auto b = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
      f[0] = a[0];
      f[1] = a[1];
      f[2] = b[0];
      f[3] = b[1];
    } else {
      f[0] = __uint_as_float(w << 16);
      f[1] = __uint_as_float(w & 0xffff0000u);
    }
  }
  __device__ __forceinline__ static uint32_t pack(const float (&f)[N]) {
    if constexpr (kFp8) {
      const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
      return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], lo, true));
    } else {
      return lo_pair(f32_to_bf16(f[0]), f32_to_bf16(f[1]));
    }
  }
};

// One wave per (page, kv head): a row of D elements takes kCl lanes of 16 bytes, so an
// instruction reads 64 / kCl rows.  Rows past the last valid one read that one again, which
// changes no minimum or maximum.  The pages of sequence b are those of positions
// [len - n, len), each recomputed over all its positions < len: what is stored depends on
// the cache alone, not on earlier calls.
//
// Bound by memory, by latency where the pages are few: one token of 64 sequences takes 3.2 us
// (1.5 MB), four fp8 prompts of 1000 .. 8192 tokens in pages of 64 8.8 us (23 MB).
template <bool kFp8, int D>
__global__ __launch_bounds__(256) void key_bounds_kernel(
    BoundsParams P, const int32_t* __restrict__ bt, const int32_t* __restrict__ ctx,
    const int32_t* __restrict__ cu) {
  constexpr int kElt = kFp8 ? 1 : 2;
  constexpr int kCl = D * kElt / 16;
  constexpr int kRows = 64 / kCl;
  using E = Elems<kFp8>;
  const int b = blockIdx.y;
  const int h = blockIdx.z * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int len = ctx[b];
  const int n = cu ? cu[b + 1] - cu[b] : 1;
  if (h >= P.num_kv_heads || n <= 0 || len <= 0) return;
  const int j = (max(len - n, 0) >> P.block_size_log2) + static_cast<int>(blockIdx.x);
  const int64_t pos = static_cast<int64_t>(j) << P.block_size_log2;
  if (pos >= len || j >= P.bt_width) return;
  const int page = bt[b * P.bt_row_stride + j];
  if (page < 0 || page >= P.num_blocks) return;
  const int rows = min(len - static_cast<int>(pos), 1 << P.block_size_log2);
  const int lane = threadIdx.x & 63;
  const int c = lane % kCl, rr = lane / kCl;
  const int64_t row_bytes = static_cast<int64_t>(P.num_kv_heads) * D * kElt;
  const uint8_t* src = P.k_cache + (static_cast<int64_t>(page) << P.block_size_log2) * row_bytes +
                       static_cast<int64_t>(h) * D * kElt + 16 * c;
  float lo[4][E::N], hi[4][E::N];
#pragma unroll
  for (int w = 0; w < 4; ++w)
#pragma unroll
    for (int e = 0; e < E::N; ++e) {
      lo[w][e] = -kNegInf;
      hi[w][e] = kNegInf;
    }
  auto fold = [&](const uint4& a, const uint4& z) {
    const uint32_t wa[4] = {a.x, a.y, a.z, a.w}, wz[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      float fa[E::N], fz[E::N];
      E::unpack(wa[w], fa);
      E::unpack(wz[w], fz);
#pragma unroll
      for (int e = 0; e < E::N; ++e) {
        lo[w][e] = min_nan(lo[w][e], fa[e]);
        hi[w][e] = max_nan(hi[w][e], fz[e]);
      }
    }
  };
  for (int r0 = 0; r0 < rows; r0 += 4 * kRows) {
    uint4 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = ld16(src + min(r0 + i * kRows + rr, rows - 1) * row_bytes);
#pragma unroll
    for (int i = 0; i < 4; ++i) fold(x[i], x[i]);
  }
  uint4 a, z;
  auto packed = [&] {
    a = make_uint4(E::pack(lo[0]), E::pack(lo[1]), E::pack(lo[2]), E::pack(lo[3]));
    z = make_uint4(E::pack(hi[0]), E::pack(hi[1]), E::pack(hi[2]), E::pack(hi[3]));
  };
  packed();
#pragma unroll
  for (int off = kCl; off < 64; off <<= 1) {
    uint4 pa, pz;
    pa.x = __shfl_xor(a.x, off, 64);
    pa.y = __shfl_xor(a.y, off, 64);
    pa.z = __shfl_xor(a.z, off, 64);
    pa.w = __shfl_xor(a.w, off, 64);
    pz.x = __shfl_xor(z.x, off, 64);
    pz.y = __shfl_xor(z.y, off, 64);
    pz.z = __shfl_xor(z.z, off, 64);
    pz.w = __shfl_xor(z.w, off, 64);
    fold(pa, pz);
    packed();
  }
  if (rr == 0) {
    uint8_t* dst = P.bounds +
                   (static_cast<int64_t>(page) * P.num_kv_heads + h) * 2 * D * kElt + 16 * c;
    *reinterpret_cast<uint4*>(dst) = a;
    *reinterpret_cast<uint4*>(dst + D * kElt) = z;
  }
}

// ---------------------------------------------------------------------------
// block_scores
// ---------------------------------------------------------------------------
struct ScoreParams {
  float* scores;
  int64_t row_stride;   // floats between the query rows of scores
  int64_t head_stride;  // and between its kv heads
  int width;            // blocks per (row, head)
  const uint16_t* q;
  int64_t q_row_stride;
  const uint8_t* bounds;
  const float* k_scale;
  int64_t bt_row_stride;
  int bt_width;
  int64_t rows;      // rows of q and scores
  int token_chunks;  // groups of 16 / slots query rows per sequence
  int num_kv_heads;
  int gqa;
  int slots_log2;    // column slots per query row: gqa rounded up to a power of two, at most 16
  int block_size_log2;
  int64_t num_blocks;
  int tiles;         // 16-page tiles per wave, at most kScoreTiles
};

// One wave: 16 pages x 16 columns per MFMA tile.  The columns are 16 / slots query rows of
// one sequence times the query heads of kv head h (a group that is no power of two repeats
// its last head, groups above 16 take several passes over the loaded bounds); the rows of
// the A operand are the pages' bounds, lo then hi, the B operands min(q, 0) and max(q, 0).
//
// Bound by memory: 32 sequences of 16000 .. 131072 tokens in pages of 16 take 143 us (655 MB,
// 4.6 TB/s, in pieces of 4 KB); one sequence of 40000 5.4 us.  More waves a SIMD are slower
// there (four 158 us).
constexpr int kScoreWaves = 8;  // of a work-group, a kv head each: a page's bounds are read whole
constexpr int kScoreTiles = 4;  // of a wave at most (8: 152 us where 4 take 141)
template <bool kFp8, int D>
__global__ __launch_bounds__(kScoreWaves * 64) void block_scores_kernel(
    ScoreParams P, const int32_t* __restrict__ bt, const int32_t* __restrict__ ctx,
    const int32_t* __restrict__ cu) {
  constexpr int kElt = kFp8 ? 1 : 2;
  constexpr int kKc = D / 32;
  using K = KChunks<kFp8, D>;
  extern __shared__ __align__(16) uint8_t turn[];  // K::kBytes for each wave
  const int lane = threadIdx.x & 63;
  const int r = lane & 15, g = lane >> 4;
  const int h = blockIdx.z * (blockDim.x >> 6) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = blockIdx.y / P.token_chunks;
  const int chunk = blockIdx.y - b * P.token_chunks;
  if (h >= P.num_kv_heads) return;
  const int len = ctx[b];
  const int t0 = cu ? cu[b] : b;
  const int n = cu ? cu[b + 1] - t0 : 1;
  const int slots = 1 << P.slots_log2;
  const int first = chunk * (16 >> P.slots_log2);  // this tile's first row of the sequence
  if (first >= n || t0 < 0 || t0 + first >= P.rows) return;
  const int i = first + (r >> P.slots_log2);       // column r's row of the sequence
  const bool row_ok = i < n && t0 + i < P.rows;
  const int nblk = min(pages_of(min(len - n + i + 1, len), P.block_size_log2), P.width);
  const int most = min(min(pages_of(len, P.block_size_log2), P.bt_width), P.width);
  const float ks = kFp8 && P.k_scale ? P.k_scale[h] : 1.f;
  const int col_blocks = (P.gqa + 15) >> 4;
  const uint16_t* qrow = P.q + static_cast<int64_t>(t0 + (row_ok ? i : first)) * P.q_row_stride;
  bf16x8_t qn[kKc], qp[kKc];  // min(q, 0) and max(q, 0) of column r (of -q for a scale below 0)
  auto load_q = [&](int cb) {
    const int head = h * P.gqa + min(16 * cb + (r & (slots - 1)), P.gqa - 1);
    const uint16_t* p = qrow + static_cast<int64_t>(head) * D;
#pragma unroll
    for (int c = 0; c < kKc; ++c) {
      const int d0 = K::dims(c, g);
      const uint4 v = *reinterpret_cast<const uint4*>(p + d0);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
      uint32_t a[4], z[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t x = w[k] ^ (ks < 0.f ? 0x80008000u : 0u);
        // by sign (a NaN goes to one side, which is enough to reach the sum)
        const uint32_t neg = ((x >> 15) & 0x00010001u) * 0xffffu;
        a[k] = x & neg;
        z[k] = x & ~neg;
      }
      qn[c] = __builtin_bit_cast(bf16x8_t, make_uint4(a[0], a[1], a[2], a[3]));
      qp[c] = __builtin_bit_cast(bf16x8_t, make_uint4(z[0], z[1], z[2], z[3]));
    }
  };
  load_q(0);
  const int32_t* bt_row = bt + b * P.bt_row_stride;
  float* srow = P.scores + static_cast<int64_t>(t0 + i) * P.row_stride + h * P.head_stride;
  const int tile0 = blockIdx.x * P.tiles;
  const int tiles = min(P.tiles, (P.width + 15) / 16 - tile0);
  const int seen = min(tiles, (most - 16 * tile0 + 15) / 16);  // tiles with pages to read
  // Lane k holds the table's entry for the wave's page k.
  static_assert(kScoreTiles * 16 <= 64, "a lane per page");
  const int my_entry = 16 * tile0 + lane < most ? bt_row[16 * tile0 + lane] : -1;
  const bool entry_ok = my_entry >= 0 && my_entry < P.num_blocks;
  const uint64_t pages_ok = __ballot(entry_ok);
  const int my_page = entry_ok ? my_entry : 0;
  uint8_t* const kx = turn + (threadIdx.x >> 6) * K::kBytes;
  const uint8_t* const base =
      P.bounds + static_cast<int64_t>(h) * 2 * D * kElt + 16 * (lane % K::kPieces);
  const int64_t page_bytes = static_cast<int64_t>(P.num_kv_heads) * 2 * D * kElt;
  struct Bounds {
    DTile<kFp8, D> lo, hi;  // (k only)
  };
  // Issues tile x's loads (row r of a tile is page 16 x + r).
  auto load = [&](int x, Bounds& t) {
#pragma unroll
    for (int i = 0; i < K::kLoads; ++i) {
      const uint8_t* row =
          base + page_bytes * __shfl(my_page, 16 * x + K::kRows * i + lane / K::kPieces, 64);
      t.lo.k[i] = ld16(row);
      t.hi.k[i] = ld16(row + D * kElt);
    }
    loads_issued();
  };
  // Scores tile x from t, whose registers take the next tile as soon as they are free.
  auto score = [&](int x, Bounds& t) {
    const int j0 = 16 * (tile0 + x);
    float s[4] = {kNegInf, kNegInf, kNegInf, kNegInf};
    if (x < seen) {
      uint4 kl[kKc], kh[kKc];
      K::put(t.lo, kx, lane);
      K::get(kx, lane, kl);
      K::put(t.hi, kx, lane);
      K::get(kx, lane, kh);
      if (x + 1 < seen) load(x + 1, t);
      for (int cb = 0; cb < col_blocks; ++cb) {
        if (cb > 0 || (col_blocks > 1 && x > 0)) load_q(cb);
        const floatx4_t u = qk_scores_n(kl, qn), v = qk_scores_n(kh, qp);
#pragma unroll
        for (int k = 0; k < 4; ++k) s[k] = cb == 0 ? u[k] + v[k] : max_nan(s[k], u[k] + v[k]);
      }
      const uint32_t cur = static_cast<uint32_t>(pages_ok >> (16 * x));
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        for (int off = 1; off < slots; off <<= 1) s[k] = max_nan(s[k], __shfl_xor(s[k], off, 64));
        const int page = 4 * g + k;
        s[k] = (cur >> page & 1) && j0 + page < nblk ? s[k] * __builtin_fabsf(ks) : kNegInf;
      }
    }
    if (row_ok && (r & (slots - 1)) == 0) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (j0 + 4 * g + k < P.width) srow[j0 + 4 * g + k] = s[k];
    }
  };
  // (One tile ahead: with two or three, a call that reads the most, 32 sequences of 16000 ..
  // 131072 tokens, takes 157 and 168 us instead of 141.)
  Bounds t;
  if (seen > 0) load(0, t);
  for (int x = 0; x < tiles; ++x) score(x, t);
}

// ---------------------------------------------------------------------------
// select_blocks
// ---------------------------------------------------------------------------
struct SelectParams {
  int32_t* indices;
  int64_t out_row_stride, out_head_stride;
  const float* scores;
  int64_t row_stride, head_stride;
  int width;
  int keep, keep_first, keep_last;
  int block_size_log2;
  int batch;
};

constexpr int kSelThreads = 512;
constexpr int kSelBins = 2048;  // 11 bits of a key: four bins a thread
static_assert(kSelBins == 4 * kSelThreads, "four bins a thread");
// Keys held in LDS (one word in 17 is left free, so that threads reading runs of keys meet
// different banks); rows with more pages are read from memory in every pass.
constexpr int kSelLdsKeys = 32768;
__host__ __device__ constexpr int sel_at(int j) { return j + (j >> 4); }

// Scores in ascending order of an unsigned key: NaN above all, -0 equal to +0.
__device__ __forceinline__ uint32_t score_key(float s) {
  if (s != s) return 0xffffffffu;
  const uint32_t u = __float_as_uint(s + 0.f);
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

__device__ __forceinline__ float key_score(uint32_t key) {  // (of a number)
  return __uint_as_float(key ^ (key >> 31 ? 0x80000000u : 0xffffffffu));
}

// Inclusive scan over the lanes of a wave (0 is the operation's identity): within rows of 16,
// then across them.
template <int kCtrl, int kRows>
__device__ __forceinline__ int moved(int v) {
  return __builtin_amdgcn_update_dpp(0, v, kCtrl, kRows, 0xf, false);
}
template <class Op>
__device__ __forceinline__ uint32_t scan_lanes(uint32_t v, Op op) {
  v = op(v, moved<0x111, 0xf>(v));     // from the lane 1 before, 2, 4, 8
  v = op(v, moved<0x112, 0xf>(v));
  v = op(v, moved<0x114, 0xf>(v));
  v = op(v, moved<0x118, 0xf>(v));
  v = op(v, moved<0x142, 0xa>(v));     // from lane 15 of the row before, into rows 1 and 3
  return op(v, moved<0x143, 0xc>(v));  // from lane 31, into rows 2 and 3
}
// Inclusive sums over the work-group's threads.  part: a word per wave and value, not in use
// since the barrier before the last.
template <int kN>
__device__ __forceinline__ void scan_threads(int (&v)[kN], int (*part)[kSelThreads / 64],
                                             int tid) {
  constexpr int kWaves = kSelThreads / 64;
  const int lane = tid & 63, wave = tid >> 6;
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    v[i] = scan_lanes(v[i], [](uint32_t a, uint32_t b) { return a + b; });
    if (lane == 63) part[i][wave] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kN; ++i)
#pragma unroll
    for (int w = 0; w < kWaves; ++w) v[i] += w < wave ? part[i][w] : 0;
}

// One work-group per (query row, kv head), in search of the key T of the lowest selected
// candidate.  First the candidates' scores are counted in equal steps between the least and the
// greatest: where the step that holds the rank has few of them, the lanes of a wave rank those.
// Otherwise (equal scores, infinities, NaN, or more pages than LDS holds) T is found digit by
// digit (11, 11 and 10 bits: a histogram of the keys that agree with the digits found so far,
// then the bin that holds the rank), until the rank takes a whole bin.  The blocks are written in
// order of their index: each thread takes a run of them, counts what is selected there (the
// blocks always kept, keys above T, and the first of the keys equal to T), and its place is the
// sum of the counts before it.
//
// Bound by latency: loads, barriers and LDS atomics in turn.  One sequence of 40000 tokens in
// pages of 16 takes 7.4 us, 85 rows of 32 sequences of 16000 .. 131072 tokens 18.6 (by digits at
// once 8.1 and 20.1, and with 256 or 1024 threads a list 10.6 / 24.8 and 8.4 / 23.0).
template <bool kLds>
__global__ __launch_bounds__(kSelThreads) void select_blocks_kernel(
    SelectParams P, const int32_t* __restrict__ ctx, const int32_t* __restrict__ cu) {
  extern __shared__ __align__(16) uint32_t keys[];  // kLds: sel_at(width) words
  __shared__ int hist[kSelBins];
  __shared__ int part[2][kSelThreads / 64];
  __shared__ int found[3];
  __shared__ uint32_t range[2][kSelThreads / 64];
  __shared__ uint32_t few[64];
  __shared__ int few_count;
  const int t = blockIdx.x, h = blockIdx.y;
  int b, vis;
  if (!query_row(cu, ctx, P.batch, t, b, vis)) return;
  const int n = min(pages_of(vis, P.block_size_log2), P.width);
  int32_t* out = P.indices + t * P.out_row_stride + h * P.out_head_stride;
  const float* row = P.scores + t * P.row_stride + h * P.head_stride;
  const int tid = threadIdx.x;
  if (n <= P.keep) {
    for (int k = tid; k < P.keep; k += kSelThreads) out[k] = k < n ? k : -1;
    return;
  }
  auto key_of = [&](int j) { return kLds ? keys[sel_at(j)] : score_key(row[j]); };
#pragma unroll
  for (int i = 0; i < 4; ++i) hist[4 * tid + i] = 0;
  const int first = P.keep_first, last = n - P.keep_last;  // candidates [first, last)
  int need = P.keep - P.keep_first - P.keep_last;          // of which so many are selected
  if constexpr (kLds) {
    // (kAhead loads in flight; those past the end read the last score once more)
    constexpr int kAhead = 8;
    uint32_t top = 0, bottom = 0;  // the greatest key and complement of a key
    for (int j0 = tid; j0 < n; j0 += kAhead * kSelThreads) {
      float s[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) s[u] = row[min(j0 + u * kSelThreads, n - 1)];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int j = j0 + u * kSelThreads;
        if (j >= n) continue;
        const uint32_t key = score_key(s[u]);
        keys[sel_at(j)] = key;
        if (j < first || j >= last) continue;
        top = max(top, key);
        bottom = max(bottom, ~key);
      }
    }
    const auto larger = [](uint32_t a, uint32_t b) { return max(a, b); };
    top = scan_lanes(top, larger);
    bottom = scan_lanes(bottom, larger);
    if ((tid & 63) == 63) {
      range[0][tid >> 6] = top;
      range[1][tid >> 6] = bottom;
    }
    if (tid == 0) few_count = 0;
  }
  __syncthreads();
  uint32_t digits = 0, known = 0;  // T, and the bits of it that count
  // (With nothing to select among the candidates T stays above every key.)
  bool whole = need == 0;
  if (whole) digits = known = 0xffffffffu;
  int equal_need = 0;  // of the keys equal to T, the first so many are selected
  // From the counts in hist, the bin that holds rank `need` from the top: found = the bin, the
  // rank in it, its count.  Clears the bins.
  auto find_bin = [&] {
    __syncthreads();
    // Thread k sums bins 2047 - 4 k .. 2044 - 4 k: the inclusive sum counts from the top.
    int bins[4], sum[1] = {0};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      bins[i] = hist[kSelBins - 1 - 4 * tid - i];
      hist[kSelBins - 1 - 4 * tid - i] = 0;
      sum[0] += bins[i];
    }
    int above = -sum[0];
    scan_threads(sum, part, tid);
    above += sum[0];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (above < need && above + bins[i] >= need) {
        found[0] = kSelBins - 1 - 4 * tid - i;
        found[1] = need - above;
        found[2] = bins[i];
      }
      above += bins[i];
    }
    __syncthreads();
  };
  if constexpr (kLds) {
    uint32_t top = 0, bottom = 0;
#pragma unroll
    for (int w = 0; w < kSelThreads / 64; ++w) {
      top = max(top, range[0][w]);
      bottom = max(bottom, range[1][w]);
    }
    bottom = ~bottom;
    // (finite scores that differ, by a number whose inverse is finite too)
    const float low = key_score(bottom), width = key_score(top) - low;
    if (!whole && top < 0xff800000u && bottom > 0x007fffffu && width > 1.0e-30f &&
        width < 3.0e38f) {
      const float scale = static_cast<float>(kSelBins) / width;
      auto step_of = [&](uint32_t key) {  // (does not decrease with the key)
        return min(static_cast<int>((key_score(key) - low) * scale), kSelBins - 1);
      };
#pragma unroll 4
      for (int j = first + tid; j < last; j += kSelThreads) atomicAdd(&hist[step_of(key_of(j))], 1);
      find_bin();
      const int step = found[0], rank = found[1], count = found[2];
      if (count <= 64) {
#pragma unroll 4
        for (int j = first + tid; j < last; j += kSelThreads) {
          const uint32_t key = key_of(j);
          if (step_of(key) != step) continue;
          const int k = atomicAdd(&few_count, 1);
          if (k < 64) few[k] = key;
        }
        __syncthreads();
        // Every wave ranks them, a lane each.
        const int lane = tid & 63;
        const uint32_t mine = lane < count ? few[lane] : 0;
        int above = 0, equal = 0;
        for (int i = 0; i < count; ++i) {
          const uint32_t other = __builtin_amdgcn_readlane(mine, i);
          above += other > mine;
          equal += other == mine;
        }
        const int src = __builtin_ctzll(
            __ballot(lane < count && above < rank && rank <= above + equal));
        digits = __builtin_amdgcn_readlane(mine, src);
        known = 0xffffffffu;
        equal_need = rank - __builtin_amdgcn_readlane(above, src);
        whole = true;
      }
    }
  }
  for (int pass = 0; pass < 3 && !whole; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const uint32_t mask = pass == 2 ? 1023u : 2047u;
#pragma unroll 4
    for (int j = first + tid; j < last; j += kSelThreads) {
      const uint32_t key = key_of(j);
      if ((key & known) == digits) atomicAdd(&hist[(key >> shift) & mask], 1);
    }
    find_bin();
    digits |= static_cast<uint32_t>(found[0]) << shift;
    known |= mask << shift;
    need = found[1];
    whole = found[2] == need;  // every key of the bin is selected: the other digits do not matter
    equal_need = need;
  }
  if (P.keep == P.keep_first + P.keep_last) equal_need = 0;
  // Keys whose known digits exceed T's, and the first equal_need of those with T's.
  const int per = (n + kSelThreads - 1) / kSelThreads;
  const int j0 = min(n, tid * per), j1 = min(n, j0 + per);
  // (from LDS a run is 64 keys at most: what is selected of it is noted in bits, and the second
  // walk only meets those)
  uint64_t above_bits = 0, equal_bits = 0;
  int above = 0, equal = 0;
#pragma unroll 4
  for (int j = j0; j < j1; ++j) {
    const bool cand = j >= first && j < last;
    const uint32_t key = cand ? key_of(j) & known : 0;
    const bool up = !cand || key > digits, eq = cand && key == digits;
    above += up;
    equal += eq;
    if (kLds) {
      above_bits |= static_cast<uint64_t>(up) << (j - j0);
      equal_bits |= static_cast<uint64_t>(eq) << (j - j0);
    }
  }
  int before[2] = {above, equal};
  scan_threads(before, part, tid);
  const int equal_before = before[1] - equal;
  int left = min(max(equal_need - equal_before, 0), equal);
  int at = before[0] - above + min(equal_before, equal_need);
  if constexpr (kLds) {
    for (uint64_t bits = left > 0 ? above_bits | equal_bits : above_bits; bits; bits &= bits - 1) {
      const int k = __builtin_ctzll(bits);
      const bool eq = equal_bits >> k & 1;
      if (eq && left == 0) continue;
      left -= eq;
      if (at < P.keep) out[at] = j0 + k;
      ++at;
    }
  } else {
    for (int j = j0; j < j1; ++j) {
      const bool cand = j >= first && j < last;
      const uint32_t key = cand ? key_of(j) & known : 0;
      const bool eq = cand && key == digits;
      if (!cand || key > digits || (eq && left > 0)) {
        if (at < P.keep) out[at] = j;
        ++at;
        left -= eq;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Launch
// ---------------------------------------------------------------------------
// Work-groups of up to 512 threads along a grid's x: their threads number less than 2^32.
constexpr int64_t kMaxGridX = (int64_t{1} << 23) - 1;

bool head_built(int d) { return d == 64 || d == 128 || d == 256; }

int log2_of(int v) { return 31 - __builtin_clz(static_cast<unsigned>(v)); }

// The checks of the paged arguments the entry points here share.
int check_paged(const char* what, int kv_dtype, int64_t bt_row_stride, int64_t bt_width,
                int64_t batch, int num_kv_heads, int head_size, int block_size,
                int64_t num_blocks) {
  FK_REQUIRE(batch >= 0 && batch <= 65535, "%s: batch %lld outside [0, 65535]", what,
             static_cast<long long>(batch));
  FK_REQUIRE(num_kv_heads > 0 && num_kv_heads <= 4 * 65535, "%s: %d kv heads", what,
             num_kv_heads);
  FK_REQUIRE(kv_dtype == FK_DTYPE_BF16 || kv_dtype == FK_DTYPE_FP8_E4M3FN,
             "%s: the cache must be bf16 or fp8 e4m3fn", what);
  FK_REQUIRE(block_size >= 16 && (block_size & (block_size - 1)) == 0,
             "%s: block_size %d must be a power of two >= 16", what, block_size);
  FK_REQUIRE(num_blocks > 0 && num_blocks <= INT_MAX, "%s: num_blocks %lld", what,
             static_cast<long long>(num_blocks));
  FK_REQUIRE(bt_width >= 0 && bt_width <= kMaxGridX && bt_row_stride >= 0,
             "%s: block table of %lld columns", what, static_cast<long long>(bt_width));
  if (!head_built(head_size))
    return set_error(FK_ERR_UNSUPPORTED, "%s: head_size %d unsupported (64, 128 or 256)", what,
                     head_size);
  return FK_OK;
}

template <bool kFp8>
void launch_bounds(const BoundsParams& P, int d, dim3 grid, hipStream_t s, const int32_t* bt,
                   const int32_t* ctx, const int32_t* cu) {
  if (d == 64)
    hipLaunchKernelGGL((key_bounds_kernel<kFp8, 64>), grid, dim3(256), 0, s, P, bt, ctx, cu);
  else if (d == 128)
    hipLaunchKernelGGL((key_bounds_kernel<kFp8, 128>), grid, dim3(256), 0, s, P, bt, ctx, cu);
  else
    hipLaunchKernelGGL((key_bounds_kernel<kFp8, 256>), grid, dim3(256), 0, s, P, bt, ctx, cu);
}

template <bool kFp8>
void launch_scores(const ScoreParams& P, int d, dim3 grid, hipStream_t s, const int32_t* bt,
                   const int32_t* ctx, const int32_t* cu) {
  const int waves = P.num_kv_heads < kScoreWaves ? P.num_kv_heads : kScoreWaves;
  if (d == 64)
    hipLaunchKernelGGL((block_scores_kernel<kFp8, 64>), grid, dim3(64 * waves),
                       (waves * KChunks<kFp8, 64>::kBytes), s, P, bt, ctx, cu);
  else if (d == 128)
    hipLaunchKernelGGL((block_scores_kernel<kFp8, 128>), grid, dim3(64 * waves),
                       (waves * KChunks<kFp8, 128>::kBytes), s, P, bt, ctx, cu);
  else
    hipLaunchKernelGGL((block_scores_kernel<kFp8, 256>), grid, dim3(64 * waves),
                       (waves * KChunks<kFp8, 256>::kBytes), s, P, bt, ctx, cu);
}

}  // namespace
}  // namespace fk

using namespace fk;

extern "C" int fk_update_key_bounds(void* key_bounds, const void* k_cache, int kv_dtype,
                                    const int32_t* block_tables, int64_t bt_row_stride,
                                    int64_t bt_width, const int32_t* cache_seqlens,
                                    const int32_t* cu_seqlens_q, int64_t batch,
                                    int64_t max_seqlen_q, int num_kv_heads, int head_size,
                                    int block_size, int64_t num_blocks, void* stream) {
  const char* what = "fk_update_key_bounds";
  if (int rc = check_paged(what, kv_dtype, bt_row_stride, bt_width, batch, num_kv_heads,
                           head_size, block_size, num_blocks))
    return rc;
  FK_REQUIRE(max_seqlen_q >= 0 && max_seqlen_q <= INT_MAX, "%s: max_seqlen_q %lld", what,
             static_cast<long long>(max_seqlen_q));
  FK_REQUIRE(cu_seqlens_q || max_seqlen_q == 1,
             "%s: without cu_seqlens_q each sequence has one new token", what);
  if (batch == 0 || max_seqlen_q == 0 || bt_width == 0) return FK_OK;
  FK_REQUIRE(key_bounds && k_cache && block_tables && cache_seqlens, "%s: null pointer", what);
  FK_REQUIRE(aligned16(key_bounds) && aligned16(k_cache),
             "%s: key_bounds and k_cache must be 16-byte aligned", what);
  BoundsParams P;
  P.bounds = static_cast<uint8_t*>(key_bounds);
  P.k_cache = static_cast<const uint8_t*>(k_cache);
  P.bt_row_stride = bt_row_stride;
  P.bt_width = static_cast<int>(bt_width);
  P.num_kv_heads = num_kv_heads;
  P.block_size_log2 = log2_of(block_size);
  P.num_blocks = num_blocks;
  // Pages that n consecutive positions can touch.
  int64_t pages = (max_seqlen_q + block_size - 2) / block_size + 1;
  if (pages > bt_width) pages = bt_width;
  const dim3 grid(static_cast<unsigned>(pages), static_cast<unsigned>(batch),
                  static_cast<unsigned>((num_kv_heads + 3) / 4));
  if (kv_dtype == FK_DTYPE_FP8_E4M3FN)
    launch_bounds<true>(P, head_size, grid, as_stream(stream), block_tables, cache_seqlens,
                        cu_seqlens_q);
  else
    launch_bounds<false>(P, head_size, grid, as_stream(stream), block_tables, cache_seqlens,
                         cu_seqlens_q);
  return check_launch(what);
}

extern "C" int fk_block_scores(float* scores, int64_t score_row_stride, int64_t score_head_stride,
                               int64_t width, const void* q, int64_t q_row_stride,
                               const void* key_bounds, int kv_dtype, const float* k_scale,
                               const int32_t* block_tables, int64_t bt_row_stride,
                               int64_t bt_width, const int32_t* cache_seqlens,
                               const int32_t* cu_seqlens_q, int64_t batch, int64_t rows,
                               int64_t max_seqlen_q, int num_heads, int num_kv_heads, int head_size,
                               int block_size, int64_t num_blocks, void* stream) {
  const char* what = "fk_block_scores";
  if (int rc = check_paged(what, kv_dtype, bt_row_stride, bt_width, batch, num_kv_heads,
                           head_size, block_size, num_blocks))
    return rc;
  FK_REQUIRE(num_heads > 0 && num_heads % num_kv_heads == 0,
             "%s: %d query heads over %d kv heads", what, num_heads, num_kv_heads);
  FK_REQUIRE(max_seqlen_q >= 0 && max_seqlen_q <= INT_MAX, "%s: max_seqlen_q %lld", what,
             static_cast<long long>(max_seqlen_q));
  FK_REQUIRE(cu_seqlens_q || max_seqlen_q == 1,
             "%s: without cu_seqlens_q each sequence has one query row", what);
  FK_REQUIRE(width >= 0 && width <= kMaxGridX, "%s: %lld blocks per row", what,
             static_cast<long long>(width));
  FK_REQUIRE(rows >= 0 && rows <= INT_MAX && (cu_seqlens_q || rows >= batch),
             "%s: %lld query rows for %lld sequences", what, static_cast<long long>(rows),
             static_cast<long long>(batch));
  if (batch == 0 || rows == 0 || max_seqlen_q == 0 || width == 0) return FK_OK;
  FK_REQUIRE(scores && q && key_bounds && block_tables && cache_seqlens, "%s: null pointer", what);
  FK_REQUIRE(aligned16(q) && aligned16(key_bounds) && q_row_stride % 8 == 0,
             "%s: q rows and key_bounds must be 16-byte aligned", what);
  ScoreParams P;
  P.scores = scores;
  P.row_stride = score_row_stride;
  P.head_stride = score_head_stride;
  P.width = static_cast<int>(width);
  P.q = static_cast<const uint16_t*>(q);
  P.q_row_stride = q_row_stride;
  P.bounds = static_cast<const uint8_t*>(key_bounds);
  P.k_scale = k_scale;
  P.bt_row_stride = bt_row_stride;
  P.bt_width = static_cast<int>(bt_width);
  P.rows = rows;
  P.num_kv_heads = num_kv_heads;
  P.gqa = num_heads / num_kv_heads;
  P.slots_log2 = P.gqa >= 16 ? 4 : P.gqa == 1 ? 0 : log2_of(P.gqa - 1) + 1;
  P.block_size_log2 = log2_of(block_size);
  P.num_blocks = num_blocks;
  const int64_t tile_rows = 16 >> P.slots_log2;
  const int64_t chunks = (max_seqlen_q + tile_rows - 1) / tile_rows;
  FK_REQUIRE(chunks * batch <= 65535, "%s: %lld groups of query rows are more than 65535", what,
             static_cast<long long>(chunks * batch));
  P.token_chunks = static_cast<int>(chunks);
  // Tiles per wave: one where that leaves each SIMD under eight waves over the call, more (a
  // wave's next tile is on its way while it scores one) where there are plenty.
  const int64_t waves = (P.width + 15) / 16 * chunks * batch * num_kv_heads;
  const int64_t per = waves / (int64_t{num_cus()} * 32);
  P.tiles = static_cast<int>(per < 1 ? 1 : per > kScoreTiles ? kScoreTiles : per);
  const int wg_heads = num_kv_heads < kScoreWaves ? num_kv_heads : kScoreWaves;
  const dim3 grid(static_cast<unsigned>((P.width + 16 * P.tiles - 1) / (16 * P.tiles)),
                  static_cast<unsigned>(chunks * batch),
                  static_cast<unsigned>((num_kv_heads + wg_heads - 1) / wg_heads));
  if (kv_dtype == FK_DTYPE_FP8_E4M3FN)
    launch_scores<true>(P, head_size, grid, as_stream(stream), block_tables, cache_seqlens,
                        cu_seqlens_q);
  else
    launch_scores<false>(P, head_size, grid, as_stream(stream), block_tables, cache_seqlens,
                         cu_seqlens_q);
  return check_launch(what);
}

extern "C" int fk_select_blocks(int32_t* block_indices, int64_t out_row_stride,
                                int64_t out_head_stride, int64_t keep, const float* scores,
                                int64_t score_row_stride, int64_t score_head_stride,
                                int64_t width, const int32_t* cache_seqlens,
                                const int32_t* cu_seqlens_q, int64_t batch, int64_t rows,
                                int num_kv_heads, int block_size, int keep_first, int keep_last,
                                void* stream) {
  const char* what = "fk_select_blocks";
  FK_REQUIRE(batch >= 0 && batch <= INT_MAX && rows >= 0 && rows <= kMaxGridX,
             "%s: %lld rows of %lld sequences", what, static_cast<long long>(rows),
             static_cast<long long>(batch));
  FK_REQUIRE(num_kv_heads > 0 && num_kv_heads <= 65535, "%s: %d kv heads", what, num_kv_heads);
  FK_REQUIRE(block_size >= 1 && (block_size & (block_size - 1)) == 0,
             "%s: block_size %d must be a power of two", what, block_size);
  FK_REQUIRE(width >= 0 && width <= INT_MAX - kSelThreads && keep >= 0 && keep <= INT_MAX,
             "%s: %lld of %lld blocks", what, static_cast<long long>(keep),
             static_cast<long long>(width));
  FK_REQUIRE(keep_first >= 0 && keep_last >= 0 &&
                 static_cast<int64_t>(keep_first) + keep_last <= keep,
             "%s: keep_first %d and keep_last %d must fit in the %lld selected blocks", what,
             keep_first, keep_last, static_cast<long long>(keep));
  if (batch == 0 || rows == 0 || keep == 0) return FK_OK;
  FK_REQUIRE(block_indices && (scores || width == 0) && cache_seqlens, "%s: null pointer", what);
  SelectParams P;
  P.indices = block_indices;
  P.out_row_stride = out_row_stride;
  P.out_head_stride = out_head_stride;
  P.scores = scores;
  P.row_stride = score_row_stride;
  P.head_stride = score_head_stride;
  P.width = static_cast<int>(width);
  P.keep = static_cast<int>(keep);
  P.keep_first = keep_first;
  P.keep_last = keep_last;
  P.block_size_log2 = log2_of(block_size);
  P.batch = static_cast<int>(batch);
  const dim3 grid(static_cast<unsigned>(rows), static_cast<unsigned>(num_kv_heads));
  if (P.width <= kSelLdsKeys)
    hipLaunchKernelGGL(select_blocks_kernel<true>, grid, dim3(kSelThreads), 4 * sel_at(P.width),
                       as_stream(stream), P, cache_seqlens, cu_seqlens_q);
  else
    hipLaunchKernelGGL(select_blocks_kernel<false>, grid, dim3(kSelThreads), 0, as_stream(stream),
                       P, cache_seqlens, cu_seqlens_q);
  return check_launch(what);
}
