// Decode attention over a cache of latent rows, in the absorbed form: every query head attends
// to the same keys, a token's row of R + P values, and the values are its first R,
//   s[t, h, j] = scale q[t, h] . row_j,   out[t, h] = sum_j softmax_j(s) row_j[0 .. R).
//
// The heads of a query row are the columns of matrix products with the keys: S^T = K Q^T, then
// O^T += V^T P^T.  Keys come through LDS once: S reads them as rows, P V the same bytes with the
// transpose loads.  Items (query row, 32 or 64 heads) of 32-key steps lie on one line, cut into
// equal ranges (fk_lines.h); where a row has an even number of items, pairs of work-groups take
// the same range for one each, side by side on an XCD, so that the second finds the keys in the
// L2 (64 rows of 128 heads: 154 us, 170 without).  An item inside one range is finished there; of
// the others each part leaves a partial state, which a second launch merges.
//
// Measured (a call, captured): 64 rows of 128 heads over 512 .. 8192 tokens 127 us (645 TFLOP/s),
// of 16 heads 78 us (4.4 TB/s), of 16 heads over fp8 51 us; 128 rows of 16 heads over fp8 up to
// 16384 158 us (4.3 TB/s).  What bounds it: 1.3 us a step of 64 heads, where the products alone
// take 0.5 and LDS 0.6.  With all tiles in the L2 a step is no shorter, without S's products or
// those of P V neither: two tiles on their way (LDS holds no more) cover as much latency as the
// chain scores, maximum, weights, barrier takes.  Slower: eight waves, four of which do S and four
// P V (64 x 128: 170 us in place of 154); words of the lines loaded three steps ahead (175).  (The fp8
// kernel of one unit spills 40 bytes a lane, touched where the line is walked, not among the loads
// into LDS, whose waits it would make longer.)
#include "fk_lines.h"
#include "fk_page_attn.h"
#include "fk_query_rows.h"

#include <type_traits>

namespace fk {
namespace {

typedef float floatx16_t __attribute__((ext_vector_type(16)));

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * 64;
constexpr int kSeqs = 128;   // sequences looked at together
constexpr int kKeys = 32;    // of a tile
// What a part costs besides its steps, in steps: first tiles, queries, state.  (64 rows of 128
// heads: 166 us with 6, 156 with 10, 151 with 14, 154 with 20; others change by less.)
constexpr int kPad = 14;
// How far a part's logits may rise above those of its first 32 keys before it is taken in two, which
// is rare and costs a state written and read.
constexpr float kFar = 32.f;
// All weights, and with them the sums, carry this factor, so that none exceeds 2^8, as in the
// other decode kernels: n keys with values to 2^120 / n have finite sums.  (The first keys' are
// about 2^-24: bf16 and the fp32 sums hold them as exactly, and products of values down to
// 2^-102 with them are normal numbers.)
constexpr float kUnit = 0x1p-24f;

struct LatentParams {
  uint16_t* out;
  int64_t out_row_stride, out_head_stride;
  const uint16_t* q;
  int64_t q_row_stride, q_head_stride;
  const uint8_t* cache;
  const float* cache_scale;
  float* lse;
  int64_t lse_head_stride;
  float scale_log2;
  int num_heads;
  int head_blocks;  // units of 32 heads of a row
  int units;        // of an item
  int team;         // work-groups that take the same keys side by side, an item each
  int batch, rows, most;
  int block_size_log2;
  int64_t num_blocks;
  int64_t bt_row_stride;
  int bt_width;
  int wgs;
  float* o;         // [2 wgs][32 units][R]
  float* ml;        // [2 wgs][32 units] (maximum, sum)
  LineRecord* records;
};

// A tile in LDS: rows of bf16 or of fp8 codes.  A wave loads eight of them.
template <int R, int P, bool kFp8>
struct Tile {
  static constexpr int kRow = (R + P) * (kFp8 ? 1 : 2);  // bytes
  static constexpr int kPieces = kRow / 16;
  static constexpr int kBytes = kKeys * kRow;
  static constexpr int kWide = kRow / 128;           // loads of 64 pieces, of eight rows
  static constexpr int kLoads = kWide + kRow % 128 / 32;  // ... and of 64 words
  static_assert(kRow % 32 == 0, "whole loads");
  // Bytes of dims 32 k on: of the four pieces (bf16) or the two (fp8).  The pieces of row t are
  // permuted: in runs of 8 by (t / 2) mod 8, or fp8, two by two, by (t / 4) mod 2; so 16 rows that
  // are read together meet no bank twice.
  static __device__ __forceinline__ int at(int row, int piece) {
    return row * kRow + 16 * (kFp8 ? piece ^ (row >> 1 & 2)
                                   : (piece & ~7) | ((piece ^ (row >> 1)) & 7));
  }
  // Where in its eight rows of the cache a lane finds what load m takes to LDS (rows from a
  // multiple of 8 on, `odd`: not of 16).
  static __device__ __forceinline__ uint32_t source(int m, int lane, bool odd) {
    const int byte = m < kWide ? 1024 * m + 16 * lane : 1024 * kWide + 256 * (m - kWide) + 4 * lane;
    const int row = byte / kRow, in = byte % kRow;
    return at(row + (odd ? 8 : 0), in >> 4) - (odd ? 8 * kRow : 0) + (in & 15);
  }
};

// 16 bytes from global memory straight into LDS: lane l of the wave writes at byte lds_addr + 16 l
// what it reads at base + off.  The compiler does not see it as a load: the kernel waits for it.
// (The scalar move covers the wait states that the load's base needs after a vector instruction
// wrote it, and the one after the write of M0.)
__device__ __forceinline__ void lds_load16(const uint8_t* base, uint32_t off, uint32_t lds_addr) {
  const uint8_t* b;
  asm volatile(
      "s_mov_b64 %0, %2\n\t"
      "global_load_lds_dwordx4 %1, %0"
      : "=&s"(b)
      : "v"(off), "s"(base), "{m0}"(lds_addr)
      : "memory");
}
// ... and 4 bytes, at 4 l.
__device__ __forceinline__ void lds_load4(const uint8_t* base, uint32_t off, uint32_t lds_addr) {
  const uint8_t* b;
  asm volatile(
      "s_mov_b64 %0, %2\n\t"
      "global_load_lds_dword %1, %0"
      : "=&s"(b)
      : "v"(off), "s"(base), "{m0}"(lds_addr)
      : "memory");
}
__device__ __forceinline__ uint32_t lds_addr_of(const void* p) {
  return static_cast<uint32_t>(
      reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const uint8_t*)p));
}
// s_waitcnt's operand for vmcnt(0) alone (vmcnt in bits 3:0 and 15:14).
constexpr int kNoLoads = 0x0f70;
// Waits until at most kLeft of the wave's loads are on their way.
template <int kLeft>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kLeft) : "memory");
}
__device__ __forceinline__ short4_t transposed(const uint8_t* p) {
  typedef __attribute__((address_space(3))) short4_t* lds_short4;
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4)p);
}
// (fp8: eight keys of a dim)
__device__ __forceinline__ uint2 transposed8(const uint8_t* p) {
  typedef int int2_t __attribute__((ext_vector_type(2)));
  typedef __attribute__((address_space(3))) int2_t* lds_int2;
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_int2)p));
}
__device__ __forceinline__ uint4 joined(short4_t a, short4_t b) {
  const uint2 x = __builtin_bit_cast(uint2, a), y = __builtin_bit_cast(uint2, b);
  return make_uint4(x.x, x.y, y.x, y.y);
}
// Eight values as a product's operand (of fp8 codes exactly).
__device__ __forceinline__ bf16x8_t operand(const uint4& x) {
  return __builtin_bit_cast(bf16x8_t, x);
}
__device__ __forceinline__ bf16x8_t operand(const uint2& x) {
  const uint2 a = fp8x4_to_bf16x4(x.x), b = fp8x4_to_bf16x4(x.y);
  return __builtin_bit_cast(bf16x8_t, make_uint4(a.x, a.y, b.x, b.y));
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const bf16x2_t x = {static_cast<__bf16>(a), static_cast<__bf16>(b)};
  return __builtin_bit_cast(uint32_t, x);
}
// The keys of a part of an item, half a tile (16) at a time.
struct Halves {
  const uint8_t* cache;
  int64_t row_bytes;
  const int32_t* table;
  int bt_width, block_size_log2;
  int64_t num_blocks;
  // Page of the half that begins at key (a multiple of 16), -1: nothing to see.
  __device__ __forceinline__ int page(int64_t key, int to) const {
    if (key >= to) return -1;
    const int64_t j = key >> block_size_log2;
    const int p = j < bt_width ? table[j] : -1;
    return p < num_blocks ? p : -1;
  }
  __device__ __forceinline__ const uint8_t* rows(int page, int key) const {
    const int64_t row = (static_cast<int64_t>(max(page, 0)) << block_size_log2) +
                        (key & ((1 << block_size_log2) - 1));
    return cache + row * row_bytes;
  }
};

// A sequence's items: teams of `units` units of 32 heads of a row each, in steps of a tile.
__device__ __forceinline__ LineItems line_items(const LatentParams& P, const SeqRows& s,
                                                int units) {
  LineItems x;
  int none;
  x.from = 0;
  row_keys(s, s.rows - 1, -1, none, x.to);
  // (past the table's end there is nothing to see)
  x.to = static_cast<int>(min(min(static_cast<int64_t>(x.to), int64_t{0x7fffff00}),
                              static_cast<int64_t>(P.bt_width) << P.block_size_log2));
  x.steps = x.to > 0 ? (x.to - 1) / kKeys + 1 : 1;
  x.items = s.rows * ((P.head_blocks + units - 1) / units / P.team);
  return x;
}

// Output of four dims of a finished column, and with dim == 0 its log-sum-exp.
__device__ __forceinline__ void write_out(const LatentParams& P, int64_t row, int head, int dim,
                                          const float4& o, float M, float L, float vsc) {
  // (1 / L may be 1 / kUnit, and a great scale times that no float.)
  const float unit = __builtin_fabsf(vsc) > 1.f ? kUnit : 1.f;
  const float f = L > 0.f ? vsc * unit / L : 0.f, g = 1.f / unit;
  *reinterpret_cast<uint2*>(P.out + row * P.out_row_stride + head * P.out_head_stride + dim) =
      make_uint2(pack2(o.x * f * g, o.y * f * g), pack2(o.z * f * g, o.w * f * g));
  if (dim == 0 && P.lse)
    P.lse[head * P.lse_head_stride + row] =
        L > 0.f ? (M + __builtin_amdgcn_logf(L * (1.f / kUnit))) * 0.6931471805599453f
                : L == 0.f ? kNegInf : L;
}

// One work-group: items of kUnits units of 32 heads of a query row, in steps of a tile.
//
// The waves share S by columns and keys, wave w = (cs, ts): half cs of the columns and keys
// 16 ts .. 16 ts + 15 (16x16x32 products), and P V by dims: wave w has dims w R / 4 .. of every
// column (32x32x16 products), so that V is read from LDS once and K twice.  P goes through LDS,
// and so do the columns' maxima.
//
// A step has one barrier.  Behind it come S of the next step and P V of this one, with the next
// step's softmax among the products of the latter.
//
// A column's weights are kUnit 2^(logit - m), m the maximum of the first step: bf16 and the fp32
// sums hold great weights as exactly as small ones, and O is not rescaled.  Where a later maximum, which
// all waves know behind the next barrier, is 2^kFar times that, the part is taken in two: the state
// so far goes to memory, and what follows begins again with its own maximum and is merged with it.
constexpr int kBuffers = 4;  // tiles in LDS, of which two are on their way
constexpr int kAhead = kBuffers - 1;
// Bytes of the tiles, whose place the outputs take at the end.
template <int R, int P, bool kFp8>
constexpr int tiles_bytes(int units) {
  const int tiles = kBuffers * Tile<R, P, kFp8>::kBytes, out = 32 * units * (R + 4) * 4;
  return tiles > out ? tiles : out;
}
// Work-groups on a CU: a tile of codes is small enough for two.
constexpr int wgs_per_cu(int units, bool fp8) { return units == 1 && fp8 ? 2 : 1; }
template <int R, int P, int kUnits, bool kFp8>
__global__ __launch_bounds__(kThreads)
__attribute__((amdgpu_waves_per_eu(wgs_per_cu(kUnits, kFp8), wgs_per_cu(kUnits, kFp8)))) void
latent_decode_kernel(
    LatentParams A, const int32_t* __restrict__ bt, const int32_t* __restrict__ ctx_lens,
    const int32_t* __restrict__ cu) {
  using T = Tile<R, P, kFp8>;
  using Raw = std::conditional_t<kFp8, uint2, uint4>;  // eight values in LDS
  constexpr int kCols = 32 * kUnits;
  constexpr int kCB = kUnits;            // blocks of 16 columns of a wave's S
  constexpr int kKc = (R + P) / 32;      // products of S
  constexpr int kOb = R / 4 / 32;        // blocks of 32 dims of a wave
  constexpr int kGroup = 3;              // K operands read from LDS at a time
  constexpr int kLoads = T::kLoads;
  static_assert(kKc % kGroup == 0 && kOb % 2 == 0, "whole groups");
  __shared__ LineLds<kThreads, kSeqs> line;
  extern __shared__ __align__(16) uint8_t lds[];
  uint8_t* const p_lds = lds + tiles_bytes<R, P, kFp8>(kUnits);  // of two steps, [columns][32 keys] bf16
  constexpr int kP = kCols * kKeys * 2;
  // [two steps][2 halves of the keys][columns]
  float* const tops = reinterpret_cast<float*>(p_lds + 2 * kP);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int r = lane & 15, g = lane >> 4;   // S
  const int n = lane & 31, kh = lane >> 5;  // P V
  const int ts = wave & 1, cs = wave >> 1;
  const float vsc = kFp8 && A.cache_scale ? *A.cache_scale : 1.f;
  const float s2 = A.scale_log2 * vsc;
  const float abs_s2 = __builtin_fabsf(s2);
  const uint32_t flip = s2 < 0.f ? 0x80008000u : 0u;
  uint32_t src[kLoads];
#pragma unroll
  for (int m = 0; m < kLoads; ++m) src[m] = T::source(m, lane, wave & 1);
  const uint32_t lds0 = lds_addr_of(lds);
  // 16 bytes (8 keys) of a column's weights, their pieces permuted against bank conflicts.
  auto p_at = [&](int col, int key) {
    return p_lds + col * 64 + 16 * (((key >> 3) ^ (col >> 2)) & 3) + 2 * (key & 7);
  };

  // One go at the steps [s_lo, s_hi) of a part: returns where it stopped, s_hi or where the maxima
  // ask for other references.  Its state goes to slot `to`, or for -1 to the output, if it got to the
  // end, otherwise to `spare` (`to` itself if that is a slot); `more`: merged with the one there.
  auto attempt = [&](int b, const SeqRows& sr, const LineItems& x, int it, int s_lo, int s_hi,
                     int64_t to, int64_t spare, bool more) -> int {
    // kUnits blocks of 32 heads of one query row, which sees keys [0, hi).
    const int items = (A.head_blocks + kUnits - 1) / kUnits;  // of a row
    const int row = it / items, head0 = 32 * kUnits * (it - row * items);
    int none, hi;
    row_keys(sr, row, -1, none, hi);
    hi = uniform(hi);
    const int s_col = 16 * kCB * cs + r;  // first of S's columns
    floatx16_t o[kUnits][kOb];  // dims 32 d + i % 4 + 8 (i / 4) + 4 kh of column n of unit u
#pragma unroll
    for (int u = 0; u < kUnits; ++u)
#pragma unroll
      for (int d = 0; d < kOb; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[u][d][i] = 0.f;
    // The reference maxima of S's columns, of O's, this lane's share of S's columns' sums, and of
    // that the last step's.
    float ms[kCB], mo[kUnits], l[kCB], last[kCB];
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      ms[u] = mo[u] = kNoMax;
      l[u] = last[u] = 0.f;
    }

    const Halves keys{A.cache, (R + P) * (kFp8 ? 1 : 2), bt + b * A.bt_row_stride, A.bt_width,
                      A.block_size_log2, A.num_blocks};
    const int steps = s_hi - s_lo;
    // The pages of 32 steps' halves, a lane each; and which of them, and of the 32 steps before,
    // there are.
    int pages = -1, looked_up = -1;
    uint64_t there = 0, there_before = 0;
    auto known = [&](int s) { return min(s, steps - 1) / 32 == looked_up; };
    auto look_up = [&](int s) {  // before the loads of step s
      if (known(s)) return;
      looked_up = min(s, steps - 1) / 32;
      pages = keys.page((static_cast<int64_t>(s_lo) + 32 * looked_up) * kKeys + 16 * lane, x.to);
      there_before = there;
      there = __ballot(pages >= 0);
    };
    // Keys that the row sees of eight rows of step s, from its key `at` on.
    auto seen = [&](int s, int at) -> int {
      const uint64_t t = s / 32 == looked_up ? there : there_before;
      return t >> (2 * (s & 31) + (at >> 4)) & 1 ? hi - ((s_lo + s) * kKeys + at) : 0;
    };
    // This wave's loads of step s (past the end, once more of the last: as many are on their way):
    // where from, and where to.
    struct Moves {
      const uint8_t* from;
      uint32_t to;
    };
    auto moves_of = [&](int s) {
      const int t = min(s, steps - 1);
      const int key = (s_lo + t) * kKeys + 8 * wave;
      const int pg = __builtin_amdgcn_readlane(pages, 2 * (t & 31) + (wave >> 1));
      return Moves{keys.rows(pg, key),
                   lds0 + s % kBuffers * T::kBytes + wave * (T::kBytes / 4)};
    };
    auto issue = [&](const Moves& m, int i) {
      if (i < T::kWide)
        lds_load16(m.from, src[i], m.to + 1024 * i);
      else
        lds_load4(m.from, src[i], m.to + 1024 * T::kWide + 256 * (i - T::kWide));
    };
    auto load = [&](int s) {
      const Moves m = moves_of(s);
#pragma unroll
      for (int i = 0; i < kLoads; ++i) issue(m, i);
    };
    // Keys that the row does not see may hold anything, infinities and NaN among it, which a zero
    // weight would not undo: their rows become zeros, among this wave's rows of step s.
    auto clear = [&](int s) {
      const int n = seen(s, 8 * wave);
      if (n >= 8) return;
      uint8_t* const at = lds + s % kBuffers * T::kBytes + wave * (T::kBytes / 4) + 16 * lane;
#pragma unroll
      for (int i = 0; i < (8 * T::kPieces + 63) / 64; ++i)
        if (64 * i + lane >= max(n, 0) * T::kPieces && 64 * i + lane < 8 * T::kPieces)
          *reinterpret_cast<uint4*>(at + 1024 * i) = make_uint4(0, 0, 0, 0);
    };
    // The first steps' loads, and the queries behind them.
    look_up(0);
    load(0);
    load(1);
    bf16x8_t qb[kCB][kKc];
#pragma unroll
    for (int cb = 0; cb < kCB; ++cb) {
      const int h = head0 + s_col + 16 * cb;
      const bool ok = h < A.num_heads;
      const uint16_t* const qp =
          A.q + (sr.row0 + row) * A.q_row_stride + (ok ? h : 0) * A.q_head_stride + 8 * g;
#pragma unroll
      for (int k = 0; k < kKc; ++k) {
        uint4 v = ok ? *reinterpret_cast<const uint4*>(qp + 32 * k) : make_uint4(0, 0, 0, 0);
        v = make_uint4(v.x ^ flip, v.y ^ flip, v.z ^ flip, v.w ^ flip);
        qb[cb][k] = __builtin_bit_cast(bf16x8_t, v);
      }
    }
    // S of step s, in logits.  Operands come in groups, one ahead of the products.  Dims 32 k + 8 g
    // of a row: of their place, k / 2 moves it by two runs, k % 2 by a permutation.
    constexpr int kRun = kFp8 ? 32 : 64;  // bytes of 32 dims
    uint32_t k_at[2];
#pragma unroll
    for (int k = 0; k < 2; ++k)
      k_at[k] = T::at(16 * ts + r, kFp8 ? 2 * k + (g >> 1) : 4 * k + g) + (kFp8 ? 8 * (g & 1) : 0);
    // (among(x): what to do among the products of the x-th group)
    auto scores = [&](int s, floatx4_t (&p)[kCB], auto among) {
      const uint8_t* const tile = lds + (s % kBuffers) * T::kBytes;
      const uint8_t* const at[2] = {tile + k_at[0], tile + k_at[1]};
      Raw kx[2][kGroup];
#pragma unroll
      for (int j = 0; j < kGroup; ++j)
        kx[0][j] = *reinterpret_cast<const Raw*>(at[j & 1] + 2 * kRun * (j >> 1));
      // (two chains of products at least: one alone would wait for each result)
      constexpr int kChains = kCB == 1 ? 2 : 1;
      floatx4_t x[kChains][kCB];
#pragma unroll
      for (int c = 0; c < kChains; ++c)
#pragma unroll
        for (int cb = 0; cb < kCB; ++cb) x[c][cb] = floatx4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k0 = 0; k0 < kKc; k0 += kGroup) {
        const int now = k0 / kGroup & 1;
        if (k0 + kGroup < kKc) {
#pragma unroll
          for (int j = 0; j < kGroup; ++j)
            kx[now ^ 1][j] = *reinterpret_cast<const Raw*>(
                at[(k0 + kGroup + j) & 1] + 2 * kRun * ((k0 + kGroup + j) >> 1));
        }
        among(k0 / kGroup);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < kGroup; ++j)
#pragma unroll
          for (int cb = 0; cb < kCB; ++cb)
            x[j % kChains][cb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                operand(kx[now][j]), qb[cb][k0 + j], x[j % kChains][cb], 0, 0, 0);
      }
#pragma unroll
      for (int cb = 0; cb < kCB; ++cb)
        p[cb] = kChains == 1 ? x[0][cb] : x[0][cb] + x[kChains - 1][cb];
    };
    // The softmax of step s, in four parts: logits, their maxima, weights.
    // (The weights are rounded to bf16 for P V, 2^-8 relative at most, of either sign; their sum
    // is of the unrounded ones.)
    auto logits = [&](int s, floatx4_t (&p)[kCB]) {
      // (without a branch, which would part the products around it)
      const int n = seen(s, 16 * ts) - 4 * g;
#pragma unroll
      for (int cb = 0; cb < kCB; ++cb)
#pragma unroll
        for (int i = 0; i < 4; ++i) p[cb][i] = i < n ? p[cb][i] * abs_s2 : kNegInf;
    };
    auto maxima = [&](int s, const floatx4_t (&p)[kCB]) {
#pragma unroll
      for (int cb = 0; cb < kCB; ++cb) {
        const float top =
            pair_max(fmaxf(fmaxf(p[cb][0], p[cb][1]), fmaxf(p[cb][2], p[cb][3])));
        tops[(s & 1) * 2 * kCols + kCols * ts + s_col + 16 * cb] = top;
      }
    };
    auto weights = [&](int s, const floatx4_t (&p)[kCB], int cb) {
      float e[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) e[i] = kUnit * __builtin_amdgcn_exp2f(p[cb][i] - ms[cb]);
      last[cb] = (e[0] + e[1]) + (e[2] + e[3]);
      *reinterpret_cast<uint2*>(p_at(s_col + 16 * cb, 16 * ts + 4 * g) + (s & 1) * kP) =
          make_uint2(pack2(e[0], e[1]), pack2(e[2], e[3]));
    };
    // Whether a maximum is too far above its reference (uniform: every wave has the same ones).
    auto too_far = [&](const float (&t)[kUnits]) {
      bool far = false;
#pragma unroll
      for (int u = 0; u < kUnits; ++u) far |= t[u] > mo[u] + kFar;
      return __ballot(far) != 0;
    };
    auto count = [&] {
#pragma unroll
      for (int cb = 0; cb < kCB; ++cb) l[cb] += last[cb];
    };
    // O += P V of step s.  Operands of 16 keys (k): lane (n, kh) has keys 16 k + 8 kh .. + 7.  In
    // a transpose load of bf16, lane 4 a + q of each 16 addresses key a (of four) and dims 4 q on;
    // of fp8, lane 2 a + q key a (of eight) and dims 8 q on.  Block d's place in a row moves by
    // two runs with d / 2 and by a permutation with d % 2.
    uint32_t v_at[kFp8 ? 1 : 2][2];
#pragma unroll
    for (int h = 0; h < (kFp8 ? 1 : 2); ++h)
#pragma unroll
      for (int d = 0; d < 2; ++d)
        v_at[h][d] =
            kFp8 ? 8 * (lane & 1) + T::at(8 * kh + (r >> 1), wave * (R / 64) + 2 * d + (g & 1))
                 : 8 * (lane & 1) + T::at(8 * kh + 4 * h + (r >> 2),
                                          wave * (R / 32) + 4 * d + 2 * (g & 1) + ((lane & 3) >> 1));
    const uint8_t* const p_from = p_at(n, 8 * kh);  // keys 16 on: pieces 2 on, of four, permuted
    const int p_next = 32 - 64 * (((kh ^ (n >> 2)) & 3) >> 1);
    auto v_raw = [&](const uint8_t* tile, int x) -> Raw {  // keys 16 (x / kOb) on, block x % kOb
      const int k = x / kOb, d = x % kOb;
      const uint8_t* const at = tile + 16 * k * T::kRow + 2 * kRun * (d >> 1);
      if constexpr (kFp8)
        return transposed8(at + v_at[0][d & 1]);
      else
        return joined(transposed(at + v_at[0][d & 1]), transposed(at + v_at[1][d & 1]));
    };
    // The first operands of P V of step s: its weights, and V's of the first group.
    constexpr int kVGroup = kOb / 2;
    struct First {
      bf16x8_t w[2][kUnits];
      Raw v[kVGroup];
    };
    auto first_operands = [&](int s, First& f) {
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int u = 0; u < kUnits; ++u)
          f.w[k][u] = __builtin_bit_cast(
              bf16x8_t, *reinterpret_cast<const uint4*>(p_from + (s & 1) * kP + 64 * 32 * u +
                                                        k * p_next));
#pragma unroll
      for (int j = 0; j < kVGroup; ++j)
        f.v[j] = v_raw(lds + (s % kBuffers) * T::kBytes, j);
    };
    // (among(x): what to do among the products of the x-th quarter)
    auto values = [&](int s, const First& f, auto among) {
      const uint8_t* const tile = lds + (s % kBuffers) * T::kBytes;
      Raw v[2][kVGroup];
#pragma unroll
      for (int j = 0; j < kVGroup; ++j) v[0][j] = f.v[j];
#pragma unroll
      for (int x0 = 0; x0 < 2 * kOb; x0 += kVGroup) {
        const int now = x0 / kVGroup & 1;
        if (x0 + kVGroup < 2 * kOb) {
#pragma unroll
          for (int j = 0; j < kVGroup; ++j) v[now ^ 1][j] = v_raw(tile, x0 + kVGroup + j);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < kVGroup; ++j) {
          const int k = (x0 + j) / kOb, d = (x0 + j) % kOb;
#pragma unroll
          for (int u = 0; u < kUnits; ++u)
            o[u][d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(operand(v[now][j]), f.w[k][u],
                                                              o[u][d], 0, 0, 0);
        }
        among(x0 / kVGroup);
      }
    };

    // A step's barrier: step s's weights and maxima and step s + 1's tile are in LDS, and step
    // s - 1 is done with.  The loads of step s + 3 are issued among its products, so that the
    // waves do not wait for their addresses to be taken.
    auto enter = [&](int s, float (&t)[kUnits]) {
      wait_loads<kLoads>();
      clear(s + 1);
      __syncthreads();
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        const float* const top = tops + (s & 1) * 2 * kCols + 32 * u + n;
        t[u] = fmaxf(top[0], top[kCols]);
      }
    };
    const auto nothing = [](int) {};
    float t[kUnits];
    First f;
    __builtin_amdgcn_s_waitcnt(kNoLoads);
    clear(0);
    load(2);
    __syncthreads();
    floatx4_t p[kCB];
    scores(0, p, nothing);
    logits(0, p);
    maxima(0, p);
    __syncthreads();
    // The references.
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int c = s_col + 16 * u;
      mo[u] = fmaxf(kNoMax, fmaxf(tops[32 * u + n], tops[kCols + 32 * u + n]));
      ms[u] = fmaxf(kNoMax, fmaxf(tops[c], tops[kCols + c]));
      weights(0, p, u);
    }
    enter(0, t);
    int s = 0;
#pragma unroll 1
    while (s + 1 < steps && !too_far(t)) {  // (step s has been entered)
      look_up(s + kAhead);
      Moves m = moves_of(s + kAhead);
      // (The wait, which the compiler knows of, as it does not of the loads into LDS: with a load
      // of its own unfinished here it would wait for it in the loop, and with it for those.)
      __builtin_amdgcn_s_waitcnt(kNoLoads);
#pragma unroll 1
      do {
        constexpr int kGroups = kKc / kGroup;
        scores(s + 1, p, [&](int x) {
          if (x < kLoads) issue(m, x);
          if (x == kGroups - 1) first_operands(s, f);
        });
        if (too_far(t)) break;  // (looked at behind the products that do not depend on it)
        count();
        values(s, f, [&](int x) {
          if (x == 0) logits(s + 1, p);
          if (x == 1) maxima(s + 1, p);
          if (x >= 2 && x - 2 < kCB) weights(s + 1, p, x - 2);
          if (x < kLoads - kGroups) issue(m, kGroups + x);
          if (x == 3) m = moves_of(s + 1 + kAhead);
        });
        static_assert(kLoads - kGroups <= 3, "all of them once");
        ++s;
        enter(s, t);
      } while (s + 1 < steps && known(s + kAhead));
    }
    if (!too_far(t)) {
      count();
      first_operands(s, f);
      values(s, f, nothing);
      ++s;
    }
    wait_loads<0>();
    __syncthreads();

    // The states, through LDS: the columns' sums, of both waves and all lanes that have keys of
    // theirs, and O, which leaves in whole rows.
    constexpr int kRow = R + 4;  // floats
    float* const xo = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int cb = 0; cb < kCB; ++cb) tops[kCols * ts + s_col + 16 * cb] = pair_sum(l[cb]);
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      if (wave == 0) tops[2 * kCols + 32 * u + n] = mo[u];
      float* const at = xo + (32 * u + n) * kRow + wave * (R / 4) + 4 * kh;
#pragma unroll
      for (int d = 0; d < kOb; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<float4*>(at + 32 * d + 8 * i) = make_float4(
              o[u][d][4 * i], o[u][d][4 * i + 1], o[u][d][4 * i + 2], o[u][d][4 * i + 3]);
    }
    __syncthreads();
    const bool last_go = s == steps;
    const int64_t slot = last_go ? to : spare;
#pragma unroll 4
    for (int i = threadIdx.x; i < kCols * (R / 4); i += kThreads) {
      const int c = i / (R / 4), dim = 4 * (i % (R / 4));
      const int head = head0 + c;
      if (head >= A.num_heads) continue;
      Folded f;
      f.o = *reinterpret_cast<const float4*>(xo + c * kRow + dim);
      f.L = tops[c] + tops[kCols + c];
      f.M = tops[2 * kCols + c];
      if (more) {
        const float2 y = *reinterpret_cast<const float2*>(A.ml + (spare * kCols + c) * 2);
        f.add(y.x, y.y, *reinterpret_cast<const float4*>(A.o + (spare * kCols + c) * R + dim));
      }
      if (slot < 0) {
        write_out(A, sr.row0 + row, head, dim, f.o, f.M, f.L, vsc);
      } else {
        *reinterpret_cast<float4*>(A.o + (slot * kCols + c) * R + dim) = f.o;
      }
    }
    __syncthreads();  // (the state before has been read)
    if (slot >= 0 && threadIdx.x < kCols) {
      const int c = threadIdx.x;
      Folded f;
      f.reset();
      f.L = tops[c] + tops[kCols + c];
      f.M = tops[2 * kCols + c];
      float2* const ml = reinterpret_cast<float2*>(A.ml + (slot * kCols + c) * 2);
      if (more) f.add(ml->x, ml->y, f.o);
      *ml = make_float2(f.M, f.L);
    }
    __syncthreads();
    return s_lo + s;
  };
  // The work-groups of a team are neighbours on an XCD, and read each tile at about the same time.
  int team = blockIdx.x / A.team, member = blockIdx.x % A.team;
  if (A.wgs % (8 * A.team) == 0) {
    const int i = blockIdx.x >> 3;
    team = i / A.team * 8 + (blockIdx.x & 7);
    member = i % A.team;
  }
  const int teams = A.wgs / A.team;
  if (blockIdx.x >= teams * A.team) {
    if (blockIdx.x < A.wgs) return;
    team = teams;  // (writes the records)
  }
  auto body = [&](int b, const SeqRows& sr, const LineItems& x, int it, int s_lo, int s_hi,
                  int64_t slot, int64_t free_slot) {
    const int64_t to = slot >= 0 ? slot * A.team + member : -1;
    const int64_t spare = slot >= 0 ? to : free_slot * A.team + member;
    bool more = false;
    while (s_lo < s_hi) {
      s_lo = attempt(b, sr, x, it * A.team + member, s_lo, s_hi, to, spare, more);
      more = true;
    }
  };
  walk_line(line, A.batch, teams, team, 1, kPad, A.records,
            [&](int b) { return seq_rows(cu, ctx_lens, b, A.rows, A.most); },
            [&](const SeqRows& s) { return line_items(A, s, kUnits); }, body);
}

// One work-group per (query row, some of its heads, kDims of their dims): merges the pieces of an
// item that ranges cut.
template <int R, int kDims, int kAhead>
__global__ __launch_bounds__(kMergeThreads) void latent_merge_kernel(
    LatentParams A, const int32_t* __restrict__ ctx_lens, const int32_t* __restrict__ cu,
    int heads, int fp8) {
  __shared__ Folded folded[kMergeThreads];
  const int t = blockIdx.y, dim0 = blockIdx.z * kDims;
  int b, vis;
  if (!query_row(cu, ctx_lens, A.batch, t, b, vis)) return;
  const SeqRows s = seq_rows(cu, ctx_lens, b, A.rows, A.most);
  const int i = t - s.row0;
  if (i < 0 || i >= s.rows) return;
  const LineRecord rec = A.records[b];
  const float vsc = fp8 && A.cache_scale ? *A.cache_scale : 1.f;
  const int h0 = blockIdx.x * heads, h1 = min(h0 + heads, A.num_heads);
  // Item by item of the row.
  for (int h = h0; h < h1;) {
    const int per = 32 * A.units, block = h / per;
    const int in = h - block * per, nc = min(h1, (block + 1) * per) - h;
    const int item = i * ((A.head_blocks + A.units - 1) / A.units) + block;
    const LinePieces pieces(rec, item / A.team, kPad);
    if (pieces.n > 1) {
      merge_pieces<kDims, kAhead>(
          0, nc, folded, [&](int) { return pieces.n; },
          [&](int k, int x, const float*& ml, const float*& o) {
            const int64_t at = (pieces.slot(k) * A.team + item % A.team) * per + in + x;
            ml = A.ml + 2 * at;
            o = A.o + at * R + dim0;
          },
          [&](int x, int dim, const float4& o, float M, float L) {
            write_out(A, t, h + x, dim0 + dim, o, M, L, vsc);
          });
      __syncthreads();
    }
    h += nc;
  }
}

struct LatentPlan {
  int wgs, units;  // work-groups at most, units of an item
  int64_t o, ml, records, bytes;
};
LatentPlan plan_of(int64_t batch, int64_t max_seqlen_q, int num_heads, int latent_size) {
  LatentPlan p{};
  p.units = num_heads > 32 ? 2 : 1;
  p.wgs = num_cus() * wgs_per_cu(p.units, true);
  auto take = [&](int64_t bytes) {
    const int64_t at = p.bytes;
    p.bytes += (bytes + 255) / 256 * 256;
    return at;
  };
  p.o = take(int64_t{2} * p.wgs * 32 * p.units * latent_size * 4);
  p.ml = take(int64_t{2} * p.wgs * 32 * p.units * 8);
  p.records = take(batch * static_cast<int64_t>(sizeof(LineRecord)));
  return p;
}

template <int R, int P, bool kFp8>
void launch(const LatentParams& A, hipStream_t s, const int32_t* bt, const int32_t* ctx,
            const int32_t* cu) {
  const unsigned lds =
      tiles_bytes<R, P, kFp8>(A.units) + 2 * 32 * A.units * (kKeys * 2 + 2 * 4);
  if (A.units == 1)
    hipLaunchKernelGGL((latent_decode_kernel<R, P, 1, kFp8>), dim3(A.wgs + 1), dim3(kThreads),
                       lds, s, A, bt, ctx, cu);
  else
    hipLaunchKernelGGL((latent_decode_kernel<R, P, 2, kFp8>), dim3(A.wgs + 1), dim3(kThreads),
                       lds, s, A, bt, ctx, cu);
  // Where rows and heads do not make two work-groups a CU, the dims are dealt out too, and with
  // them threads to share a column's pieces; where they make so few that a thread would take more
  // than two rounds of columns, so that its loads overlap others' (64 rows of 128 heads: 13 us, 17
  // with whole rows; 128 rows of 16 heads 8 us with whole rows, 10 otherwise).  An item is rarely
  // in more than four pieces then, and loads for eight of them cost 22 us in place of 17.
  const int heads = merge_cols(A.rows, 1, A.num_heads);
  const dim3 grid((A.num_heads + heads - 1) / heads, A.rows);
  auto merge = [&](auto kernel, int dims) {
    hipLaunchKernelGGL(kernel, dim3(grid.x, grid.y, R / dims), dim3(kMergeThreads), 0, s, A, ctx,
                       cu, heads, kFp8 ? 1 : 0);
  };
  if (static_cast<int64_t>(grid.x) * grid.y < num_cus())
    merge(latent_merge_kernel<R, 64, 8>, 64);
  else if (heads * (R / 4) > 2 * kMergeThreads)
    merge(latent_merge_kernel<R, 128, 4>, 128);
  else
    merge(latent_merge_kernel<R, R, 4>, R);
}

}  // namespace
}  // namespace fk

using namespace fk;

extern "C" int fk_latent_decode(void* out, int64_t out_row_stride, int64_t out_head_stride,
                                const void* q, int64_t q_row_stride, int64_t q_head_stride,
                                const void* cache, int cache_dtype, const float* cache_scale,
                                const int32_t* block_tables, int64_t bt_row_stride,
                                int64_t bt_width, const int32_t* cache_seqlens,
                                const int32_t* cu_seqlens_q, int64_t batch, int64_t rows,
                                int64_t max_seqlen_q, int num_heads, int latent_size,
                                int rope_size, int block_size, int64_t num_blocks, float scale,
                                float* lse, int64_t lse_head_stride, void* workspace,
                                int64_t workspace_bytes, void* stream) {
  const char* what = "fk_latent_decode";
  FK_REQUIRE(batch >= 0 && batch <= 65535 && rows >= 0 && rows <= 65535,
             "%s: batch %lld or rows %lld outside [0, 65535]", what, static_cast<long long>(batch),
             static_cast<long long>(rows));
  FK_REQUIRE(num_heads > 0 && num_heads <= 65535, "%s: %d heads", what, num_heads);
  FK_REQUIRE(max_seqlen_q >= 1 && max_seqlen_q <= 65535 && max_seqlen_q * num_heads <= 0x7fffffff,
             "%s: max_seqlen_q %lld", what, static_cast<long long>(max_seqlen_q));
  FK_REQUIRE(cache_dtype == FK_DTYPE_BF16 || cache_dtype == FK_DTYPE_FP8_E4M3FN,
             "%s: the cache must be bf16 or fp8 e4m3fn", what);
  FK_REQUIRE(!cache_scale || cache_dtype == FK_DTYPE_FP8_E4M3FN, "%s: a bf16 cache has no scale",
             what);
  FK_REQUIRE(block_size >= 16 && block_size <= (1 << 30) && (block_size & (block_size - 1)) == 0,
             "%s: block_size %d must be a power of two >= 16", what, block_size);
  FK_REQUIRE(num_blocks > 0 && num_blocks <= 0x7fffffff, "%s: num_blocks %lld", what,
             static_cast<long long>(num_blocks));
  FK_REQUIRE(bt_width >= 0 && bt_width <= 0x7fffffff && bt_row_stride >= 0,
             "%s: block table of %lld columns", what, static_cast<long long>(bt_width));
  if (latent_size != 512 || rope_size != 64)
    return set_error(FK_ERR_UNSUPPORTED, "%s: rows of %d + %d unsupported (512 + 64)", what,
                     latent_size, rope_size);
  FK_REQUIRE(aligned16(q) && aligned16(out) && aligned16(cache) && q_row_stride % 8 == 0 &&
                 q_head_stride % 8 == 0 && out_row_stride % 8 == 0 && out_head_stride % 8 == 0,
             "%s: q, out and the cache must have 16-byte aligned rows", what);
  if (batch == 0 || rows == 0) return FK_OK;
  FK_REQUIRE(out && q && cache && block_tables && cache_seqlens, "%s: null pointer", what);
  if (!cu_seqlens_q) max_seqlen_q = 1;
  const LatentPlan plan = plan_of(batch, max_seqlen_q, num_heads, latent_size);
  if (workspace_bytes < plan.bytes || !workspace)
    return set_error(FK_ERR_WORKSPACE, "%s: workspace of %lld bytes, %lld needed", what,
                     static_cast<long long>(workspace_bytes), static_cast<long long>(plan.bytes));
  FK_REQUIRE(aligned16(workspace), "%s: workspace must be 16-byte aligned", what);
  uint8_t* const ws = static_cast<uint8_t*>(workspace);
  LatentParams A{};
  A.out = static_cast<uint16_t*>(out);
  A.out_row_stride = out_row_stride;
  A.out_head_stride = out_head_stride;
  A.q = static_cast<const uint16_t*>(q);
  A.q_row_stride = q_row_stride;
  A.q_head_stride = q_head_stride;
  A.cache = static_cast<const uint8_t*>(cache);
  A.cache_scale = cache_scale;
  A.lse = lse;
  A.lse_head_stride = lse_head_stride;
  A.scale_log2 = scale * kLog2e;
  A.num_heads = num_heads;
  A.batch = static_cast<int>(batch);
  A.rows = static_cast<int>(rows);
  A.most = static_cast<int>(max_seqlen_q);
  A.block_size_log2 = 31 - __builtin_clz(static_cast<unsigned>(block_size));
  A.num_blocks = num_blocks;
  A.bt_row_stride = bt_row_stride;
  A.bt_width = static_cast<int>(bt_width);
  A.wgs = num_cus() * wgs_per_cu(plan.units, cache_dtype == FK_DTYPE_FP8_E4M3FN);
  A.head_blocks = (num_heads + 31) / 32;
  A.units = plan.units;
  A.team = (A.head_blocks + plan.units - 1) / plan.units % 2 == 0 ? 2 : 1;
  A.o = reinterpret_cast<float*>(ws + plan.o);
  A.ml = reinterpret_cast<float*>(ws + plan.ml);
  A.records = reinterpret_cast<LineRecord*>(ws + plan.records);
  hipStream_t s = as_stream(stream);
  if (cache_dtype == FK_DTYPE_FP8_E4M3FN)
    launch<512, 64, true>(A, s, block_tables, cache_seqlens, cu_seqlens_q);
  else
    launch<512, 64, false>(A, s, block_tables, cache_seqlens, cu_seqlens_q);
  return check_launch(what);
}

extern "C" int fk_latent_decode_plan(int64_t batch, int64_t max_seqlen_q, int num_heads,
                                     int latent_size, int64_t* workspace_bytes) {
  FK_REQUIRE(workspace_bytes, "fk_latent_decode_plan: null output pointer");
  FK_REQUIRE(batch >= 0 && batch <= 65535 && max_seqlen_q >= 1 && max_seqlen_q <= 65535 &&
                 num_heads > 0 && num_heads <= 65535 && latent_size > 0 && latent_size <= 65536,
             "fk_latent_decode_plan: invalid argument");
  *workspace_bytes = batch == 0 ? 0 : plan_of(batch, max_seqlen_q, num_heads, latent_size).bytes;
  return FK_OK;
}
