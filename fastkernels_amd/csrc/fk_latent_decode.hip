// Decode attention over a cache of latent rows, in the absorbed form: every query head attends
// to the same keys, a token's row of R + P values, and the values are its first R,
//   s[t, h, j] = scale q[t, h] . row_j,   out[t, h] = sum_j softmax_j(s) row_j[0 .. R).
//
// The query rows of a sequence times the heads are the columns of matrix products with the
// keys: S^T = K Q^T, then O^T += V^T P^T.  Keys come through LDS once: S reads them as rows, P V
// the same bytes with the transpose loads.  Items (sequence, 64 columns) of 32-key steps lie on
// one line, cut into equal ranges, one per CU (fk_lines.h).  An item inside one range is finished
// there; of the others each part leaves a partial state, which a second launch merges.
//
// LDS holds a tile (32 keys) as rows of bf16; the 16-byte pieces of row t are permuted within
// each run of 8 by (t / 2) mod 8, which with the row's length of 128 bytes more than a multiple
// of 256 spreads what 16 lanes read at a time over all banks.
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
constexpr int kPad = 14;     // what a part costs besides its steps, in steps
// (Weights to 2^32: with values up to 2^90 their sums stay finite.  No logits of trained models come
// near it.)
constexpr float kFar = 32.f;

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

// A tile in LDS.
template <int R, int P>
struct Tile {
  static constexpr int kRow = 2 * (R + P);        // bytes
  static constexpr int kPieces = kRow / 16;
  static constexpr int kBytes = kKeys * kRow;
  static constexpr int kMoves = kPieces / 8;  // of 64 pieces, of eight rows
  static_assert(kPieces % 8 == 0, "whole runs of pieces, whole moves of eight rows");
  static __device__ __forceinline__ int at(int row, int piece) {
    return row * kRow + 16 * ((piece & ~7) | ((piece ^ (row >> 1)) & 7));
  }
  // Where in its eight rows of the cache a lane finds the piece that goes to LDS bytes
  // 1024 m + 16 lane of them (rows from a multiple of 8 on, `odd`: not of 16).
  static __device__ __forceinline__ uint32_t source(int m, int lane, bool odd) {
    const int x = 64 * m + lane;
    const int row = x / kPieces, slot = x % kPieces;
    return row * kRow + 16 * ((slot & ~7) | ((slot ^ ((row >> 1) + (odd ? 4 : 0))) & 7));
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
__device__ __forceinline__ bf16x8_t joined(short4_t a, short4_t b) {
  const uint2 x = __builtin_bit_cast(uint2, a), y = __builtin_bit_cast(uint2, b);
  return __builtin_bit_cast(bf16x8_t, make_uint4(x.x, x.y, y.x, y.y));
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
  const float f = L > 0.f ? vsc / L : 0.f;
  *reinterpret_cast<uint2*>(P.out + row * P.out_row_stride + head * P.out_head_stride + dim) =
      make_uint2(pack2(o.x * f, o.y * f), pack2(o.z * f, o.w * f));
  if (dim == 0 && P.lse)
    P.lse[head * P.lse_head_stride + row] =
        L > 0.f ? (M + __builtin_amdgcn_logf(L)) * 0.6931471805599453f : L == 0.f ? kNegInf : L;
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
// A column's weights are 2^(logit - m), m the maximum of the first step: bf16 and the fp32 sums
// hold great weights as exactly as small ones, and O is not rescaled.  Where a later maximum, which
// all waves know behind the next barrier, is 2^kFar times that, the part is taken in two: the state
// so far goes to memory, and what follows begins again with its own maximum and is merged with it.
constexpr int tiles_of(bool fp8) { return fp8 ? 3 : 4; }
template <int R, int P, int kUnits, bool kFp8>
__global__ __launch_bounds__(kThreads)
__attribute__((amdgpu_waves_per_eu(1, 1))) void latent_decode_kernel(
    LatentParams A, const int32_t* __restrict__ bt, const int32_t* __restrict__ ctx_lens,
    const int32_t* __restrict__ cu) {
  using T = Tile<R, P>;
  constexpr int kCols = 32 * kUnits;
  constexpr int kCB = kUnits;            // blocks of 16 columns of a wave's S
  constexpr int kKc = (R + P) / 32;      // products of S
  constexpr int kOb = R / 4 / 32;        // blocks of 32 dims of a wave
  constexpr int kGroup = 3;              // K operands read from LDS at a time
  constexpr int kMoves = T::kMoves;      // of a wave and tile: eight rows
  static_assert(kKc % kGroup == 0 && kOb % 2 == 0, "whole groups");
  // Tiles in LDS: bf16 four, of which two are on their way; fp8 three, and the codes of two to
  // come (a wave's own eight rows each).
  constexpr int kBuffers = tiles_of(kFp8);
  constexpr int kCodes = 8 * (R + P);    // bytes of a wave's codes of a tile
  constexpr int kWide = kCodes / 1024, kCodeMoves = kWide + kCodes % 1024 / 256;
  static_assert(kCodes % 512 == 0, "whole moves");
  __shared__ LineLds<kThreads, kSeqs> line;
  extern __shared__ __align__(16) uint8_t lds[];
  uint8_t* const p_lds = lds + 4 * T::kBytes;  // of two steps, [columns][32 keys] bf16
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
  // A wave loads eight rows of a tile.
  uint32_t src[kFp8 ? 1 : kMoves];
#pragma unroll
  for (int m = 0; m < (kFp8 ? 1 : kMoves); ++m)
    src[m] = kFp8 ? lane : T::source(m, lane, wave & 1);
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
      const uint32_t to = kFp8 ? 3 * T::kBytes + ((s & 1) * 4 + wave) * kCodes
                               : s % kBuffers * T::kBytes + wave * (T::kBytes / 4);
      return Moves{keys.rows(pg, key), lds0 + to};
    };
    constexpr int kLoads = kFp8 ? kCodeMoves : kMoves;
    auto issue = [&](const Moves& m, int i) {
      if constexpr (!kFp8)
        lds_load16(m.from, src[i], m.to + 1024 * i);
      else if (i < kWide)
        lds_load16(m.from + 1024 * i, 16 * src[0], m.to + 1024 * i);
      else
        lds_load4(m.from + 1024 * kWide + 256 * (i - kWide), 4 * src[0],
                  m.to + 1024 * kWide + 256 * (i - kWide));
    };
    auto load = [&](int s) {
      const Moves m = moves_of(s);
#pragma unroll
      for (int i = 0; i < kLoads; ++i) issue(m, i);
    };
    // Keys that the row does not see may hold anything, infinities and NaN among it, which a zero
    // weight would not undo: their rows become zeros.  bf16: among this wave's rows of step s.
    auto clear = [&](int s) {
      const int n = seen(s, 8 * wave);
      if (n >= 8) return;
      uint8_t* const at = lds + s % kBuffers * T::kBytes + wave * (T::kBytes / 4) + 16 * lane;
#pragma unroll
      for (int i = 0; i < kMoves; ++i)
        if (64 * i + lane >= max(n, 0) * T::kPieces)
          *reinterpret_cast<uint4*>(at + 1024 * i) = make_uint4(0, 0, 0, 0);
    };
    // fp8: this wave's codes of step s, which have come, become a tile's rows; the i-th 512 bytes.
    // (Piece 64 i + lane of the eight rows: bytes 8 (64 i + lane) of the codes.)
    uint32_t row_at[kFp8 ? kMoves : 1];
#pragma unroll
    for (int i = 0; i < (kFp8 ? kMoves : 0); ++i) {
      const int piece = 64 * i + lane;
      row_at[i] = T::at(8 * wave + piece / T::kPieces, piece % T::kPieces);
    }
    auto codes = [&](int s, int i) {
      return *reinterpret_cast<const uint2*>(lds + 3 * T::kBytes + ((s & 1) * 4 + wave) * kCodes +
                                             8 * lane + 512 * i);
    };
    auto convert = [&](int s, int n, int i, uint2 v) {
      const bool ok = lane < n * T::kPieces - 64 * i;
      v = make_uint2(ok ? v.x : 0, ok ? v.y : 0);
      const uint2 a = fp8x4_to_bf16x4(v.x), c = fp8x4_to_bf16x4(v.y);
      *reinterpret_cast<uint4*>(lds + s % kBuffers * T::kBytes + row_at[kFp8 ? i : 0]) =
          make_uint4(a.x, a.y, c.x, c.y);
    };
    auto convert_all = [&](int s) {
      const int n = min(max(seen(s, 8 * wave), 0), 8);
#pragma unroll
      for (int i = 0; i < kMoves; ++i) convert(s, n, i, codes(s, i));
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
    // S of step s, in logits.  Operands come in groups, one ahead of the products.  Piece 4 k + g
    // of a row: of its place, k / 2 moves it by 128 bytes, k % 2 by a permutation.
    const uint32_t k_at[2] = {static_cast<uint32_t>(T::at(16 * ts + r, g)),
                              static_cast<uint32_t>(T::at(16 * ts + r, 4 + g))};
    // (among(x): what to do among the products of the x-th group)
    auto scores = [&](int s, floatx4_t (&p)[kCB], auto among) {
      const uint8_t* const tile = lds + (s % kBuffers) * T::kBytes;
      const uint8_t* const at[2] = {tile + k_at[0], tile + k_at[1]};
      uint4 kx[2][kGroup];
#pragma unroll
      for (int j = 0; j < kGroup; ++j)
        kx[0][j] = *reinterpret_cast<const uint4*>(at[j & 1] + 128 * (j >> 1));
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
            kx[now ^ 1][j] = *reinterpret_cast<const uint4*>(at[(k0 + kGroup + j) & 1] +
                                                             128 * ((k0 + kGroup + j) >> 1));
        }
        among(k0 / kGroup);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < kGroup; ++j)
#pragma unroll
          for (int cb = 0; cb < kCB; ++cb)
            x[j % kChains][cb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                __builtin_bit_cast(bf16x8_t, kx[now][j]), qb[cb][k0 + j], x[j % kChains][cb], 0,
                0, 0);
      }
#pragma unroll
      for (int cb = 0; cb < kCB; ++cb)
        p[cb] = kChains == 1 ? x[0][cb] : x[0][cb] + x[kChains - 1][cb];
    };
    // The softmax of step s, in four parts: logits, their maxima, weights.
    // (The weights are rounded to bf16 for P V, 2^-9 relative at most, of either sign; their sum
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
      for (int i = 0; i < 4; ++i) e[i] = __builtin_amdgcn_exp2f(p[cb][i] - ms[cb]);
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
    // a transpose load, lane 4 a + q of each 16 addresses key a and dims 4 q .. 4 q + 3; block d's
    // place in a row moves by 128 bytes with d / 2 and by a permutation with d % 2.
    uint32_t v_at[2][2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int d = 0; d < 2; ++d)
        v_at[h][d] = 8 * (lane & 1) +
                     T::at(8 * kh + 4 * h + (r >> 2),
                           wave * (R / 32) + 4 * d + 2 * (g & 1) + ((lane & 3) >> 1));
    const uint8_t* const p_from = p_at(n, 8 * kh);  // keys 16 on: pieces 2 on, of four, permuted
    const int p_next = 32 - 64 * (((kh ^ (n >> 2)) & 3) >> 1);
    auto v_operand = [&](const uint8_t* tile, int x) {  // keys 16 (x / kOb) on, block x % kOb
      const int k = x / kOb, d = x % kOb;
      const int off = 16 * k * T::kRow + 128 * (d >> 1);
      return joined(transposed(tile + v_at[0][d & 1] + off), transposed(tile + v_at[1][d & 1] + off));
    };
    // The first operands of P V of step s: its weights, and V's of the first group.
    constexpr int kVGroup = kOb / 2;
    struct First {
      bf16x8_t w[2][kUnits], v[kVGroup];
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
        f.v[j] = v_operand(lds + (s % kBuffers) * T::kBytes, j);
    };
    // (among(x): what to do among the products of the x-th quarter)
    auto values = [&](int s, const First& f, auto among) {
      const uint8_t* const tile = lds + (s % kBuffers) * T::kBytes;
      bf16x8_t v[2][kVGroup];
#pragma unroll
      for (int j = 0; j < kVGroup; ++j) v[0][j] = f.v[j];
#pragma unroll
      for (int x0 = 0; x0 < 2 * kOb; x0 += kVGroup) {
        const int now = x0 / kVGroup & 1;
        if (x0 + kVGroup < 2 * kOb) {
#pragma unroll
          for (int j = 0; j < kVGroup; ++j) v[now ^ 1][j] = v_operand(tile, x0 + kVGroup + j);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < kVGroup; ++j) {
          const int k = (x0 + j) / kOb, d = (x0 + j) % kOb;
#pragma unroll
          for (int u = 0; u < kUnits; ++u)
            o[u][d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v[now][j], f.w[k][u], o[u][d], 0, 0,
                                                              0);
        }
        among(x0 / kVGroup);
      }
    };

    floatx4_t p[kCB], next[kCB];
    // A step's barrier: step s's weights and maxima and step s + 1's tile are in LDS, and step
    // s - 1 is done with.  The loads (bf16: of step s + 3, fp8: of s + 4, with the conversion of
    // s + 2) are issued among its products, so that the waves do not wait for their addresses to
    // be taken.
    auto enter = [&](int s, float (&t)[kUnits]) {
      if constexpr (!kFp8) {
        wait_loads<kLoads>();
        clear(s + 1);
      }
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
    if constexpr (kFp8) {
      convert_all(0);
      convert_all(1);
      load(2);
      load(3);
    } else {
      clear(0);
      load(2);
    }
    __syncthreads();
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
    constexpr int kAhead = kFp8 ? 4 : 3;
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
        int rows = 0;
        uint2 raw[3];  // codes on their way from LDS
        if constexpr (kFp8) {
          wait_loads<kLoads>();
          rows = min(max(seen(s + 2, 8 * wave), 0), 8);
#pragma unroll
          for (int i = 0; i < 3; ++i) raw[i] = codes(s + 2, i);
        }
        scores(s + 1, next, [&](int x) {
          if constexpr (kFp8) {
            convert(s + 2, rows, x, raw[x % 3]);
            raw[x % 3] = codes(s + 2, x + 3);
          } else {
            issue(m, x);
          }
          if (x == kGroups - 1) first_operands(s, f);
        });
        if (too_far(t)) break;  // (looked at behind the products that do not depend on it)
        count();
        values(s, f, [&](int x) {
          if (x == 0) logits(s + 1, next);
          if (x == 1) maxima(s + 1, next);
          if (x >= 2 && x - 2 < kCB) weights(s + 1, next, x - 2);
          if constexpr (kFp8) {
            if (x < kMoves - kGroups) convert(s + 2, rows, kGroups + x, raw[x]);
            if (x == 3) {
              // (the codes have been read, whose place the loads take)
              __builtin_amdgcn_sched_barrier(0);
              asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
              for (int i = 0; i < kLoads; ++i) issue(m, i);
            }
          } else if (x < kMoves - kGroups) {
            issue(m, kGroups + x);
          }
          if (x == 3) m = moves_of(s + 1 + kAhead);
        });
        static_assert(kGroups % 3 == 0 && kMoves - kGroups == 3, "all of them once");
        p[0] = next[0];
        if constexpr (kCB == 2) p[1] = next[1];
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
    static_assert(4 * kCols * kRow <= 4 * T::kBytes, "O fits");
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
  int wgs, units;
  int64_t o, ml, records, bytes;
};
LatentPlan plan_of(int64_t batch, int64_t max_seqlen_q, int num_heads, int latent_size) {
  LatentPlan p{};
  p.units = num_heads > 32 ? 2 : 1;
  p.wgs = num_cus();
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
  const unsigned lds = 4 * Tile<R, P>::kBytes + 2 * 32 * A.units * (kKeys * 2 + 2 * 4);
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
  A.wgs = plan.wgs;
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
