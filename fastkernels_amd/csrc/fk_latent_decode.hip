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
constexpr int kKeys = 32;    // of a tile
constexpr int kBuffers = 4;  // tiles in LDS

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
  static constexpr int kMoves = kKeys * kPieces / 64;  // 64-piece moves of a tile
  static_assert(kPieces % 8 == 0 && kKeys / 2 * kPieces % 64 == 0, "whole moves of half a tile");
  static __device__ __forceinline__ int at(int row, int piece) {
    return row * kRow + 16 * ((piece & ~7) | ((piece ^ (row >> 1)) & 7));
  }
  // Where in its half's rows of the cache (elements of kElt bytes) lane `lane` of move m of
  // the half finds the piece that goes to LDS bytes 1024 m + 16 lane of the half.
  template <int kElt>
  static __device__ __forceinline__ uint32_t source(int m, int lane) {
    const int x = 64 * m + lane;
    const int row = x / kPieces, slot = x % kPieces;
    return row * (R + P) * kElt + 8 * kElt * ((slot & ~7) | ((slot ^ (row >> 1)) & 7));
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
__device__ __forceinline__ bf16x8_t masked(bf16x8_t v, const uint32_t (&m)[4]) {
  const uint4 x = __builtin_bit_cast(uint4, v);
  return __builtin_bit_cast(bf16x8_t,
                            make_uint4(x.x & m[0], x.y & m[1], x.z & m[2], x.w & m[3]));
}
// Masks of the four words that hold eight 16-bit values, from a bit each.
__device__ __forceinline__ void word_masks(uint32_t bits, uint32_t (&m)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    m[i] = (bits >> (2 * i) & 1 ? 0xffffu : 0u) | (bits >> (2 * i + 1) & 1 ? 0xffff0000u : 0u);
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const bf16x2_t x = {static_cast<__bf16>(a), static_cast<__bf16>(b)};
  return __builtin_bit_cast(uint32_t, x);
}
__device__ __forceinline__ float halves_max(float v) {
  const auto c = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(c[0]), __uint_as_float(c[1]));
}
__device__ __forceinline__ float halves_sum(float v) {
  const auto c = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(c[0]) + __uint_as_float(c[1]);
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

// O *= alpha, in place among the accumulators: the compiler would copy them out and back around
// every step for it.  (The waits: vector instructions read a product's result 18 later at the
// earliest, and products what those wrote 2 later.)
template <int N>
__device__ __forceinline__ void scale_acc(floatx16_t (&o)[N], float alpha) {
#pragma unroll
  for (int d = 0; d < N; ++d) {
    asm volatile("s_nop 15\n\ts_nop 3" : "+a"(o[d]), "+v"(alpha));
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float x = o[d][i], t;
      asm volatile(
          "v_accvgpr_read_b32 %1, %0\n\t"
          "v_mul_f32 %1, %1, %2\n\t"
          "v_accvgpr_write_b32 %0, %1"
          : "+a"(x), "=&v"(t)
          : "v"(alpha));
      o[d][i] = x;
    }
    asm volatile("s_nop 3" : "+a"(o[d]));
  }
}

// A sequence's items: `units` units (32 heads of a row) each, in steps of a tile.
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
  x.items = (s.rows * P.head_blocks + units - 1) / units;
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

// One work-group: items of kUnits units of 32 heads (of one query row each), in steps of a tile.
//
// The waves share S by columns and keys, wave w = (cs, ts): half cs of the columns and keys
// 16 ts .. 16 ts + 15 (16x16x32 products), and P V by dims: wave w has dims w R / 4 .. of every
// column (32x32x16 products), so that V is read from LDS once and K twice.  P goes through LDS,
// and so do the columns' maxima.
//
// A step has one barrier.  Behind it come S of the next step and P V of this one, with the next
// step's softmax among the products of the latter: its weights are made with the reference maxima
// as they are, and only where the maxima, which are all known behind the next barrier, ask for
// others is P made again.
template <int R, int P, int kUnits, bool kFp8>
__global__ __launch_bounds__(kThreads)
__attribute__((amdgpu_waves_per_eu(1, 1))) void latent_decode_kernel(
    LatentParams A, const int32_t* __restrict__ bt, const int32_t* __restrict__ ctx_lens,
    const int32_t* __restrict__ cu) {
  using T = Tile<R, P>;
  constexpr int kCols = 32 * kUnits;
  constexpr int kCB = kUnits;                 // blocks of 16 columns of a wave's S
  constexpr int kKc = (R + P) / 32;           // products of S
  constexpr int kOb = R / 4 / 32;             // blocks of 32 dims of a wave
  constexpr int kMoves = T::kMoves / kWaves;  // of a wave and tile
  static_assert(T::kMoves / 2 % kMoves == 0, "a wave's moves are of one half");
  constexpr int kGroup = kFp8 && kUnits == 2 ? 2 : 3;  // K operands read from LDS at a time
  static_assert(kKc % kGroup == 0 && kOb % 2 == 0, "whole groups");
  __shared__ LineLds<kThreads> line;
  extern __shared__ __align__(16) uint8_t lds[];
  uint8_t* const p_lds = lds + kBuffers * T::kBytes;  // of two steps, [columns][32 keys] bf16
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
  const int half = wave * kMoves / (T::kMoves / 2);
  const int move0 = wave * kMoves % (T::kMoves / 2);  // of the half
  uint32_t src[kMoves];
#pragma unroll
  for (int m = 0; m < kMoves; ++m) src[m] = T::template source<kFp8 ? 1 : 2>(move0 + m, lane);
  const uint32_t dst0 = half * (T::kBytes / 2) + move0 * 1024;
  const uint32_t lds0 = lds_addr_of(lds);
  // 16 bytes (8 keys) of a column's weights, their pieces permuted against bank conflicts.
  auto p_at = [&](int col, int key) {
    return p_lds + col * 64 + 16 * (((key >> 3) ^ (col >> 2)) & 3) + 2 * (key & 7);
  };

  auto body = [&](int b, const SeqRows& sr, const LineItems& x, int it, int s_lo, int s_hi,
                  int64_t slot) {
    // Row, first head and visible keys of the units; one that there is not has no heads.
    int row_i[kUnits], head0[kUnits], hi[kUnits];
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int unit = min(it * kUnits + u, sr.rows * A.head_blocks - 1);
      int none;
      row_i[u] = unit / A.head_blocks;
      head0[u] = it * kUnits + u > unit ? A.num_heads
                                        : 32 * (unit - row_i[u] * A.head_blocks);
      row_keys(sr, row_i[u], -1, none, hi[u]);
      hi[u] = uniform(hi[u]);
    }
    const int all_hi = min(hi[0], hi[kUnits - 1]);
    const int su = kUnits == 2 ? cs : 0;  // unit of S's columns
    const int my_hi = su ? hi[kUnits - 1] : hi[0];
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
    // The pages of the next 32 steps' halves, a lane each; and which of them, and of the 32
    // steps before, there are.
    int pages = -1, looked_up = -1;
    uint64_t there = 0, there_before = 0;
    uint2 raw[kFp8 ? kMoves : 1];
    // This wave's loads of step s: where from, and bf16: where to.
    struct Moves {
      const uint8_t* from;
      uint32_t to;
    };
    auto moves_of = [&](int s) {
      s = min(s, steps - 1);  // (past the end, once more: as many loads are on their way)
      const int key0 = (s_lo + s) * kKeys;
      if (s / 32 != looked_up) {
        looked_up = s / 32;
        pages = keys.page(static_cast<int64_t>(key0) + 16 * lane, x.to);
        there_before = there;
        there = __ballot(pages >= 0);
      }
      const int pg = __builtin_amdgcn_readlane(pages, 2 * (s & 31) + half);
      return Moves{keys.rows(pg, key0 + 16 * half), lds0 + (s % kBuffers) * T::kBytes + dst0};
    };
    // Issues the i-th of them: bf16 into LDS, fp8 into raw.
    auto issue = [&](const Moves& m, int i) {
      if constexpr (kFp8)
        raw[i] = ld8(m.from + src[i]);
      else
        lds_load16(m.from, src[i], m.to + 1024 * i);
    };
    auto load = [&](int s) {
      const Moves m = moves_of(s);
#pragma unroll
      for (int i = 0; i < kMoves; ++i) issue(m, i);
    };
    // fp8: what was loaded, as bf16, into step s's buffer.
    auto put = [&](int s) {
      uint8_t* const dst = lds + (s % kBuffers) * T::kBytes + dst0 + 16 * lane;
#pragma unroll
      for (int i = 0; i < (kFp8 ? kMoves : 0); ++i) {
        const uint2 a = fp8x4_to_bf16x4(raw[i].x), c = fp8x4_to_bf16x4(raw[i].y);
        *reinterpret_cast<uint4*>(dst + 1024 * i) = make_uint4(a.x, a.y, c.x, c.y);
      }
    };
    auto halves_of = [&](int s) -> uint32_t {
      return (s / 32 == looked_up ? there : there_before) >> (2 * (s & 31)) & 3;
    };
    // Whether every column sees all keys of step s.
    auto whole = [&](int s) { return (s_lo + s + 1) * kKeys <= all_hi && halves_of(s) == 3; };

    // The first steps' loads, and the queries behind them.
    load(0);
    if constexpr (kFp8) put(0);
    load(1);
    bf16x8_t qb[kCB][kKc];
#pragma unroll
    for (int cb = 0; cb < kCB; ++cb) {
      const int h = (su ? head0[kUnits - 1] : head0[0]) + (s_col + 16 * cb) % 32;
      const bool ok = h < A.num_heads;
      const uint16_t* const qp =
          A.q + (sr.row0 + (su ? row_i[kUnits - 1] : row_i[0])) * A.q_row_stride +
          (ok ? h : 0) * A.q_head_stride + 8 * g;
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
#pragma unroll
      for (int cb = 0; cb < kCB; ++cb) p[cb] = floatx4_t{0.f, 0.f, 0.f, 0.f};
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
            p[cb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                __builtin_bit_cast(bf16x8_t, kx[now][j]), qb[cb][k0 + j], p[cb], 0, 0, 0);
      }
    };
    // The softmax of step s, in four parts: logits, their maxima, weights.
    // (The weights are rounded to bf16 for P V, 2^-9 relative at most, of either sign; their sum
    // is of the unrounded ones.)
    auto logits = [&](int s, floatx4_t (&p)[kCB]) {
      // (keys that this lane's column sees, from its first one on; without a branch, which would
      // part the products around it)
      const int seen = halves_of(s) >> ts & 1 ? my_hi - ((s_lo + s) * kKeys + 16 * ts + 4 * g) : 0;
#pragma unroll
      for (int cb = 0; cb < kCB; ++cb)
#pragma unroll
        for (int i = 0; i < 4; ++i) p[cb][i] = i < seen ? p[cb][i] * abs_s2 : kNegInf;
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
    // Whether a maximum is too far above its reference (uniform: every wave has the same ones);
    // then the references move and the step's weights are made again.
    auto too_far = [&](const float (&t)[kUnits]) {
      bool far = false;
#pragma unroll
      for (int u = 0; u < kUnits; ++u) far |= t[u] > mo[u] + kLazyMax;
      return __ballot(far) != 0;
    };
    auto move = [&](int s, const floatx4_t (&p)[kCB], const float (&t)[kUnits]) {
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        const float m_new = fmaxf(mo[u], t[u]);
        scale_acc(o[u], __builtin_amdgcn_exp2f(mo[u] - m_new));
        mo[u] = m_new;
      }
      const float* const top = tops + (s & 1) * 2 * kCols;
#pragma unroll
      for (int cb = 0; cb < kCB; ++cb) {
        const int c = s_col + 16 * cb;
        const float m_new = fmaxf(ms[cb], fmaxf(top[c], top[kCols + c]));
        l[cb] *= __builtin_amdgcn_exp2f(ms[cb] - m_new);
        ms[cb] = m_new;
        weights(s, p, cb);
      }
      __syncthreads();
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
    auto values = [&](int s, const First& f, auto is_masked, auto among) {
      constexpr bool kMasked = decltype(is_masked)::value;
      const uint8_t* const tile = lds + (s % kBuffers) * T::kBytes;
      // Keys that the row does not see may hold anything, infinities and NaN among it: zeros.
      uint32_t mask[2][kUnits][4];
      if constexpr (kMasked) {
        const uint32_t halves = halves_of(s);
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int u = 0; u < kUnits; ++u) {
            uint32_t bits = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int t = (s_lo + s) * kKeys + 16 * k + 8 * kh + i;
              bits |= (halves >> k & 1) && t < hi[u] ? 1u << i : 0u;
            }
            word_masks(bits, mask[k][u]);
          }
      }
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
            o[u][d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                kMasked ? masked(v[now][j], mask[k][u]) : v[now][j], f.w[k][u], o[u][d], 0, 0, 0);
        }
        among(x0 / kVGroup);
      }
    };

    floatx4_t p[kCB], next[kCB];
    // A step's barrier: step s's weights and maxima and step s + 1's tile are in LDS, and step
    // s - 1 is done with.  Its loads, of step s + 3, are issued among its products, so that the
    // waves do not wait for their addresses to be taken.
    auto enter = [&](int s, float (&t)[kUnits]) {
      if constexpr (!kFp8) wait_loads<kMoves>();
      __syncthreads();
      if constexpr (kFp8) put(s + 2);
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        const float* const top = tops + (s & 1) * 2 * kCols + 32 * u + n;
        t[u] = fmaxf(top[0], top[kCols]);
      }
    };
    const auto nothing = [](int) {};
    float t[kUnits];
    First f;
    if constexpr (!kFp8) wait_loads<0>();
    __syncthreads();
    if constexpr (kFp8) put(1);
    load(2);
    scores(0, p, nothing);
    logits(0, p);
    maxima(0, p);
    __syncthreads();
    // The first references.
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
    while (true) {  // (step s has been entered)
      if (too_far(t)) move(s, p, t);
      if (s + 1 < steps && whole(s)) {
        // The steps that need nothing special, in a loop of their own: where such a step met
        // another, the compiler would copy O around.
#pragma unroll 1
        do {
          count();
          const Moves m = moves_of(s + 3);
          scores(s + 1, next, [&](int x) {
            issue(m, x);
            if (x == kKc / kGroup - 1) first_operands(s, f);
          });
          constexpr int kDone = kKc / kGroup;
          static_assert(kDone <= kMoves && kDone + 8 >= kMoves, "every load is issued once");
          values(s, f, std::false_type{}, [&](int x) {
            if (x == 0) logits(s + 1, next);
            if (x == 1) maxima(s + 1, next);
            if (x >= 2 && x - 2 < kCB) weights(s + 1, next, x - 2);
#pragma unroll
            for (int i = 0; i < 2; ++i)
              if (kDone + 2 * x + i < kMoves) issue(m, kDone + 2 * x + i);
          });
#pragma unroll
          for (int cb = 0; cb < kCB; ++cb) p[cb] = next[cb];
          ++s;
          enter(s, t);
        } while (s + 1 < steps && whole(s) && !too_far(t));
      } else {
        count();
        load(s + 3);
        first_operands(s, f);
        values(s, f, std::true_type{}, nothing);
        if (++s == steps) break;
        scores(s, p, nothing);
        logits(s, p);
        maxima(s, p);
#pragma unroll
        for (int cb = 0; cb < kCB; ++cb) weights(s, p, cb);
        enter(s, t);
      }
    }
    wait_loads<0>();
    __syncthreads();

    // The states, through LDS: the columns' sums, of both waves and all lanes that have keys of
    // theirs, and O, which leaves in whole rows.
    constexpr int kRow = R + 4;  // floats
    float* const xo = reinterpret_cast<float*>(lds);
    static_assert(4 * kCols * kRow <= kBuffers * T::kBytes, "O fits");
#pragma unroll
    for (int cb = 0; cb < kCB; ++cb) {
      l[cb] = pair_sum(l[cb]);
      tops[kCols * ts + s_col + 16 * cb] = l[cb];
    }
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      if (wave == 0) tops[2 * kCols + 32 * u + n] = mo[u];
      float* const to = xo + (32 * u + n) * kRow + wave * (R / 4) + 4 * kh;
#pragma unroll
      for (int d = 0; d < kOb; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<float4*>(to + 32 * d + 8 * i) = make_float4(
              o[u][d][4 * i], o[u][d][4 * i + 1], o[u][d][4 * i + 2], o[u][d][4 * i + 3]);
    }
    __syncthreads();
#pragma unroll 4
    for (int i = threadIdx.x; i < kCols * (R / 4); i += kThreads) {
      const int c = i / (R / 4), dim = 4 * (i % (R / 4));
      const int u = c / 32, head = (u ? head0[kUnits - 1] : head0[0]) + c % 32;
      if (head >= A.num_heads) continue;
      const float4 z = *reinterpret_cast<const float4*>(xo + c * kRow + dim);
      const float L = tops[c] + tops[kCols + c], M = tops[2 * kCols + c];
      if (slot < 0) {
        write_out(A, sr.row0 + (u ? row_i[kUnits - 1] : row_i[0]), head, dim, z, M, L, vsc);
      } else {
        *reinterpret_cast<float4*>(A.o + (slot * kCols + c) * R + dim) = z;
        if (dim == 0)
          *reinterpret_cast<float2*>(A.ml + (slot * kCols + c) * 2) = make_float2(M, L);
      }
    }
    __syncthreads();
  };
  walk_line<kThreads>(line, A.batch, A.wgs, blockIdx.x, 1, A.records,
                      [&](int b) { return seq_rows(cu, ctx_lens, b, A.rows, A.most); },
                      [&](const SeqRows& s) { return line_items(A, s, kUnits); }, body);
}

// One work-group per (query row, some of its heads, kDims of their dims): merges the pieces of an
// item that ranges cut.
template <int R, int kDims>
__global__ __launch_bounds__(kMergeThreads) void latent_merge_kernel(
    LatentParams A, const int32_t* __restrict__ ctx_lens, const int32_t* __restrict__ cu,
    int heads, int fp8) {
  __shared__ Folded folded[kMergeThreads];
  const int t = blockIdx.y, dim0 = blockIdx.z * kDims;
  int b, vis;
  if (!query_row(cu, ctx_lens, A.batch, t, b, vis)) return;
  const SeqRows s = seq_rows(cu, ctx_lens, b, A.rows, A.most);
  const int i = t - s.row0;
  if (i >= s.rows) return;
  const LineRecord rec = A.records[b];
  const float vsc = fp8 && A.cache_scale ? *A.cache_scale : 1.f;
  const int h0 = blockIdx.x * heads, h1 = min(h0 + heads, A.num_heads);
  // Unit by unit of the row's heads.
  for (int h = h0; h < h1;) {
    const int unit = i * A.head_blocks + h / 32;
    const int in = 32 * (unit % A.units) + h % 32;
    const int nc = min(h1, (h / 32 + 1) * 32) - h;
    const LinePieces pieces(rec, unit / A.units);
    if (pieces.n > 1) {
      merge_pieces<kDims>(
          0, nc, folded, [&](int) { return pieces.n; },
          [&](int k, int x, const float*& ml, const float*& o) {
            const int64_t at = pieces.slot(k) * (32 * A.units) + in + x;
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
  p.units = max_seqlen_q * ((num_heads + 31) / 32) > 1 ? 2 : 1;
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
  const unsigned lds = kBuffers * Tile<R, P>::kBytes + 2 * 32 * A.units * (kKeys * 2 + 2 * 4);
  if (A.units == 1)
    hipLaunchKernelGGL((latent_decode_kernel<R, P, 1, kFp8>), dim3(A.wgs + 1), dim3(kThreads),
                       lds, s, A, bt, ctx, cu);
  else
    hipLaunchKernelGGL((latent_decode_kernel<R, P, 2, kFp8>), dim3(A.wgs + 1), dim3(kThreads),
                       lds, s, A, bt, ctx, cu);
  // Where rows and heads do not make two work-groups a CU, the dims are dealt out too, and with
  // them threads to share a column's pieces.
  const int heads = merge_cols(A.rows, 1, A.num_heads);
  const dim3 grid((A.num_heads + heads - 1) / heads, A.rows);
  if (static_cast<int64_t>(grid.x) * grid.y < num_cus())
    hipLaunchKernelGGL((latent_merge_kernel<R, 64>), dim3(grid.x, grid.y, R / 64),
                       dim3(kMergeThreads), 0, s, A, ctx, cu, heads, kFp8 ? 1 : 0);
  else
    hipLaunchKernelGGL((latent_merge_kernel<R, R>), grid, dim3(kMergeThreads), 0, s, A, ctx, cu,
                       heads, kFp8 ? 1 : 0);
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
