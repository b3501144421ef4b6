// The 4-bit cache format (OCP microscaling fp4): blocks of 32 dims of one token and kv head,
// each a power of two 2^(E - 127) (one byte E; 255: the block is NaN) times 32 e2m1 codes
// (0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign).
//
// K codes     [page][head][token][D / 2]            two dims a byte, the even one low
// V codes     [page][head][token / 4][16][4][D / 32]  four tokens side by side, for each
//             sixteenth of the head: what a lane of P V takes is one load
// K, V scales [page][head][D / 32][token]           a lane's eight keys are one load
#pragma once

#include "fk_attn_tile.h"

namespace fk {

// Scale byte i of four in a word, as the conversions' scale operand: they take its exponent
// field alone, so what else the shift leaves in the word does not count.
template <int kByte>
__device__ __forceinline__ float scale_of(uint32_t w) {
  return __uint_as_float(kByte == 3 ? w >> 1 : w << (23 - 8 * kByte));
}
// The two codes of byte i of w as bf16 values times the scale: exact up to the scale 2^125, and
// beyond it but for values of 2^128 and more (a store makes none), which become infinities.
template <int kByte>
__device__ __forceinline__ uint32_t fp4x2_to_bf16x2(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t,
                            __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, kByte));
}
// The eight codes of a word.
__device__ __forceinline__ uint4 fp4x8_to_bf16x8(uint32_t w, float scale) {
  return make_uint4(fp4x2_to_bf16x2<0>(w, scale), fp4x2_to_bf16x2<1>(w, scale),
                    fp4x2_to_bf16x2<2>(w, scale), fp4x2_to_bf16x2<3>(w, scale));
}
// Scale byte of a block whose greatest magnitude is `top`: the exponent of top rounded to two
// significant bits, less that of the format's greatest power (4).  Rounded so, top is at most 7
// of the block's units, and every value at most half a step of the grid from its code.  (With
// top's own exponent, 6 would stand for values up to 8.)  From 1.75 2^127 on that scale's code would
// be 2^128, which reads back as an infinity: such values become 1.5 2^127, the greatest below it.
constexpr uint32_t kTopScale = 252;
// Scales above it may have infinities among their values, or NaN (255).
__device__ __forceinline__ bool all_finite(uint32_t e) { return e <= kTopScale; }
__device__ __forceinline__ uint32_t block_scale(float top) {
  const uint32_t u = __float_as_uint(top);
  if (u >= 0x7f800000u) return 255;  // infinity, NaN
  const uint32_t e = (u + 0x200000u) >> 23;
  return e > 2 ? min(e - 2, kTopScale) : 0;
}

}  // namespace fk
