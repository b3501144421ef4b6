// Key rows (and the key bounds of pages, which have their layout) from memory to the operand of
// the scores' matrix instructions.
#pragma once

#include "fk_attn_tile.h"

namespace fk {

// Keeps the loads before it before it: the compiler otherwise sinks them to just before their
// first use, a step later, and their latency is no longer hidden.
__device__ __forceinline__ void loads_issued() { asm volatile("" ::: "memory"); }

// K rows on their way to the scores' operand.  The operand has a key per lane (lane (r, g): 16
// bytes at 64 c + 16 g of key r), so that loads straight into it meet another row with every
// lane, and the cache takes them one lane at a time; and each of them takes half a cache line,
// whose other half then waits behind the first's miss.  They are loaded in whole rows instead,
// and a round trip through the wave's own LDS turns them.  There, chunk c holds bytes 64 c ..
// 64 c + 63 of the 16 rows; a row's four pieces are rotated by half its number, and rows trade
// places with their neighbours in odd chunks, so that neither side has bank conflicts.
template <bool kFp8, int D>
struct KChunks {
  static constexpr int kLoads = DTile<kFp8, D>::kKLoads;
  static constexpr int kBytes = 1024 * kLoads;  // of a tile
  static constexpr int kPieces = 4 * kLoads;    // 16-byte pieces of a row
  static constexpr int kRows = 64 / kPieces;    // rows per load
  static __device__ __forceinline__ int at(int row, int chunk, int piece) {
    return 1024 * chunk + 64 * (row ^ (chunk & 1)) + 16 * ((piece + (row >> 1)) & 3);
  }
  static __device__ __forceinline__ void put(const DTile<kFp8, D>& t, uint8_t* kx, int lane) {
    const int piece = lane % kPieces;
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      *reinterpret_cast<uint4*>(kx + at(kRows * i + lane / kPieces, piece >> 2, piece & 3)) =
          t.k[i];
  }
  // The first of the eight dims that lanes (r, g) hold of bf16 operand c.
  static __device__ __forceinline__ int dims(int c, int g) {
    return kFp8 ? 64 * (c >> 1) + 16 * g + 8 * (c & 1) : 32 * c + 8 * g;
  }
  static __device__ __forceinline__ void get(const uint8_t* kx, int lane, uint4 (&k)[D / 32]) {
    DTile<kFp8, D> t;
#pragma unroll
    for (int c = 0; c < kLoads; ++c)
      t.k[c] = *reinterpret_cast<const uint4*>(kx + at(lane & 15, c, lane >> 4));
    k_chunks_d(t, k);
  }
};

}  // namespace fk
