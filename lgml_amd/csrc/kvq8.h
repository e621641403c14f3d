// Places in the tiles of the Q8_0 KV pool, and its rounding.
#pragma once

#include "common.h"

namespace lgmlh {

// A (block, KV head) tile of K or V: 64 D int8 values, then the f16 scales
// [D / 32][64 cells]. Values are placed so that one 16-byte load a lane gives its
// part of two of the attention's 16x16x32 operands:
//   K: [D / 64][cell][4][2][8], dim 64 j + 32 b + 8 q + e at (j, cell, q, b, e)
//   V: [D][4][2][8], cell 32 b + 8 q + e at (d, q, b, e)
// The scales' order is the one in which a lane has 8 cells of a block of 32
// dims in 16 bytes.
__host__ __device__ constexpr int q8_tile_bytes(int D) { return 68 * D; }
// K's dim d of a cell, V's (d, cell), the scale of dims 32 b .. + 31
__device__ __forceinline__ int q8_k_at(int cell, int d) {
  return ((d / 64 * 64 + cell) * 4 + d % 32 / 8) * 16 + d % 64 / 32 * 8 + d % 8;
}
__device__ __forceinline__ int q8_v_at(int d, int cell) {
  return d * 64 + cell % 32 / 8 * 16 + cell / 32 * 8 + cell % 8;
}
__device__ __forceinline__ int q8_scale_at(int D, int b, int cell) {
  return 64 * D + 2 * (b * 64 + cell);
}

// The f32 product x y to the nearest integer, halves away from zero, below 2^23:
// the largest number under a half takes a half up to the next integer (its sum
// rounds there) and nothing below it. The product is rounded by itself first, as
// the format defines it: in an fma with the sum, a product just below a half that
// rounds to it goes down (6 of 1.3e8 normal values).
__device__ __forceinline__ int round_away(float x, float y) {
#pragma clang fp contract(off)
  const float p = x * y;
  return (int)(p + __builtin_copysignf(0x1.fffffep-2f, p));
}

}  // namespace lgmlh
