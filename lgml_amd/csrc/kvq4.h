// Places in the tiles of the Q4_0 KV pool, and its rounding.
#pragma once

#include "common.h"

namespace lgmlh {

// A (block, KV head) tile of K or V: 32 D bytes of 4-bit values n, which stand for
// (n - 8) d, then the f16 scales d [D / 32][64 cells]. Values are placed so that one
// 16-byte load a lane (8 of K's heads of 64) gives its part of the attention's
// 16x16x32 operands, and so that no byte holds two cells: a cell's values are whole
// bytes, written without a read.
//   K: [D / 32 U][cell][4][U][4 bytes], U = min(4, D / 32): dims 32 (U j + u) + 8 q ..
//      + 7 of a cell are the word (j, cell, q, u), dim e of them its bits from 4 (e /
//      2) + 16 (e % 2) on: a shift and a mask take a pair (e, e + 1) into the two
//      halves of a register.
//   V: [D / 32][16][4][2][8 bytes]: byte (j, r, q, b, .) of cell 32 b + 8 q + e holds
//      dims 32 j + r (its low half) and 32 j + 16 + r, a row of each of two operands;
//      the bytes of cells e, e + 1 (e even) are two apart, for the same mask.
// The scales stand as the Q8_0 tile's.
__host__ __device__ constexpr int q4_tile_bytes(int D) { return 36 * D; }
__host__ __device__ constexpr int q4_k_words(int D) { return D >= 128 ? 4 : D / 32; }  // U
// K's word of the 8 dims from d on (a multiple of 8)
__device__ __forceinline__ int q4_k_at(int D, int cell, int d) {
  const int U = q4_k_words(D);
  return (((d / (32 * U) * 64 + cell) * 4 + d % 32 / 8) * U + d / 32 % U) * 4;
}
// V's byte of a cell for row p = 16 j + r (dims 32 j + r and 32 j + 16 + r)
__device__ __forceinline__ int q4_v_byte(int e) { return (e & 4) | (e & 1) << 1 | (e >> 1 & 1); }
__device__ __forceinline__ int q4_v_at(int p, int cell) {
  return p * 64 + cell % 32 / 8 * 16 + cell / 32 * 8 + q4_v_byte(cell % 8);
}
__device__ __forceinline__ int q4_scale_at(int D, int b, int cell) { return 32 * D + 2 * (b * 64 + cell); }

// n of x for id = 1 / d: the product is rounded to f32 by itself, then its sum with
// 8.5 (an fma of both would round once).
__device__ __forceinline__ uint32_t q4_round(float x, float id) {
#pragma clang fp contract(off)
  const float p = x * id;
  return (uint32_t)__builtin_amdgcn_fmed3f(p + 8.5f, 0.0f, 15.0f);
}

}  // namespace lgmlh
