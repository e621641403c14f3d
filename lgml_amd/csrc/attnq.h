// What the attention kernels over quantised KV blocks share (formats of an f16 scale
// per 32 values): the arithmetic, scores, V's scales and P dv, and what the rows of an
// item see of a block. F is the format: its head size D, and DV, the factor of V's scales in the
// packed products.
//
// s_rc = q_r . k_c = sum_b dk_cb (q_rb . kn_cb) over the blocks b of 32 dims: the
// whole numbers kn are exact in f16, a 16x16x32 f16 MFMA takes one block of q as
// f16 hi + lo against them, and its f32 result is scaled by the cell's dk into
// S^T. q rows are scaled by a power of two to just below 2^15, so that hi + lo
// carries 22 bits of every element down to 2^-17 of the row's largest.
// o_rd = sum_c (p_rc dv_cb) vn_cd, b = d / 32: dv goes into P, per block of 32
// dims, and P dv enters the MFMAs as f16 hi + lo; O and l are 2^13 DV times as large.
// Where each dv that a row sees of the block is 0 or in [2^-8, 2^2) / DV (largest
// values of 0.03 to 31), P is split once and multiplied by DV dv in packed f16,
// the product's rounding caught by an fma: hi = P_hi dv, lo = P_lo dv + (P_hi dv -
// hi), 24 operations a lane. hi + lo keep 22 bits of a p DV dv of 2^-15 or more there,
// and are at most 2^-38 off below: the dv of a cell of weight 1 keeps its bits. Else
// P dv is made in f32 and scaled by the power of two that puts the row's largest of
// the 32 dims at 2^14 to 2^15 (22 bits down to 2^-16 of it, at most 2^-39 of it off
// below), the products scaled back as they add to O^T, some 200 operations; a cell
// that a row does not see has p and dv as zeros there, so that nothing in it (a
// scale that is infinite or NaN) reaches the row. Scaled by the largest dv instead,
// a row that attends to one quiet cell among loud ones had the loud ones' step: V
// 1e-4 of the others' was 5e-5 of itself off. The second way takes a decode of 64
// sequences at 128 to 4096 cells over Q8_0, 32 / 8 heads of 128, 80 us where the first
// takes 58 (cells in the memory-side cache).
#pragma once

#include <type_traits>

#include "attn.h"

namespace lgmlh {

__device__ __forceinline__ f32x4 mfma16q(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// The value is made here (else the compiler moves the sums of a block's products
// behind its last one, and all of them wait in registers).
__device__ __forceinline__ void here(f32x4 &v) { asm volatile("" : "+v"(v)); }
__device__ __forceinline__ float pow2(int e) { return __builtin_amdgcn_ldexpf(1.0f, e); }

// The largest v of a row's four quads: lanes 16, then 32 apart change places on
// the vector ALU (a shuffle goes through the LDS unit, which operands fill).
__device__ __forceinline__ float quads_max(float v) {
  const uint32_t a = __builtin_bit_cast(uint32_t, v);
  const auto p = __builtin_amdgcn_permlane16_swap(a, a, false, false);
  v = fmaxf(__builtin_bit_cast(float, (uint32_t)p[0]), __builtin_bit_cast(float, (uint32_t)p[1]));
  const uint32_t b = __builtin_bit_cast(uint32_t, v);
  const auto q = __builtin_amdgcn_permlane32_swap(b, b, false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)q[0]), __builtin_bit_cast(float, (uint32_t)q[1]));
}

// The lane, of which what follows is made anew where it is used: held over a loop, it
// takes registers that heads of 256 do not have.
__device__ __forceinline__ int lane_anew() {
  int lane = threadIdx.x;
  asm volatile("" : "+v"(lane));
  return lane & 63;
}

// A block's word from the lane's first cell, 8 quad, on.
__device__ __forceinline__ uint64_t lane_cells(uint64_t word) { return word >> (lane_anew() >> 1 & 24); }

// |scale| as the f16's bits, where NaN is above the infinity: the largest of 8,
// and the least but for zeros, less 1 (none: 0xffff). Floats of the numbers go
// through the lanes' maxima.
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ float high_bits(u32x4 s) {
  u16x2 w[4];
#pragma unroll
  for (int i = 0; i < 4; i++) w[i] = __builtin_bit_cast(u16x2, s[i] & 0x7fff7fffu);
  const u16x2 m = __builtin_elementwise_max(__builtin_elementwise_max(w[0], w[1]), __builtin_elementwise_max(w[2], w[3]));
  return (float)(m[0] > m[1] ? m[0] : m[1]);
}
__device__ __forceinline__ float low_bits(u32x4 s) {
  u16x2 w[4];
#pragma unroll
  for (int i = 0; i < 4; i++) w[i] = __builtin_bit_cast(u16x2, s[i] & 0x7fff7fffu) - u16x2{1, 1};
  const u16x2 m = __builtin_elementwise_min(__builtin_elementwise_min(w[0], w[1]), __builtin_elementwise_min(w[2], w[3]));
  return (float)(m[0] < m[1] ? m[0] : m[1]);
}
// Whether scales go by the packed products: each is 0 or in [2^-8, 2^2) / F::DV.
// (Up to 2^15 with P's and its own factor; from there on a p of 1 keeps 22 bits.)
template <typename F>
__device__ __forceinline__ bool plain_range(float low, float high) {
  constexpr int ONE = 15 - __builtin_ctz(F::DV);  // the exponent's bits of 1 / DV
  return high < (float)((ONE + 2) << 10) && low >= (float)(((ONE - 8) << 10) - 1);
}
// The scales of a lane's cells (32 h + 8 quad + e) of one block of 32 dims, those
// of cells that word leaves out as zeros.
__device__ __forceinline__ void seen_scales(u32x4 &s0, u32x4 &s1, uint64_t word) {
  word = lane_cells(word);
  const uint32_t w0 = (uint32_t)word, w1 = (uint32_t)(word >> 32);
#pragma unroll
  for (int i = 0; i < 4; i++) {
    s0[i] &= (w0 >> 2 * i & 1 ? 0xffffu : 0) | (w0 >> 2 * i & 2 ? 0xffff0000u : 0);
    s1[i] &= (w1 >> 2 * i & 1 ? 0xffffu : 0) | (w1 >> 2 * i & 2 ? 0xffff0000u : 0);
  }
}

// The exponent of the row's largest P dv of one block of 32 dims (the least of use).
__device__ __forceinline__ int largest_pdv(const f32x4 (&st)[4], const f16x8 (&dv)[2]) {
  float mx = 0.0f;
#pragma unroll
  for (int h = 0; h < 2; h++)
#pragma unroll
    for (int e = 0; e < 8; e++) mx = fmaxf(mx, fabsf(st[2 * h + (e >> 2)][e & 3] * (float)dv[h][e]));
  const int ex = __builtin_amdgcn_frexp_expf(quads_max(mx));  // it is in [2^(ex - 1), 2^ex)
  return ex < -100 ? -100 : ex;
}

// x0 and x1 as f16 hi + lo: hi by truncation, lo takes up what it leaves.
__device__ __forceinline__ void split2(float x0, float x1, f16x2 &hi, f16x2 &lo) {
  hi = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_pkrtz(x0, x1));
  lo = f16x2{(f16)fmaf((float)hi[0], -1.0f, x0), (f16)fmaf((float)hi[1], -1.0f, x1)};
}
// P dv from P's halves in packed f16, the rounding of hi caught in lo.
template <typename H>
__device__ __forceinline__ void packed_pdv(H ph, H pl, H dv, H &hi, H &lo) {
  hi = ph * dv;
  lo = __builtin_elementwise_fma(pl, dv, __builtin_elementwise_fma(ph, dv, -hi));
}
// S^T of a block: read(b, p, k, d) gives the K operands of tiles 2 p and 2 p + 1
// and the lane's cells' dk for block b of dims, query(b, hi, lo) the row's. A step
// reads the next step's operands and issues this one's products, and adds the
// last one's, scaled, while they run. (Two tiles a step: with four, heads of 256
// spill, and each spill is waited for.)
template <int NB, typename R, typename Q>
__device__ __forceinline__ void scores_q(f32x4 (&st)[4], R read, Q query) {
  f16x8 k[2][2], d[2], hi, lo;
  f32x4 acc[2][2];
#pragma unroll
  for (int ct = 0; ct < 4; ct++) st[ct] = f32x4{0, 0, 0, 0};
  read(0, 0, k[0], d[0]);
  auto add = [&](int p) {
#pragma unroll
    for (int t = 0; t < 2; t++) {
      f32x4 &s = st[2 * p + t];
#pragma unroll
      for (int i = 0; i < 4; i++) s[i] = fmaf((float)d[p][4 * t + i], acc[p][t][i], s[i]);
      here(s);
    }
  };
#pragma unroll
  for (int b = 0; b < NB; b++) {
    query(b, hi, lo);
#pragma unroll
    for (int p = 0; p < 2; p++) {
#pragma unroll
      for (int t = 0; t < 2; t++) acc[p][t] = mfma16q(k[p][t], hi, f32x4{0, 0, 0, 0});
#pragma unroll
      for (int t = 0; t < 2; t++) acc[p][t] = mfma16q(k[p][t], lo, acc[p][t]);
      if (b + p > 0) add(p ^ 1);
      if (p == 0 || b + 1 < NB) read(b + p, p ^ 1, k[p ^ 1], d[p ^ 1]);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  add(1);
}

// A lane's row of an item: its token of the item, its head among the G (1, 2, 4, 8
// or 16) of the KV head, and whether the item has it.
struct RowOf {
  int row, quad, rtok, head;
  bool valid;
  __device__ __forceinline__ RowOf(int lane, int G, int ntok)
      : row(lane & 15), quad(lane >> 4), rtok(row >> __builtin_ctz(G)), head(row & (G - 1)), valid(rtok < ntok) {}
};

// What the rows of an item see of a block of a causal, ring or tree plan.
struct Sight {
  int ring, window;     // of the plan; ring LGMLH_PLAN_TREE: a tree
  int p_first, p_last;  // the item's first and last slots
  int b_tree;
  int G, ntok;
  const uint64_t *vis;  // the mask words of the item's first token
  Sight() = default;
  __device__ __forceinline__ Sight(int seq_off, int npast, int tok0, int n, int G, int ring, int window,
                                   const uint64_t *vis)
      : ring(ring), window(window), p_first(npast + (tok0 - seq_off)), p_last(p_first + n - 1), b_tree(npast / KV_BLOCK),
        G(G), ntok(n), vis(ring < 0 ? vis + (int64_t)tok0 * window : nullptr) {}
  // Whether some row of the item does not see all of a block (the same for the
  // wave, and for every plan that shows the rows the same cells), and the lane's
  // row's word then (0 of a row that the item does not have).
  __device__ __forceinline__ bool masks(int blk, uint64_t &w) const {
    if (ring < 0 ? blk < b_tree : blk * 64 + 63 <= p_first && (ring == 0 || blk * 64 > p_last - window)) return false;
    const RowOf r(lane_anew(), G, ntok);
    w = r.valid ? word(blk, r.rtok) : 0;
    return ring >= 0 || __builtin_amdgcn_ballot_w64(r.valid && ~w != 0) != 0;
  }
  __device__ __forceinline__ uint64_t word(int blk, int rtok) const {
    if (ring < 0) return vis[rtok * window + blk - b_tree];
    const int p_row = p_first + rtok;  // the row's last visible slot
    const int hi = p_row - blk * 64, lo = ring > 0 ? p_row - window + 1 - blk * 64 : 0;
    uint64_t w = hi >= 63 ? ~(uint64_t)0 : hi < 0 ? 0 : ((uint64_t)2 << hi) - 1;
    if (lo >= 64)
      w = 0;
    else if (lo > 0)
      w &= ~(uint64_t)0 << lo;
    return w;
  }
};

}  // namespace lgmlh
