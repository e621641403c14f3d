// Paged GQA attention over Q8_0 KV blocks (gfx950): the work items, rows and
// merge of attn.hip over the tiles of kvq8.hip.
//
// s_rc = q_r . k_c = sum_b dk_cb (q_rb . k8_cb) over the blocks b of 32 dims: the
// 8-bit values are exact in f16, a 16x16x32 f16 MFMA takes one block of q as
// f16 hi + lo against them, and its f32 result is scaled by the cell's dk into
// S^T. q rows are scaled by a power of two to just below 2^15, so that hi + lo
// carries 22 bits of every element down to 2^-17 of the row's largest.
// o_rd = sum_c (p_rc dv_cb) v8_cd, b = d / 32: dv goes into P, per block of 32
// dims, and P dv enters the MFMAs as f16 hi + lo; O and l are Q8_O times as large.
// Where each dv that a row sees of the block is 0 or in [2^-12, 2^-2) (largest
// values of 0.03 to 31), P is split once and multiplied by Q8_DV dv in packed f16,
// the product's rounding caught by an fma: hi = P_hi dv, lo = P_lo dv + (P_hi dv -
// hi), 24 operations a lane. hi + lo keep 22 bits of a p dv of 2^-19 or more there,
// and are at most 2^-42 off below: the dv of a cell of weight 1 keeps its bits. Else
// P dv is made in f32 and scaled by the power of two that puts the row's largest of
// the 32 dims at 2^14 to 2^15 (22 bits down to 2^-16 of it, at most 2^-39 of it off
// below), the products scaled back as they add to O^T, some 200 operations; a cell
// that a row does not see has p and dv as zeros there, so that nothing in it (a
// scale that is infinite or NaN) reaches the row. Scaled by the largest dv instead,
// a row that attends to one quiet cell among loud ones had the loud ones' step: V
// 1e-4 of the others' was 5e-5 of itself off. The second way takes the decode of 64
// sequences below 80 us where the first takes 58 (cells in the memory-side cache).
//
// Bounds. One token of 64 sequences at 128 to 4096 cells, 32 / 8 heads of 128, is
// 63 + 5 us from HBM: 296 MB at 4.7 TB/s in the first (54 with the cells in the
// memory-side cache). Trees of 61 tokens of 8 sequences at 1024 to 16384 cells, 8
// / 4 heads of 256, are 144 + 10 us: 35 GFLOP (16-bit halves of q and P make them
// 70) in 176 workgroups of 256 CUs, whose waves wait in turn for LDS: 98 reads of 1
// KB a wave and block, 6300 cycles of a CU's at 128 bytes, where the products of
// a SIMD's two waves fill 4096.
#include <type_traits>

#include "attn.h"

namespace lgmlh {

constexpr float Q8_P = 8192.0f;       // the scale of P in its halves
constexpr float Q8_DV = 16.0f;        // of V's scales in the packed products
constexpr float Q8_O = Q8_P * Q8_DV;  // of O^T and l
constexpr int SHARED_MAX = ATTN_SHARED;  // the most items of a shared run

__device__ __forceinline__ f32x4 mfma16q(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// 4 int8 as f16: 1024 + (v + 128) is the f16 0x6400 + (v + 128).
__device__ __forceinline__ void half4(uint32_t w, f16x2 &a, f16x2 &b) {
  w ^= 0x80808080u;
  const f16x2 off = {(f16)1152.0f, (f16)1152.0f};
  a = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) - off;
  b = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) - off;
}
__device__ __forceinline__ f16x8 half8(uint32_t w0, uint32_t w1) {
  f16x2 a, b, c, d;
  half4(w0, a, b);
  half4(w1, c, d);
  return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// The value is made here (else the compiler moves the sums of a block's products
// behind its last one, and all of them wait in registers).
__device__ __forceinline__ void here(f32x4 &v) { asm volatile("" : "+v"(v)); }
__device__ __forceinline__ float pow2(int e) { return __builtin_amdgcn_ldexpf(1.0f, e); }

template <int D>
struct Q8Frag {
  static constexpr int TILE = 68 * D, NB = D / 32, J = D / 64, DT = D / 16;
};

// The largest v of a row's four quads: lanes 16, then 32 apart change places on
// the vector ALU (a shuffle goes through the LDS unit, which the shared kernel's
// operands fill).
__device__ __forceinline__ float quads_max(float v) {
  const uint32_t a = __builtin_bit_cast(uint32_t, v);
  const auto p = __builtin_amdgcn_permlane16_swap(a, a, false, false);
  v = fmaxf(__builtin_bit_cast(float, (uint32_t)p[0]), __builtin_bit_cast(float, (uint32_t)p[1]));
  const uint32_t b = __builtin_bit_cast(uint32_t, v);
  const auto q = __builtin_amdgcn_permlane32_swap(b, b, false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)q[0]), __builtin_bit_cast(float, (uint32_t)q[1]));
}

// q row pieces -> B operands, hi and lo, of the row scaled by 2^(15 - e); the
// factor of the scores that undoes it.
template <int NB>
__device__ __forceinline__ float split_q(const f32x4 (&qa)[2 * NB], bool rvalid, float scale_log2,
                                         f16x8 (&hi)[NB], f16x8 (&lo)[NB]) {
  float mx = 0.0f;
#pragma unroll
  for (int i = 0; i < 2 * NB; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) mx = fmaxf(mx, fabsf(qa[i][j]));
  mx = quads_max(mx);
  int e = __builtin_amdgcn_frexp_expf(mx);
  e = e < -110 ? -110 : e;
  const float up = rvalid ? pow2(15 - e) : 0.0f;
#pragma unroll
  for (int b = 0; b < NB; b++)
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float x = rvalid ? qa[2 * b + (i >> 2)][i & 3] * up : 0.0f;
      hi[b][i] = (f16)x;
      lo[b][i] = (f16)(x - (float)hi[b][i]);
    }
  return scale_log2 * pow2(e - 15);
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

// Scores (scaled, in units of log2) -> P in place, the running maximum and sum,
// the rescale of O^T. masked: cells without a bit in word are dropped. l is of the
// lane's own cells; the quads' add up at the end.
template <int DT>
__device__ __forceinline__ void softmax_q8(f32x4 (&st)[4], float rscale, bool masked, uint64_t word,
                                           float &m, float &l, f32x4 (&o)[DT]) {
#pragma unroll
  for (int ct = 0; ct < 4; ct++)
#pragma unroll
    for (int i = 0; i < 4; i++) st[ct][i] *= rscale;  // (of vectors: the factor would be held four times)
  if (masked) {  // wave-uniform
    word = lane_cells(word);  // s_cell(ct, 4 quad + i) = 8 quad + s_cell(ct, i)
#pragma unroll
    for (int ct = 0; ct < 4; ct++)
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (!(word >> s_cell(ct, i) & 1)) st[ct][i] = -INFINITY;
  }
  float mx = -INFINITY;
#pragma unroll
  for (int ct = 0; ct < 4; ct++)
#pragma unroll
    for (int i = 0; i < 4; i++) mx = fmaxf(mx, st[ct][i]);
  mx = quads_max(mx);
  const float m_new = fmaxf(m, mx);
  const float m_use = m_new == -INFINITY ? 0.0f : m_new;
  float rs = 0.0f;
#pragma unroll
  for (int ct = 0; ct < 4; ct++)
#pragma unroll
    for (int i = 0; i < 4; i++) {
      st[ct][i] = __builtin_amdgcn_exp2f(st[ct][i] - m_use);  // exp2(-inf) = 0
      rs += st[ct][i];
    }
  if (__builtin_amdgcn_ballot_w64(m_new != m)) {
    const float alpha = __builtin_amdgcn_exp2f(m - m_use);
    l *= alpha;
#pragma unroll
    for (int dt = 0; dt < DT; dt++) o[dt] *= alpha;
  }
  l += rs;
  m = m_new;
}

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
// Whether scales go by the packed products: each is 0 or in [2^-12, 2^-2). (Up to
// 2^15 with P's and its own factor; from 2^-12 on a p of 1 keeps 22 bits.)
__device__ __forceinline__ bool plain_range(float low, float high) {
  return high < (float)0x3400 && low >= (float)(0x0c00 - 1);
}
// Whether a lane's 8 scales of a group of 32 dims (the group's 64 in 8 aligned
// lanes) leave the group to the packed products.
__device__ __forceinline__ bool plain_scales(u32x4 sc) {
  return plain_range(-group_max<8>(-low_bits(sc)), group_max<8>(high_bits(sc)));
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
// P of the cells 32 h + 8 quad + e, Q8_P times as large.
__device__ __forceinline__ void split_p(const f32x4 (&st)[4], int h, f16x8 &hi, f16x8 &lo) {
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const f32x4 &s = st[2 * h + (e >> 2)];
    f16x2 a, b;
    split2(s[e & 3] * Q8_P, s[(e & 3) + 1] * Q8_P, a, b);
    hi[e] = a[0];
    hi[e + 1] = a[1];
    lo[e] = b[0];
    lo[e + 1] = b[1];
  }
}
// P dv of those cells times up, or (MASKED) of a plain row as the packed products
// make it. (What other calls make alike is not held for this one: the copies are
// opaque.)
template <bool MASKED>
__device__ __forceinline__ void weigh_p(const f32x4 (&st)[4], int h, f16x8 dv, bool plain, float up, f16x8 &hi,
                                        f16x8 &lo) {
  float q8_p = Q8_P;
  asm volatile("" : "+s"(q8_p), "+v"(dv));
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const float p0 = st[2 * h + (e >> 2)][e & 3], p1 = st[2 * h + (e >> 2)][(e & 3) + 1];
    f16x2 a, b;
    split2(p0 * (float)dv[e] * up, p1 * (float)dv[e + 1] * up, a, b);
    if constexpr (MASKED) {
      f16x2 c, d, ph, pl;
      split2(p0 * q8_p, p1 * q8_p, ph, pl);
      packed_pdv(ph, pl, f16x2{dv[e], dv[e + 1]} * (f16)Q8_DV, c, d);
      a = plain ? c : a;
      b = plain ? d : b;
    }
    hi[e] = a[0];
    hi[e + 1] = a[1];
    lo[e] = b[0];
    lo[e + 1] = b[1];
  }
}

// S^T of a block: read(b, p, k, d) gives the K operands of tiles 2 p and 2 p + 1
// and the lane's cells' dk for block b of dims, query(b, hi, lo) the row's. A step
// reads the next step's operands and issues this one's products, and adds the
// last one's, scaled, while they run. (Two tiles a step: with four, heads of 256
// spill, and each spill is waited for.)
template <int NB, typename R, typename Q>
__device__ __forceinline__ void scores_q8(f32x4 (&st)[4], R read, Q query) {
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

// V's scales as the packed products take them.
__device__ __forceinline__ u32x4 times_dv(u32x4 s) {
  f16x8 v = __builtin_bit_cast(f16x8, s);
  v *= (f16)Q8_DV;
  return __builtin_bit_cast(u32x4, v);
}

// O^T += V^T (P dv)^T over a block. scale(b, h): the lane's cells' dv; frag(t, kc):
// V's operand. plain (the same for the wave): plain_scales of all the block's cells,
// whose scales are Q8_DV times as large here. Which way a row's part is made goes
// by the scales of the cells it sees, and by nothing else, so that a row has the
// same bits in any group of rows: in a plain block all its rows' cells are plain.
template <int D, typename S, typename V>
__device__ __forceinline__ void values_q8(f32x4 (&o)[D / 16], const f32x4 (&st)[4], bool plain,
                                          bool masked, uint64_t word, S scale, V frag) {
  constexpr int NB = D / 32;
  if (plain) {
    // a step reads the next 16 dims' V (and makes the next block's P dv) while
    // the products of this one run
    f16x8 ph[2], pl[2], hi[2], lo[2], v[2][2];
    split_p(st, 0, ph[0], pl[0]);
    split_p(st, 1, ph[1], pl[1]);
    auto fetch = [&](int t) {
#pragma unroll
      for (int kc = 0; kc < 2; kc++) v[t & 1][kc] = frag(t, kc);
    };
    auto weigh = [&](int b) {
#pragma unroll
      for (int h = 0; h < 2; h++) packed_pdv(ph[h], pl[h], __builtin_bit_cast(f16x8, scale(b, h)), hi[h], lo[h]);
    };
    fetch(0);
    weigh(0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int t = 0; t < D / 16; t++) {
#pragma unroll
      for (int kc = 0; kc < 2; kc++) {
        o[t] = mfma16q(v[t & 1][kc], hi[kc], o[t]);
        o[t] = mfma16q(v[t & 1][kc], lo[kc], o[t]);
      }
      if (t + 1 < D / 16) fetch(t + 1);
      if (t % 2 == 1 && t / 2 + 1 < NB) weigh(t / 2 + 1);
      __builtin_amdgcn_sched_barrier(0);
    }
    return;
  }
  auto weighed = [&](auto some_hidden, bool row_plain) __attribute__((always_inline)) {
    constexpr bool MASKED = decltype(some_hidden)::value;
#pragma unroll
    for (int b = 0; b < NB; b++) {
      u32x4 s0 = scale(b, 0), s1 = scale(b, 1);
      if constexpr (MASKED) seen_scales(s0, s1, word);
      const f16x8 dv[2] = {__builtin_bit_cast(f16x8, s0), __builtin_bit_cast(f16x8, s1)};
      const int ex = largest_pdv(st, dv);
      const float up = pow2(15 - ex), back = Q8_O * pow2(ex - 15);
      f32x4 acc[2];
#pragma unroll
      for (int t = 0; t < 2; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[t][i] = row_plain ? o[2 * b + t][i] : 0.0f;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        f16x8 hi, lo;
        weigh_p<MASKED>(st, h, dv[h], row_plain, up, hi, lo);
#pragma unroll
        for (int t = 0; t < 2; t++) {
          const f16x8 v = frag(2 * b + t, h);
          acc[t] = mfma16q(v, hi, acc[t]);
          acc[t] = mfma16q(v, lo, acc[t]);
        }
      }
#pragma unroll
      for (int t = 0; t < 2; t++) {
        f32x4 &ot = o[2 * b + t];
#pragma unroll
        for (int i = 0; i < 4; i++) ot[i] = row_plain ? acc[t][i] : fmaf(acc[t][i], back, ot[i]);
        here(ot);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  if (!masked) {  // wave-uniform: all rows see all of the block, none is plain
    weighed(std::false_type{}, false);
    return;
  }
  // each row takes its own way
  float low = 65535.0f, high = 0.0f;
#pragma unroll 1
  for (int b = 0; b < NB; b++) {
    u32x4 s0 = scale(b, 0), s1 = scale(b, 1);
    seen_scales(s0, s1, word);
    low = fminf(low, fminf(low_bits(s0), low_bits(s1)));
    high = fmaxf(high, fmaxf(high_bits(s0), high_bits(s1)));
  }
  weighed(std::true_type{}, plain_range(-quads_max(-low), quads_max(high)));
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

template <int D>
__global__ void __launch_bounds__(64, D <= 128 ? 2 : 1)
paged_attn_q8_kernel(const float *__restrict__ q, int H, int Hkv, float scale_log2,
                     const uint8_t *__restrict__ kpool, const uint8_t *__restrict__ vpool,
                     const int32_t *__restrict__ items, const int32_t *__restrict__ seq_off,
                     const int32_t *__restrict__ seq_npast, const int32_t *__restrict__ block_tab,
                     int max_blocks, int ring, int window, float *__restrict__ out,
                     f16 *__restrict__ planes, int64_t npad, int xf, float *__restrict__ part,
                     const int32_t *__restrict__ order, int n_order,
                     const uint64_t *__restrict__ vis) {
  typedef Q8Frag<D> F;
  constexpr int NB = F::NB, J = F::J, DT = F::DT;
  __shared__ __align__(16) f16x8 qsh[NB * 64], qsl[NB * 64];
  const int lane = threadIdx.x;
  const int slot = (int)(blockIdx.x / (uint32_t)Hkv), kvh = (int)(blockIdx.x % (uint32_t)Hkv);
  const int item = slot < n_order ? order[slot] : slot;
  const int G = H / Hkv;
  const int s = items[4 * item + 0], tok0 = items[4 * item + 1];
  const int ntok = items[4 * item + 2] & 31, mg = (items[4 * item + 2] >> 5) - 1;
  const int blo = items[4 * item + 3] & 0xffff, bhi = (items[4 * item + 3] >> 16) & 0xffff;
  const int npast = seq_npast[s];
  Sight see;
  see.ring = ring;
  see.window = window;
  see.p_first = npast + (tok0 - seq_off[s]);
  see.p_last = see.p_first + ntok - 1;
  see.b_tree = npast / KV_BLOCK;
  see.G = G;
  see.ntok = ntok;
  see.vis = ring < 0 ? vis + (int64_t)tok0 * window : nullptr;

  const int32_t *bt = block_tab + (int64_t)s * max_blocks;
  auto tile = [&](const uint8_t *pool, int blk) {
    const int64_t b = ring > 0 ? bt[blk % ring] : bt[blk];
    return pool + (b * Hkv + kvh) * (int64_t)F::TILE;
  };
  // A block's values in registers, a lane's place in a tile being the same in
  // all (the tile's own address stays scalar). Its scales come 16 bytes a lane and
  // go through LDS: in registers they are 16 lanes' copies, as many as the values.
  constexpr int SR = D > 128 ? 2 : 1;    // registers' worth: K's and V's, or K's then V's
  constexpr int SL = D > 128 ? 64 : NB * 8;  // lanes of K's scales
  u32x4 kq[4][J], vq[DT], sreg[SR];
  const int row = lane & 15, quad = lane >> 4;
  const uint32_t koff = (8 * (row >> 2) + (row & 3)) * 64 + quad * 16, voff = row * 64 + quad * 16;
  auto load_k = [&](int blk) {
    const uint8_t *t = tile(kpool, blk);
#pragma unroll
    for (int ct = 0; ct < 4; ct++)
#pragma unroll
      for (int j = 0; j < J; j++)
        kq[ct][j] = *(const u32x4 *)(t + (j * 4096 + s_cell(ct, 0) * 64) + koff);
  };
  auto load_v = [&](int blk) {
    const uint8_t *t = tile(vpool, blk);
#pragma unroll
    for (int dt = 0; dt < DT; dt++) vq[dt] = *(const u32x4 *)(t + dt * 1024 + voff);
  };
  auto load_s = [&](int blk) {
    const uint8_t *k = tile(kpool, blk) + 64 * D, *v = tile(vpool, blk) + 64 * D;
    if constexpr (SR == 2) {
      sreg[0] = *(const u32x4 *)(k + lane * 16u);
      sreg[1] = *(const u32x4 *)(v + lane * 16u);
    } else {
      sreg[0] = *(const u32x4 *)((lane < SL ? k : v) + lane % SL * 16u);
    }
  };
  __shared__ __align__(16) u32x4 scl[SR * 64];  // K's scales, then V's
  auto store_s = [&](bool plain) {
    if (SR == 2) scl[lane] = sreg[0];
    u32x4 v = sreg[SR - 1];
    if (plain && (SR == 2 || lane >= SL)) v = times_dv(v);
    scl[(SR - 1) * 64 + lane] = v;
  };
  auto scale_of = [&](int v, int b, int h) { return scl[v * SL + b * 8 + h * 4 + quad]; };
  float rscale;
  {
    const RowOf r(lane, G, ntok);
    const float *qr = q + ((int64_t)(tok0 + (r.valid ? r.rtok : ntok - 1)) * H + kvh * G + r.head) * D;
    f32x4 qa[2 * NB];
#pragma unroll
    for (int b = 0; b < NB; b++) {
      qa[2 * b] = *(const f32x4 *)(qr + 32 * b + 8 * r.quad);
      qa[2 * b + 1] = *(const f32x4 *)(qr + 32 * b + 8 * r.quad + 4);
    }
    const int b_first = blo < bhi ? blo : 0;  // block 0 of a planned sequence is a pool block
    load_s(b_first);
    load_k(b_first);
    load_v(b_first);
    f16x8 hi[NB], lo[NB];
    rscale = split_q<NB>(qa, r.valid, scale_log2, hi, lo);
#pragma unroll
    for (int b = 0; b < NB; b++) {
      qsh[b * 64 + lane] = hi[b];
      qsl[b * 64 + lane] = lo[b];
    }
  }
  f32x4 o[DT];
#pragma unroll
  for (int i = 0; i < DT; i++) o[i] = f32x4{0, 0, 0, 0};
  float m = -INFINITY, l = 0.0f;

  auto block = [&](int blk, auto next) __attribute__((always_inline)) {
    constexpr bool NEXT = decltype(next)::value;
    const int nxt = blk + 1 < bhi ? blk + 1 : blk;
    f32x4 st[4];
    int ql_at = lane;
    asm volatile("" : "+v"(ql_at));  // Q's operands are read anew: held, they spill others
    // (the lanes of K's scales have no part in this)
    const bool plain = !__builtin_amdgcn_ballot_w64(!plain_scales(sreg[SR - 1]) &&
                                                    (SR == 2 || (lane >= SL && lane < 2 * SL)));
    store_s(plain);
    if constexpr (NEXT) load_s(nxt);
    scores_q8<NB>(
        st,
        [&](int b, int p, f16x8(&k)[2], f16x8 &d) {
#pragma unroll
          for (int t = 0; t < 2; t++) {
            const u32x4 w = kq[2 * p + t][b / 2];
            k[t] = half8(w[2 * (b & 1)], w[2 * (b & 1) + 1]);
          }
          d = __builtin_bit_cast(f16x8, scale_of(0, b, p));
        },
        [&](int b, f16x8 &hi, f16x8 &lo) {
          hi = qsh[b * 64 + ql_at];
          lo = qsl[b * 64 + ql_at];
        });
    if constexpr (NEXT) load_k(nxt);
    uint64_t word = ~(uint64_t)0;
    const bool masked = see.masks(blk, word);
    softmax_q8<DT>(st, rscale, masked, word, m, l, o);
    __builtin_amdgcn_sched_barrier(0);
    values_q8<D>(o, st, plain, masked, word,
                 [&](int b, int h) { return scale_of(1, b, h); },
                 [&](int t, int kc) { return half8(vq[t][2 * kc], vq[t][2 * kc + 1]); });
    if constexpr (NEXT) load_v(nxt);
  };
  for (int blk = blo; blk + 1 < bhi; blk++) block(blk, std::true_type{});
  if (blo < bhi) block(bhi - 1, std::false_type{});
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  const RowOf r(lane_anew(), G, ntok);
  finish_item<D>(o, m, l * Q8_O, mg, r.valid, tok0, r.rtok, kvh * G + r.head, ntok, G, r.row, r.quad, item, kvh, Hkv,
                 H, out, planes, npad, xf, part);
}

// Shared runs (a chunk's or a tree's query groups in sets): a workgroup of W waves
// per (run, KV head), wave w on the run's item w of a half of the set (W = 4) or
// of the whole (W = 8). Each block is loaded once, 16 bytes a lane, made f16 on its
// way into LDS, and read from there by every wave, whose arithmetic is the
// per-item kernel's: an item gives the same bits in either. The next block's
// bytes are in flight while this one is used. Two buffers take one barrier a
// block; where two workgroups of one buffer each share a CU (heads of 256, W =
// 4) there are two. LDS slots of 16 B: K slot (cell, c) holds dims 8 (c ^ swk), V
// slot (d, c) cells 8 (c ^ swv): a fragment's 16 rows touch every bank once.
template <int D, int W>
__global__ void __launch_bounds__(64 * W, 2)
paged_attn_q8_shared_kernel(const float *__restrict__ q, int H, int Hkv, float scale_log2,
                            const uint8_t *__restrict__ kpool, const uint8_t *__restrict__ vpool,
                            const int32_t *__restrict__ items, const int32_t *__restrict__ shared,
                            const int32_t *__restrict__ seq_off,
                            const int32_t *__restrict__ seq_npast,
                            const int32_t *__restrict__ block_tab, int max_blocks, int ring,
                            int window, float *__restrict__ out, f16 *__restrict__ planes,
                            int64_t npad, int xf, float *__restrict__ part,
                            const uint64_t *__restrict__ vis) {
  typedef Q8Frag<D> F;
  constexpr int NB = F::NB, DT = F::DT, KC = D / 8;
  constexpr int CH = D / (8 * W);           // 16-byte pieces a thread: K's 4 D, then V's
  constexpr int BUFS = D == 256 && W == 4 ? 1 : 2;
  constexpr int TILE = 64 * D;              // f16 of a tile
  __shared__ __align__(16) f16 kb[BUFS][TILE], vb[BUFS][TILE];
  __shared__ __align__(16) u32x4 scl[BUFS][2 * NB * 8];  // K's scales, then V's
  __shared__ int odd_scales[BUFS];  // some of V's are not plain_scales

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = W < SHARED_MAX ? (int)blockIdx.z * W : 0;
  const int first = shared[2 * blockIdx.x] + half, n = shared[2 * blockIdx.x + 1] - half;
  if (n <= 0) return;  // a set of one half
  const int kvh = blockIdx.y;
  const int G = H / Hkv;
  const bool active = wave < n;
  const int item = first + (active ? wave : 0);
  const int s = items[4 * first + 0];
  const int blo = items[4 * first + 3] & 0xffff, bhi = (items[4 * first + 3] >> 16) & 0xffff;
  const int tok0 = items[4 * item + 1];
  const int ntok = items[4 * item + 2] & 31, mg = (items[4 * item + 2] >> 5) - 1;
  const int npast = seq_npast[s];
  Sight see;
  see.ring = ring;
  see.window = window;
  see.p_first = npast + (tok0 - seq_off[s]);
  see.p_last = see.p_first + ntok - 1;
  see.b_tree = npast / KV_BLOCK;
  see.G = G;
  see.ntok = ntok;
  see.vis = ring < 0 ? vis + (int64_t)tok0 * window : nullptr;

  const int32_t *bt = block_tab + (int64_t)s * max_blocks;
  u32x4 raw[CH], sraw;
  // (a thread's places are made anew each block, from an opaque copy of its number:
  // held over the loop they are a dozen registers, and heads of 256 have none)
  auto load = [&](int blk) {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const int64_t at = ((int64_t)bt[blk] * Hkv + kvh) * F::TILE;
#pragma unroll
    for (int i = 0; i < CH; i++) {
      const int c = i * 64 * W + tid;  // a wave's pieces are K's or V's
      raw[i] = i * 64 * W + 64 * wave < 4 * D ? *(const u32x4 *)(kpool + at + c * 16u)
                                              : *(const u32x4 *)(vpool + at + (c - 4 * D) * 16u);
    }
    if (tid < NB * 16)
      sraw = *(const u32x4 *)((tid < NB * 8 ? kpool : vpool) + at + 64 * D + tid % (NB * 8) * 16u);
  };
  auto store = [&](int buf) {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
#pragma unroll
    for (int i = 0; i < CH; i++) {
      const int c = i * 64 * W + tid;
      const f16x8 lo = half8(raw[i][0], raw[i][1]), hi = half8(raw[i][2], raw[i][3]);
      if (i * 64 * W + 64 * wave < 4 * D) {  // (j, cell, quad): dims of blocks 2 j and 2 j + 1
        const int j = c >> 8, cell = c >> 2 & 63, qd = c & 3;
        *(f16x8 *)(kb[buf] + (cell * KC + ((8 * j + qd) ^ swk<D>(cell))) * 8) = lo;
        *(f16x8 *)(kb[buf] + (cell * KC + ((8 * j + 4 + qd) ^ swk<D>(cell))) * 8) = hi;
      } else {  // (d, quad): cells 8 quad .. and 32 + 8 quad ..
        const int d = (c - 4 * D) >> 2, qd = c & 3;
        *(f16x8 *)(vb[buf] + (d * 8 + (qd ^ swv(d))) * 8) = lo;
        *(f16x8 *)(vb[buf] + (d * 8 + ((4 + qd) ^ swv(d))) * 8) = hi;
      }
    }
    // V's scales are in one wave (NB * 8 lanes from lane NB * 8 on)
    bool plain = false;
    if (wave == NB * 8 / 64) {
      const bool odd = !plain_scales(sraw) && tid >= NB * 8 && tid < NB * 16;
      plain = __builtin_amdgcn_ballot_w64(odd) == 0;
      if (lane == 0) odd_scales[buf] = !plain;
    }
    if (tid < NB * 16) scl[buf][tid] = plain && tid >= NB * 8 ? times_dv(sraw) : sraw;
  };
  if (blo < bhi) load(blo);
  // Q's operands in registers, but for the last block of dims of heads of 256 (LDS)
  constexpr int QR = D == 256 ? NB - 1 : NB;
  __shared__ f16x8 q_last[D == 256 ? 2 * 64 * W : 1];
  f16x8 qh[NB], ql[NB];
  float rscale;
  {
    const RowOf r(lane, G, ntok);
    const float *qr = q + ((int64_t)(tok0 + (r.valid ? r.rtok : ntok - 1)) * H + kvh * G + r.head) * D;
    f32x4 qa[2 * NB];
#pragma unroll
    for (int b = 0; b < NB; b++) {
      qa[2 * b] = *(const f32x4 *)(qr + 32 * b + 8 * r.quad);
      qa[2 * b + 1] = *(const f32x4 *)(qr + 32 * b + 8 * r.quad + 4);
    }
    rscale = split_q<NB>(qa, r.valid, scale_log2, qh, ql);
    if constexpr (QR < NB) {  // read by the lane that writes it
      q_last[tid] = qh[QR];
      q_last[64 * W + tid] = ql[QR];
    }
  }
  f32x4 o[DT];
#pragma unroll
  for (int i = 0; i < DT; i++) o[i] = f32x4{0, 0, 0, 0};
  float m = -INFINITY, l = 0.0f;

  // A lane's places in the tiles: the swizzles take from the cell and from d what
  // only the lane's row decides, and from a block of dims its two low bits. The
  // rest of an address is constant.
  constexpr int KB = NB < 4 ? NB : 4;

  for (int blk = blo; blk < bhi; blk++) {
    const int buf = BUFS == 2 ? (blk - blo) & 1 : 0;
    if (BUFS == 1 && blk > blo) lds_sync();  // everyone is done with the buffer
    store(buf);
    if (blk + 1 < bhi) load(blk + 1);
    lds_sync();
    if (!active || blk * 64 > see.p_last) continue;
    // places in this buffer, made here from an opaque copy of the lane: otherwise every
    // fragment's address is made ahead of the loop and takes a register
    int at = lane;
    asm volatile("" : "+v"(at));
    const int arow = at & 15, aquad = at >> 4, r0 = s_cell(0, arow);
    int ka[KB], va[2], sa = buf * (2 * NB * 8) + aquad;
#pragma unroll
    for (int b = 0; b < KB; b++) {
      ka[b] = buf * TILE + (r0 * KC + ((b * 4 + aquad) ^ swk<D>(r0))) * 8;
      asm volatile("" : "+v"(ka[b]));
    }
#pragma unroll
    for (int kc = 0; kc < 2; kc++) {
      va[kc] = buf * TILE + (arow * 8 + ((kc * 4 + aquad) ^ swv(arow))) * 8;
      asm volatile("" : "+v"(va[kc]));
    }
    asm volatile("" : "+v"(sa));
    const u32x4 *sc = scl[0] + sa;
    f32x4 st[4];
    scores_q8<NB>(
        st,
        [&](int b, int p, f16x8(&k)[2], f16x8 &d) {
#pragma unroll
          for (int t = 0; t < 2; t++)
            k[t] = *(const f16x8 *)(kb[0] + ka[b % KB] + (s_cell(2 * p + t, 0) * KC + b / 4 * 16) * 8);
          d = __builtin_bit_cast(f16x8, sc[b * 8 + 4 * p]);
        },
        [&](int b, f16x8 &hi, f16x8 &lo) {
          hi = b < QR ? qh[b] : q_last[64 * wave + at];
          lo = b < QR ? ql[b] : q_last[64 * (W + wave) + at];
        });
    uint64_t word = ~(uint64_t)0;
    const bool masked = see.masks(blk, word);
    softmax_q8<DT>(st, rscale, masked, word, m, l, o);
    __builtin_amdgcn_sched_barrier(0);
    values_q8<D>(o, st, odd_scales[buf] == 0, masked, word,
                 [&](int b, int h) { return sc[NB * 8 + b * 8 + 4 * h]; },
                 [&](int t, int kc) { return *(const f16x8 *)(vb[0] + va[kc] + t * 1024); });
  }
  if (!active) return;
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  const RowOf r(lane_anew(), G, ntok);
  finish_item<D>(o, m, l * Q8_O, mg, r.valid, tok0, r.rtok, kvh * G + r.head, ntok, G, r.row, r.quad, item, kvh, Hkv,
                 H, out, planes, npad, xf, part);
}

template <int D>
static void launch_attn_q8(const float *q, int H, int Hkv, float scale_log2, const void *kp,
                           const void *vp, const lgmlh_ubatch *ub, float *out, f16 *planes,
                           int64_t npad, int xf, float *part, hipStream_t st) {
  const uint64_t *vis =
      ub->ring == LGMLH_PLAN_TREE ? plan_vis(ub) : nullptr;
  if (ub->n_single > 0)
    hipLaunchKernelGGL(paged_attn_q8_kernel<D>, dim3((uint32_t)ub->n_single * Hkv), dim3(64), 0, st,
                       q, H, Hkv, scale_log2, (const uint8_t *)kp, (const uint8_t *)vp, ub->items,
                       ub->seq_off, ub->seq_npast, ub->block_tab, ub->max_blocks, ub->ring,
                       ub->window, out, planes, npad, xf, part, ub->order,
                       ub->order ? ub->n_single : 0, vis);
  if (ub->n_shared > 0) {
    // sets of up to half a workgroup's waves on average: workgroups of half as many
    const bool small = ub->n_items - ub->n_single <= SHARED_MAX / 2 * ub->n_shared;
    const auto kern = small ? paged_attn_q8_shared_kernel<D, SHARED_MAX / 2>
                            : paged_attn_q8_shared_kernel<D, SHARED_MAX>;
    hipLaunchKernelGGL(kern, dim3(ub->n_shared, Hkv, small ? 2 : 1),
                       dim3(64 * (small ? SHARED_MAX / 2 : SHARED_MAX)), 0, st, q, H, Hkv, scale_log2,
                       (const uint8_t *)kp, (const uint8_t *)vp, ub->items, ub->shared, ub->seq_off,
                       ub->seq_npast, ub->block_tab, ub->max_blocks, ub->ring, ub->window, out,
                       planes, npad, xf, part, vis);
  }
  merge_dev(D, ub, H, Hkv, part, out, planes, npad, xf, st);
}

// paged_attention_dev over Q8_0 pools.
int paged_attention_q8_dev(const float *q, int n_head, int n_head_kv, int head_dim, float scale,
                           const void *kpool, const void *vpool, const lgmlh_ubatch *ub, float *out,
                           f16 *planes, int64_t npad, void *workspace, size_t workspace_bytes,
                           hipStream_t st, int xf) {
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) {
    set_error("paged_attention_q8: head_dim %d not supported (64, 128, 256)", head_dim);
    return LGMLH_EINVAL;
  }
  if (((uintptr_t)kpool | (uintptr_t)vpool) & 15) {
    set_error("paged_attention_q8: pools are 16-byte aligned");
    return LGMLH_EINVAL;
  }
  int run = 0;
  LGMLH_TRY(attn_check("paged_attention_q8", q, n_head, n_head_kv, head_dim, kpool, vpool, ub, out,
                       planes, xf, workspace, workspace_bytes, &run));
  if (!run) return LGMLH_OK;
  const float sl = scale * LOG2E;
  float *part = (float *)workspace;
  switch (head_dim) {
    case 64: launch_attn_q8<64>(q, n_head, n_head_kv, sl, kpool, vpool, ub, out, planes, npad, xf, part, st); break;
    case 128: launch_attn_q8<128>(q, n_head, n_head_kv, sl, kpool, vpool, ub, out, planes, npad, xf, part, st); break;
    default: launch_attn_q8<256>(q, n_head, n_head_kv, sl, kpool, vpool, ub, out, planes, npad, xf, part, st); break;
  }
  return hip_check(hipGetLastError(), "paged_attention_q8");
}

}  // namespace lgmlh

using namespace lgmlh;

extern "C" int lgmlh_paged_attention_q8(const float *q, int n_head, int n_head_kv, int head_dim,
                                        float scale, const void *kpool, const void *vpool,
                                        const lgmlh_ubatch *ub, float *out, void *workspace,
                                        size_t workspace_bytes, void *stream) {
  if (!out) {
    set_error("paged_attention_q8: bad arguments");
    return LGMLH_EINVAL;
  }
  return paged_attention_q8_dev(q, n_head, n_head_kv, head_dim, scale, kpool, vpool, ub, out,
                                nullptr, 0, workspace, workspace_bytes, as_stream(stream), XF_SPLIT);
}
