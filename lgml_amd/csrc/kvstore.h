// Rows of f32 into the cells of a KV pool of any type: rounding 8 values of a row, and
// V's turn from rows into tiles.
#pragma once

#include "kvq4.h"
#include "kvq8.h"
#include "kvwindow.h"

namespace lgmlh {

constexpr int KV_THREADS = 256;

__host__ __device__ constexpr int kv_tile_bytes(int type, int D) {
  return type == LGMLH_Q8_0 ? q8_tile_bytes(D) : type == LGMLH_Q4_0 ? q4_tile_bytes(D) : 128 * D;
}
// The tile of cell c (>= 0) of one head: head is the first block's. (The bytes of a
// block are counted in 31 bits.)
template <int TYPE, int D, typename P>
__device__ __forceinline__ P *kv_tile(P *head, int64_t c, int Hkv) {
  return head + (uint64_t)(uint32_t)((uint64_t)c >> 6) * (uint32_t)(Hkv * kv_tile_bytes(TYPE, D));
}

// 8 values of a row, the 4 lanes of a block of 32 together, in the format's steps (f32);
// returns the block's d. Q8_0: d = max |x| / 127, q = x (1 / d) rounded with halves away
// from zero. Q4_0: m the value of largest size (the first of them), d = m / -8, n =
// min(15, trunc(x (1 / d) + 8.5)).
template <int TYPE>
__device__ __forceinline__ float quant8(const float (&v)[8], uint32_t (&q)[8]) {
  float amax = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; e++) amax = fmaxf(amax, fabsf(v[e]));
  amax = group_max<4>(amax);
  const float d = TYPE == LGMLH_Q8_0 ? amax / 127.0f : group_first_abs<4>(v, amax) * -0.125f;
  const float id = d != 0.0f ? 1.0f / d : 0.0f;
#pragma unroll
  for (int e = 0; e < 8; e++) q[e] = TYPE == LGMLH_Q8_0 ? (uint32_t)round_away(v[e], id) & 0xff : q4_round(v[e], id);
  return d;
}
__device__ __forceinline__ uint32_t q4_k_word(const uint32_t (&q)[8]) {
  uint32_t w = 0;
#pragma unroll
  for (int e = 0; e < 8; e++) w |= q[e] << (4 * (e / 2) + 16 * (e % 2));
  return w;
}
__device__ __forceinline__ uint32_t bytes4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return a | b << 8 | c << 16 | d << 24;
}

// V of W consecutive tokens of one head, from rows into tiles by way of LDS: 8 values a
// thread and step, then 8 tokens whose cells are 8 in a row from a multiple of 8 on (a
// whole group) are 8 values in a row of each dim (of Q4_0: of each byte's pair of dims);
// tokens in no whole group go value by value. A group belongs to the window that has
// its first token, which also takes the up to 7 of it that lie past its own.
template <int TYPE, int D, int W>
struct VTurn {
  typedef typename std::conditional<TYPE == LGMLH_F16, uint16_t, uint8_t>::type T;
  static constexpr int LINES = TYPE == LGMLH_Q4_0 ? D / 2 : D;  // of a tile, 64 cells each
  static constexpr int PAD = LINES + 4 / (int)sizeof(T), ROWS = W + CELL_HALO, GROUPS = W / CELL_GROUP;
  static constexpr int G8 = D / 8, STEP = KV_THREADS / G8, IT = (ROWS + STEP - 1) / STEP;
  CellWindow<W> win;
  alignas(4) T turn[ROWS * PAD];
  uint16_t scale[TYPE == LGMLH_F16 ? 1 : D / 32 * W];

  // A cell's place in a line, and the place of cell e of 8 among a group's values.
  __device__ __forceinline__ static int cell_at(int cell) {
    return TYPE == LGMLH_F16 ? cell : TYPE == LGMLH_Q8_0 ? q8_v_at(0, cell) : q4_v_at(0, cell);
  }
  __device__ __forceinline__ static constexpr int place(int e) {
    return TYPE == LGMLH_Q4_0 ? (e & 4) | (e & 1) << 1 | (e >> 1 & 1) : e;
  }
  // All threads of a workgroup of KV_THREADS. src: the head's values of token j0, rows
  // `stride` apart; pool: the tensor.
  __device__ __forceinline__ void store(const float *__restrict__ src, int64_t stride, uint8_t *__restrict__ pool,
                                        int h, int Hkv, const int64_t *__restrict__ cells, int64_t j0, int64_t n,
                                        int64_t n_cells) {
    const int tid = threadIdx.x, g8 = tid % G8, t0 = tid / G8;
    const int left = (int)(n - j0 < ROWS ? n - j0 : ROWS);
    uint8_t *head = pool + (int64_t)h * kv_tile_bytes(TYPE, D);
    f32x4 x[IT][2];
#pragma unroll
    for (int i = 0; i < IT; i++) {
      const int t = t0 + i * STEP;
      const float *row = src + t * stride + 8 * g8;
      x[i][0] = t < left ? *(const f32x4_u *)row : f32x4{0, 0, 0, 0};
      x[i][1] = t < left ? *(const f32x4_u *)(row + 4) : f32x4{0, 0, 0, 0};
    }
    win.fill(cells, j0, n, n_cells, true);
#pragma unroll
    for (int i = 0; i < IT; i++) {
      const int t = t0 + i * STEP;
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] = x[i][e >> 2][e & 3];
      if constexpr (TYPE == LGMLH_F16) {
        if (t < left)
#pragma unroll
          for (int e = 0; e < 8; e += 2)
            *(uint32_t *)(turn + t * PAD + 8 * g8 + e) = f2h(v[e]) | (uint32_t)f2h(v[e + 1]) << 16;
      } else {
        uint32_t q[8];
        const float d = quant8<TYPE>(v, q);
        uint32_t lo = bytes4(q[0], q[1], q[2], q[3]), hi = bytes4(q[4], q[5], q[6], q[7]);
        int line = 8 * g8;
        bool mine = t < left;
        if constexpr (TYPE == LGMLH_Q4_0) {
          // the lanes of a block's first 16 dims take the bytes with their partners' dims
          lo |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)lo, DPP_XOR2, 0xF, 0xF, false) << 4;
          hi |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)hi, DPP_XOR2, 0xF, 0xF, false) << 4;
          line = g8 / 4 * 16 + g8 % 4 * 8;
          mine &= g8 % 4 < 2;
        }
        if (g8 % 4 == 0 && t < left && t < W) scale[g8 / 4 * W + t] = f2h(d);
        if (mine) {
          *(uint32_t *)(turn + t * PAD + line) = lo;
          *(uint32_t *)(turn + t * PAD + line + 4) = hi;
        }
      }
    }
    __syncthreads();
    if constexpr (TYPE != LGMLH_F16)  // the scales with tokens along the lanes, as a tile has them
      for (int i = tid; i < D / 32 * W; i += KV_THREADS) {
        const int64_t c = win.cell(i % W);
        const int at = TYPE == LGMLH_Q8_0 ? q8_scale_at(D, i / W, (int)c & 63) : q4_scale_at(D, i / W, (int)c & 63);
        if (c >= 0) *(uint16_t *)(kv_tile<TYPE, D>(head, c, Hkv) + at) = scale[i];
      }
    // a thread's group or lone token is the same in every step
    if (const int g = tid % GROUPS; g < win.n_lead) {
      const int t = win.lead[g];
      const int64_t c = win.cell(t);
      T *tile = (T *)kv_tile<TYPE, D>(head, c, Hkv) + cell_at((int)c & 63);
#pragma unroll 4
      for (int p = tid / GROUPS; p < LINES; p += KV_THREADS / GROUPS) {
        const T *s = turn + t * PAD + p;
        uint32_t q[2 * sizeof(T)] = {};
        constexpr int BITS = 8 * sizeof(T), IN = 32 / BITS;
#pragma unroll
        for (int e = 0; e < 8; e++) q[place(e) / IN] |= (uint32_t)s[e * PAD] << BITS * (place(e) % IN);
        if constexpr (TYPE == LGMLH_F16)
          *(u32x4 *)(tile + 64 * p) = u32x4{q[0], q[1], q[2], q[3]};
        else
          *(u32x2 *)(tile + 64 * p) = u32x2{q[0], q[1]};
      }
    }
    const int no = win.n_lone, sh = lone_bits(no);
    if (const int k = tid & ((1 << sh) - 1); k < no) {
      const int t = win.lone[k];
      const int64_t c = win.cell(t);
      T *tile = (T *)kv_tile<TYPE, D>(head, c, Hkv) + cell_at((int)c & 63);
#pragma unroll 8
      for (int p = tid >> sh; p < LINES; p += KV_THREADS >> sh) tile[64 * p] = turn[t * PAD + p];
    }
  }
};

}  // namespace lgmlh
