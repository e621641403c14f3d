// What the attention kernels over 64-cell KV blocks share: the rows of a wave,
// the order of a block's cells in its MFMA tiles, and the end of a work item.
#pragma once

#include <math.h>

#include "common.h"
#include "split.h"

namespace lgmlh {

constexpr int ROWS = 16;      // MFMA rows per wave
constexpr float LOG2E = 1.4426950408889634f;
constexpr float ATTN_P = 32768.0f;  // the scale of P

__device__ __forceinline__ f32x4 mfma16(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ f16x8 load_f16x8(const uint16_t *p) {
  return __builtin_bit_cast(f16x8, *(const u32x4 *)p);
}

// The cells of the S^T tiles. MFMA row r of tile ct is cell 32 (ct / 2) + 8 (r /
// 4) + 4 (ct % 2) + r % 4 of the block: the 4 values that lane quad q holds of
// tiles 2j and 2j + 1 are then cells 32 j + 8 q .. + 7, the B operand of the
// second product over the V^T tile's own order of cells, and P never leaves
// the registers. (With P through LDS and K and V fragments read as they were
// needed, a 512-token chunk after 1024 tokens, 32 / 8 heads of 128, took 65.7
// us; 59.6 here. 300 tokens beside 16 sequences, 8 / 4 heads of 64: 42.0 and
// 34.6.)
__device__ __forceinline__ int s_cell(int ct, int r) {
  return 32 * (ct >> 1) + 8 * (r >> 2) + 4 * (ct & 1) + (r & 3);
}

// Partial state of one (item, kv head): O^T rows then m, l per row.
template <int D>
struct Partial {
  static constexpr int floats = ROWS * D + 2 * ROWS;
};

// The Q8_K blocks of the output product's X (ggml's arithmetic) from the
// rows of an item in one run: a block (256 values) is 256 / D heads of one
// token, rows row .. of one row group and all four quads: value
// (row % HB) D + 16 dt + 4 quad + i of the block. The same steps as
// q8k_block8 (largest |x| and its first occurrence, iscale = -127 / max,
// q = min(127, nearest-even(iscale x)), d = 1 / iscale, the 16 sums of 16
// q); every lane takes part in the reductions, lanes of rows past the
// item's store nothing.
template <int D>
__device__ __forceinline__ void finish_q8k(const f32x4 (&o)[D / 16], float l, bool rvalid,
                                           int64_t n, int rhead, int H, int row, int quad,
                                           f16 *__restrict__ planes, int64_t npad) {
  constexpr int DT = D / 16, HB = 256 / D;
  const int64_t K = (int64_t)H * D;
  f32x4 y[DT];
  float amax = 0.0f, mx = 0.0f;
  int at = 1 << 30;
  const int kb = (row % HB) * D + quad * 4;
#pragma unroll
  for (int dt = 0; dt < DT; dt++) {
    y[dt] = o[dt] / l;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float a = fabsf(y[dt][i]);
      if (a > amax) {
        amax = a;
        mx = y[dt][i];
        at = kb + dt * 16 + i;
      }
    }
  }
#pragma unroll
  for (int s = 1; s < HB; s <<= 1) q8k_amax_step(amax, mx, at, s);
  q8k_amax_step(amax, mx, at, 16);
  q8k_amax_step(amax, mx, at, 32);
  const float iscale = amax == 0.0f ? 0.0f : -127.0f / mx;
  const int64_t col = (int64_t)rhead * D + quad * 4;
  f16 *qrow = planes + n * K;
  f16 *bsrow = planes + q8_bs_off(npad, K) + n * (K / 16);
#pragma unroll
  for (int dt = 0; dt < DT; dt++) {
    float qv[4], s = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      qv[i] = amax == 0.0f ? 0.0f : fminf(127.0f, __builtin_rintf(iscale * y[dt][i]));
      s += qv[i];
    }
    s += __shfl_xor(s, 16);
    s += __shfl_xor(s, 32);
    if (rvalid) {
      *(f16x4 *)(qrow + col + dt * 16) = f16x4{(f16)qv[0], (f16)qv[1], (f16)qv[2], (f16)qv[3]};
      if (quad == 0) bsrow[(col + dt * 16) >> 4] = (f16)s;
    }
  }
  if (rvalid && quad == 0 && row % HB == 0) {
    float *dp = (float *)((char *)planes + q8_d_off(npad, K));
    dp[n * (K / 256) + (int64_t)rhead * D / 256] = amax == 0.0f ? 0.0f : 1.0f / iscale;
  }
}

// The Q8_0 blocks of the output product's X (ggml's arithmetic, a Q8_0
// output matrix) from the rows of an item in one run: block g of a head is
// its d tiles 2g and 2g + 1, held by the row's four quads; the steps of
// q80_block8 (d = amax / 127, q = roundf(x / d), d kept as f16).
template <int D>
__device__ __forceinline__ void finish_q80(const f32x4 (&o)[D / 16], float l, bool rvalid,
                                           int64_t n, int rhead, int H, int quad,
                                           f16 *__restrict__ planes, int64_t npad) {
  constexpr int DT = D / 16;
  const int64_t K = (int64_t)H * D;
  float *dp = (float *)((char *)planes + q8_d_off(npad, K));
#pragma unroll
  for (int g = 0; g < DT / 2; g++) {
    const f32x4 y0 = o[2 * g] / l, y1 = o[2 * g + 1] / l;
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; i++) amax = fmaxf(amax, fmaxf(fabsf(y0[i]), fabsf(y1[i])));
    amax = fmaxf(amax, __shfl_xor(amax, 16));
    amax = fmaxf(amax, __shfl_xor(amax, 32));
    const float dd = amax / 127.0f;
    const float id = dd != 0.0f ? 1.0f / dd : 0.0f;
    if (rvalid) {
      const int64_t col = (int64_t)rhead * D + 32 * g + quad * 4;
      f16x4 h0, h1;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        h0[i] = (f16)__builtin_roundf(y0[i] * id);
        h1[i] = (f16)__builtin_roundf(y1[i] * id);
      }
      *(f16x4 *)(planes + n * K + col) = h0;
      *(f16x4 *)(planes + n * K + col + 16) = h1;
      if (quad == 0) dp[n * (K / 32) + (col >> 5)] = (float)(f16)dd;
    }
  }
}

// The end of a work item: lane holds O^T[d = dt*16 + quad*4 + i][row].
// A group in one run writes o / l (as the merge divides: a token's output
// does not depend on whether its group was split) to out or, with planes,
// to the output product's X in the form xf (split planes, or Q8_K blocks);
// a run of a split group writes its partial state (rows in use only) for
// the merge.
template <int D>
__device__ __forceinline__ void finish_item(const f32x4 (&o)[D / 16], float m, float l, int mg,
                                            bool rvalid, int tok0, int rtok, int rhead, int ntok,
                                            int G, int row, int quad, int item, int kvh, int Hkv,
                                            int H, float *__restrict__ out,
                                            f16 *__restrict__ planes, int64_t npad, int xf,
                                            float *__restrict__ part) {
  constexpr int DT = D / 16;
  if (mg < 0) {
    if constexpr (D >= 64) {
      if (planes && xf == XF_Q8K) {  // wave-uniform
        finish_q8k<D>(o, l, rvalid, tok0 + rtok, rhead, H, row, quad, planes, npad);
        return;
      }
    }
    if constexpr (D >= 32) {
      if (planes && xf == XF_Q80) {
        finish_q80<D>(o, l, rvalid, tok0 + rtok, rhead, H, quad, planes, npad);
        return;
      }
    }
    if (rvalid) {
      const int64_t n = tok0 + rtok;
      if (planes) {
        // split planes of the output product's X: the lanes of a row hold
        // 8 values of each 32-value group (d tiles 2g and 2g + 1)
        const int64_t K = (int64_t)H * D, k0 = (int64_t)rhead * D;
#pragma unroll
        for (int g = 0; g < DT / 2; g++) {
          float s = 0.0f;
#pragma unroll
          for (int h2 = 0; h2 < 2; h2++) {
            const f32x4 y = o[2 * g + h2] / l;
            const float v[4] = {y[0], y[1], y[2], y[3]};
            split_store4(planes, npad, K, n, k0 + (2 * g + h2) * 16 + quad * 4, v);
            s += v[0] + v[1] + v[2] + v[3];
          }
          s += __shfl_xor(s, 16);
          s += __shfl_xor(s, 32);
          if (quad == 0) split_store_gsum(planes, npad, K, n, (k0 >> 5) + g, s);
        }
      } else {
        float *orow = out + (n * H + rhead) * D;
#pragma unroll
        for (int dt = 0; dt < DT; dt++) *(f32x4 *)(orow + dt * 16 + quad * 4) = o[dt] / l;
      }
    }
    return;
  }
  const int nrows = ntok * G;
  float *pp = part + ((int64_t)item * Hkv + kvh) * Partial<D>::floats;
  if (row < nrows) {
#pragma unroll
    for (int dt = 0; dt < DT; dt++) *(f32x4 *)(pp + row * D + dt * 16 + quad * 4) = o[dt];
    if (quad == 0) {
      pp[ROWS * D + row] = m;
      pp[ROWS * D + ROWS + row] = l;
    }
  }
}

// The chunks' places in the rows of K and V tiles in LDS (shared runs).
template <int D>
__device__ __forceinline__ int swk(int r) {  // distinct over the 16 rows of a tile (s_cell)
  return D / 8 >= 16 ? (r & 3) | ((r >> 1) & 12) : ((r >> 1) & 1) | ((r >> 2) & 6);
}
__device__ __forceinline__ int swv(int r) { return (r >> 1) & 7; }

// What the tokens of a tree plan see, in the blocks that hold the pass's own
// tokens: bit c of word w of token t is cell c of block npast / 64 + w
// (lgmlh_plan_tree). They stand behind the plan's last arrays (items, merge,
// shared, order; `order` itself may be another or NULL).
inline const uint64_t *plan_vis(const lgmlh_ubatch *ub) {
  auto align16 = [](int64_t x) { return (x + 15) & ~int64_t(15); };
  return (const uint64_t *)((const char *)ub->items + 16 * (int64_t)ub->n_items +
                            16 * (int64_t)ub->n_merge + align16(8 * (int64_t)ub->n_shared) +
                            align16(4 * (int64_t)ub->n_single));
}

// The fixed-order merge of a plan's split groups (attn.hip), for the kernels
// that leave partial states of the same form.
void merge_dev(int head_dim, const lgmlh_ubatch *ub, int H, int Hkv, const float *part, float *out,
               f16 *planes, int64_t npad, int xf, hipStream_t st);
// The same with many splits merged in slices side by side (heads of 64, 128 and 256).
void merge_slices_dev(int head_dim, const lgmlh_ubatch *ub, int H, int Hkv, const float *part, float *out,
                      f16 *planes, int64_t npad, int xf, hipStream_t st);
bool attn_q8k_fits(int head_dim, int G);
int attn_check(const char *what, const float *q, int n_head, int n_head_kv, int head_dim,
               const void *kpool, const void *vpool, const lgmlh_ubatch *ub, const float *out,
               const f16 *planes, int xf, const void *workspace, size_t workspace_bytes, int *run);

}  // namespace lgmlh
