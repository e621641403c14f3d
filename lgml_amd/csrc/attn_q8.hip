// Paged GQA attention over Q8_0 KV blocks (gfx950): the work items, rows and
// merge of attn.hip over the tiles of kvq8.hip.
//
// s_rc = q_r . k_c = sum_b dk_cb (q_rb . k8_cb) over the blocks b of 32 dims: the
// 8-bit values are exact in f16, a 16x16x32 f16 MFMA takes one block of q as
// f16 hi + lo against them, and its f32 result is scaled by the cell's dk into
// S^T. q rows are scaled by a power of two to just below 2^15, so that hi + lo
// carries 22 bits of every element down to 2^-17 of the row's largest.
// o_rd = sum_c (p_rc dv_cb) v8_cd, b = d / 32: dv goes into P, per block of 32
// dims, P dv as f16 hi + lo scaled by the power of two that puts the row's
// largest dv of the block at 2^14 to 2^15; the f32 result, scaled back, adds to
// O^T. A cell that a row does not see has its p and dv as zeros, so that nothing
// in it (a scale that is infinite or NaN) reaches the row.
#include <type_traits>

#include "attn.h"

namespace lgmlh {

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
__device__ __forceinline__ float pow2(int e) { return __builtin_amdgcn_ldexpf(1.0f, e); }

template <int D>
struct Q8Frag {
  static constexpr int TILE = 68 * D, NB = D / 32, J = D / 64, DT = D / 16;
};

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
  mx = fmaxf(mx, __shfl_xor(mx, 16));
  mx = fmaxf(mx, __shfl_xor(mx, 32));
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

// Scores (scaled, in units of log2) -> P in place, the running maximum and sum,
// the rescale of O^T. masked: cells without a bit in word are dropped.
template <int DT>
__device__ __forceinline__ void softmax_q8(f32x4 (&st)[4], float rscale, bool masked, uint64_t word,
                                           int quad, float &m, float &l, f32x4 (&o)[DT]) {
#pragma unroll
  for (int ct = 0; ct < 4; ct++) st[ct] *= rscale;
  if (masked) {  // wave-uniform
#pragma unroll
    for (int ct = 0; ct < 4; ct++)
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (!(word >> s_cell(ct, 4 * quad + i) & 1)) st[ct][i] = -INFINITY;
  }
  float mx = -INFINITY;
#pragma unroll
  for (int ct = 0; ct < 4; ct++)
#pragma unroll
    for (int i = 0; i < 4; i++) mx = fmaxf(mx, st[ct][i]);
  mx = fmaxf(mx, __shfl_xor(mx, 16));
  mx = fmaxf(mx, __shfl_xor(mx, 32));
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
  rs += __shfl_xor(rs, 16);
  rs += __shfl_xor(rs, 32);
  if (__builtin_amdgcn_ballot_w64(m_new != m)) {
    const float alpha = __builtin_amdgcn_exp2f(m - m_use);
    l *= alpha;
#pragma unroll
    for (int dt = 0; dt < DT; dt++) o[dt] *= alpha;
  }
  l += rs;
  m = m_new;
}

// P dv of one block of 32 dims as f16 hi + lo (cells 32 h + 8 quad + e), scaled;
// the factor that undoes it. sc: the lane's cells' scales.
__device__ __forceinline__ float weigh_p(const f32x4 (&st)[4], const u32x4 (&sc)[2], bool masked,
                                         uint64_t word, int quad, f16x8 (&ph)[2], f16x8 (&pl)[2]) {
  f16x8 dv[2] = {__builtin_bit_cast(f16x8, sc[0]), __builtin_bit_cast(f16x8, sc[1])};
  if (masked) {
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const uint32_t bits = (uint32_t)(word >> (32 * h + 8 * quad)) & 0xff;
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (!(bits >> e & 1)) dv[h][e] = (f16)0.0f;
    }
  }
  f16x8 big = __builtin_elementwise_max(dv[0], dv[1]);
  f16x4 b4 = __builtin_elementwise_max(f16x4{big[0], big[1], big[2], big[3]},
                                       f16x4{big[4], big[5], big[6], big[7]});
  float mx = fmaxf(fmaxf((float)b4[0], (float)b4[1]), fmaxf((float)b4[2], (float)b4[3]));
  mx = fmaxf(mx, __shfl_xor(mx, 16));
  mx = fmaxf(mx, __shfl_xor(mx, 32));
  const int ex = __builtin_amdgcn_frexp_expf(mx);  // mx in [2^(ex - 1), 2^ex)
  const float up = pow2(15 - ex);
#pragma unroll
  for (int h = 0; h < 2; h++)
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const float x = st[2 * h + (e >> 2)][e & 3] * up * (float)dv[h][e];
      ph[h][e] = (f16)x;
      pl[h][e] = (f16)(x - (float)ph[h][e]);
    }
  return pow2(ex - 15);
}

// What a row (its last visible slot p_row, its token's mask words) sees of a
// block of a causal, ring or tree plan.
struct Sight {
  int ring, window;        // of the plan; ring LGMLH_PLAN_TREE: a tree
  int p_first, p_row, p_last;  // the item's first slot, the row's own, the item's last
  int b_tree;
  const uint64_t *vrow;
  bool rvalid;
  __device__ __forceinline__ bool full(int blk) const {
    if (ring < 0) return blk < b_tree;
    return blk * 64 + 63 <= p_first && (ring == 0 || blk * 64 > p_last - window);
  }
  __device__ __forceinline__ uint64_t word(int blk) const {
    if (!rvalid) return 0;
    if (ring < 0) return vrow[blk - b_tree];
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
  const int row = lane & 15, quad = lane >> 4;
  const int rtok = row / G, rhead = kvh * G + row % G;
  const bool rvalid = rtok < ntok;
  const int npast = seq_npast[s];
  Sight see;
  see.ring = ring;
  see.window = window;
  see.p_first = npast + (tok0 - seq_off[s]);
  see.p_row = see.p_first + rtok;
  see.p_last = see.p_first + ntok - 1;
  see.b_tree = npast / KV_BLOCK;
  see.vrow = ring < 0 ? vis + (int64_t)(tok0 + (rvalid ? rtok : 0)) * window : nullptr;
  see.rvalid = rvalid;

  const int32_t *bt = block_tab + (int64_t)s * max_blocks;
  auto tile = [&](const uint8_t *pool, int blk) {
    const int64_t b = ring > 0 ? bt[blk % ring] : bt[blk];
    return pool + (b * Hkv + kvh) * (int64_t)F::TILE;
  };
  u32x4 kq[4][J], ksc[NB][2], vq[DT], vsc[NB][2];
  auto load_sc = [&](const uint8_t *t, u32x4(&sc)[NB][2]) {
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
      for (int h = 0; h < 2; h++)
        sc[b][h] = *(const u32x4 *)(t + 64 * D + 2 * (b * 64 + 32 * h + 8 * quad));
  };
  auto load_k = [&](int blk) {
    const uint8_t *t = tile(kpool, blk);
#pragma unroll
    for (int ct = 0; ct < 4; ct++)
#pragma unroll
      for (int j = 0; j < J; j++)
        kq[ct][j] = *(const u32x4 *)(t + ((j * 64 + s_cell(ct, row)) * 4 + quad) * 16);
    load_sc(t, ksc);
  };
  auto load_v = [&](int blk) {
    const uint8_t *t = tile(vpool, blk);
#pragma unroll
    for (int dt = 0; dt < DT; dt++) vq[dt] = *(const u32x4 *)(t + (dt * 16 + row) * 64 + quad * 16);
    load_sc(t, vsc);
  };
  float rscale;
  {
    const float *qr = q + ((int64_t)(tok0 + (rvalid ? rtok : ntok - 1)) * H + rhead) * D;
    f32x4 qa[2 * NB];
#pragma unroll
    for (int b = 0; b < NB; b++) {
      qa[2 * b] = *(const f32x4 *)(qr + 32 * b + 8 * quad);
      qa[2 * b + 1] = *(const f32x4 *)(qr + 32 * b + 8 * quad + 4);
    }
    const int b_first = blo < bhi ? blo : 0;  // block 0 of a planned sequence is a pool block
    load_k(b_first);
    load_v(b_first);
    f16x8 hi[NB], lo[NB];
    rscale = split_q<NB>(qa, rvalid, scale_log2, hi, lo);
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
#pragma unroll
    for (int ct = 0; ct < 4; ct++) st[ct] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int b = 0; b < NB; b++) {
      const f16x8 qh = qsh[b * 64 + lane], ql = qsl[b * 64 + lane];
#pragma unroll
      for (int ct = 0; ct < 4; ct++) {
        const u32x4 w = kq[ct][b / 2];
        const f16x8 k = half8(w[2 * (b & 1)], w[2 * (b & 1) + 1]);
        f32x4 acc = mfma16q(k, qh, f32x4{0, 0, 0, 0});
        acc = mfma16q(k, ql, acc);
        const f16x8 d = __builtin_bit_cast(f16x8, ksc[b][ct >> 1]);
#pragma unroll
        for (int i = 0; i < 4; i++) st[ct][i] = fmaf((float)d[4 * (ct & 1) + i], acc[i], st[ct][i]);
      }
    }
    if constexpr (NEXT) load_k(nxt);
    const bool masked = !see.full(blk);
    const uint64_t word = masked ? see.word(blk) : ~(uint64_t)0;
    softmax_q8<DT>(st, rscale, masked, word, quad, m, l, o);
#pragma unroll
    for (int b = 0; b < NB; b++) {
      f16x8 ph[2], pl[2];
      const float back = weigh_p(st, vsc[b], masked, word, quad, ph, pl);
#pragma unroll
      for (int t = 0; t < 2; t++) {
        const u32x4 w = vq[2 * b + t];
        f32x4 acc = {0, 0, 0, 0};
#pragma unroll
        for (int kc = 0; kc < 2; kc++) {
          const f16x8 v = half8(w[2 * kc], w[2 * kc + 1]);
          acc = mfma16q(v, ph[kc], acc);
          acc = mfma16q(v, pl[kc], acc);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) o[2 * b + t][i] = fmaf(acc[i], back, o[2 * b + t][i]);
      }
    }
    if constexpr (NEXT) load_v(nxt);
  };
  for (int blk = blo; blk + 1 < bhi; blk++) block(blk, std::true_type{});
  if (blo < bhi) block(bhi - 1, std::false_type{});
  finish_item<D>(o, m, l, mg, rvalid, tok0, rtok, rhead, ntok, G, row, quad, item, kvh, Hkv, H, out,
                 planes, npad, xf, part);
}

template <int D>
static void launch_attn_q8(const float *q, int H, int Hkv, float scale_log2, const void *kp,
                           const void *vp, const lgmlh_ubatch *ub, float *out, f16 *planes,
                           int64_t npad, int xf, float *part, hipStream_t st) {
  const uint64_t *vis =
      ub->ring == LGMLH_PLAN_TREE ? plan_vis(ub->order, ub->n_single) : nullptr;
  hipLaunchKernelGGL(paged_attn_q8_kernel<D>, dim3((uint32_t)ub->n_items * Hkv), dim3(64), 0, st, q,
                     H, Hkv, scale_log2, (const uint8_t *)kp, (const uint8_t *)vp, ub->items,
                     ub->seq_off, ub->seq_npast, ub->block_tab, ub->max_blocks, ub->ring, ub->window,
                     out, planes, npad, xf, part, ub->order, ub->order ? ub->n_single : 0, vis);
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
