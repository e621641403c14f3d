// Norms, rotation by positions of several axes, and the KV store of a pass's rows
// (gfx950).
#include <math.h>

#include <type_traits>

#include "kvstore.h"

namespace lgmlh {

// Dims i and i + n_rot / 2 of a head turn by the angle pos[a][t] base^(-2 i / n_rot) /
// ff[i], a the pair's axis. The angle is made in 64 bits, in turns: in 32 a position
// of 100000 is off by 0.4% of a radian and more.
struct AxesRope {
  int n_rot, interleaved;
  int end[3];      // sections one after the other: the first pair behind axis 0, 1, 2
  double log2_step;  // log2 of base^(-2 / n_rot)
  const float *ff;
  const int32_t *pos;  // (4, n)
  __device__ __forceinline__ int axis(int i) const {
    if (!interleaved) return (i >= end[0]) + (i >= end[1]) + (i >= end[2]);
    const int a = i % 3;  // in turn; what an axis has no pairs left for goes by axis 0
    const int mine = a == 0 ? end[0] : a == 1 ? end[1] - end[0] : end[2] - end[1];
    return i < 3 * mine ? a : 0;
  }
  __device__ __forceinline__ void angle(int i, int64_t t, int64_t n, float &c, float &s) const {
    const double freq = exp2(log2_step * i) * 0.15915494309189533577;  // over 2 pi
    double turns = (double)pos[axis(i) * n + t] * freq;
    if (ff) turns /= (double)ff[i];
    sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
  }
};

// The sum over aligned groups of W lanes (8, 16 or 32), the same in each.
template <int W>
__device__ __forceinline__ float lanes_sum(float v) {
  v += dpp_f<DPP_XOR1>(v);
  v += dpp_f<DPP_XOR2>(v);
  v += dpp_f<DPP_HALF_MIRROR>(v);
  if constexpr (W > 8) v += dpp_f<DPP_MIRROR>(v);
  if constexpr (W > 16) v += __shfl_xor(v, 16);
  return v;
}

// What a wave wrote to LDS is there for its other lanes.
__device__ __forceinline__ void wave_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// A workgroup takes a token's q and k heads, 512 / D of them a wave and step, 8 dims a
// lane: lane l of a head's D / 8 has the pairs from 4 l on (4 dims of each half), or
// 8 dims behind the rotated ones. The token's angles are made once, a thread each,
// while the rows of STEPS steps are on their way. K rows turn in LDS into 8 dims in a
// row a lane, as they are stored. q's rows pass the caches by: 4096 tokens of 32 / 4
// heads of 128, 159 MB, take 28 us, 5.6 TB/s, with cached stores 31; 64 tokens 5 either way.
// Into pools of f16, Q8_0 and Q4_0, 2048 tokens of 32 / 8 heads of 128 (92 to 86 MB) are 15.8,
// 15.5 and 15.6 us, 8 / 4 heads of 256 (59 to 53 MB) 12.1, 11.7 and 12.0.
constexpr int AXES_STEPS = 4;
template <int TYPE, int D>
__device__ __forceinline__ void turn_heads(const float *__restrict__ qkv, int64_t n, int H, int Hkv, const AxesRope &r,
                                           const float *__restrict__ q_norm, const float *__restrict__ k_norm,
                                           float eps, uint8_t *__restrict__ kp, int64_t n_cells,
                                           const int64_t *__restrict__ cells, float *__restrict__ q_out, int64_t t,
                                           float *cs, float (&rows)[KV_THREADS / 64][512]) {
  constexpr int L = D / 8, AT = 64 / L, ALL = KV_THREADS / L;  // lanes of a head, heads of a wave, of a workgroup
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane % L, half = r.n_rot / 2, last = H + Hkv;
  const bool turns = 4 * l < half;
  const int at0 = turns ? 4 * l : 8 * l, at1 = turns ? at0 + half : at0 + 4;
  const float *row = qkv + t * (int64_t)(H + 2 * Hkv) * D;
  f32x4 a[AXES_STEPS], b[AXES_STEPS];
  auto load = [&](int base) {
#pragma unroll
    for (int i = 0; i < AXES_STEPS; i++) {
      const int h = base + i * ALL + wave * AT + lane / L;
      a[i] = b[i] = f32x4{0, 0, 0, 0};
      if (h < last) {
        a[i] = *(const f32x4_u *)(row + h * D + at0);
        b[i] = *(const f32x4_u *)(row + h * D + at1);
      }
    }
  };
  load(0);
  f32x4 qw[2], kw[2];
  if (q_norm) {
    qw[0] = *(const f32x4_u *)(q_norm + at0);
    qw[1] = *(const f32x4_u *)(q_norm + at1);
  }
  if (k_norm) {
    kw[0] = *(const f32x4_u *)(k_norm + at0);
    kw[1] = *(const f32x4_u *)(k_norm + at1);
  }
  const int64_t cell = cells[t];
  const bool stored = (uint64_t)cell < (uint64_t)n_cells;
  if ((int)threadIdx.x < half) r.angle(threadIdx.x, t, n, cs[threadIdx.x], cs[D / 2 + threadIdx.x]);
  lds_sync();
  f32x4 c = {1, 1, 1, 1}, s = {0, 0, 0, 0};
  if (turns) {
    c = *(const f32x4 *)(cs + at0);
    s = *(const f32x4 *)(cs + D / 2 + at0);
  }
  for (int base = 0; base < last; base += AXES_STEPS * ALL) {
    if (base) load(base);
#pragma unroll
    for (int i = 0; i < AXES_STEPS; i++) {
      const int h0 = base + i * ALL + wave * AT;
      if (h0 >= last) break;  // the same for the wave
      const int h = h0 + lane / L;
      const bool has = h < last, is_k = h >= H;
      if (q_norm || k_norm) {
        float sum = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; e++) sum = fmaf(a[i][e], a[i][e], fmaf(b[i][e], b[i][e], sum));
        sum = lanes_sum<L>(sum);
        const float scale = 1.0f / sqrtf(sum / (float)D + eps);
        if (is_k ? k_norm != nullptr : q_norm != nullptr) {
          a[i] = a[i] * scale * (is_k ? kw[0] : qw[0]);
          b[i] = b[i] * scale * (is_k ? kw[1] : qw[1]);
        }
      }
      f32x4 x, y;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        x[e] = fmaf(a[i][e], c[e], -b[i][e] * s[e]);
        y[e] = fmaf(a[i][e], s[e], b[i][e] * c[e]);
      }
      if (has && !is_k) {
        float *out = q_out + (t * H + h) * (int64_t)D;
        __builtin_nontemporal_store(x, (f32x4_u *)(out + at0));
        __builtin_nontemporal_store(y, (f32x4_u *)(out + at1));
      }
      if (h0 + AT <= H) continue;  // the same for the wave: q heads alone
      float *mine = rows[wave] + lane / L * D;
      *(f32x4 *)(mine + at0) = x;
      *(f32x4 *)(mine + at1) = y;
      wave_lds();
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] = mine[8 * l + e];
      wave_lds();
      uint32_t q[8];
      float d = 0.0f;
      if constexpr (TYPE != LGMLH_F16) d = quant8<TYPE>(v, q);
      if (!has || !is_k || !stored) continue;
      uint8_t *tile = kv_tile<TYPE, D>(kp + (int64_t)(h - H) * kv_tile_bytes(TYPE, D), cell, Hkv);
      const int o = (int)cell & 63;
      if constexpr (TYPE == LGMLH_F16) {
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; e++) w[e] = f2h(v[2 * e]) | (uint32_t)f2h(v[2 * e + 1]) << 16;
        *(u32x4 *)(tile + (o * D + 8 * l) * 2) = w;
      } else if constexpr (TYPE == LGMLH_Q8_0) {
        *(u32x2 *)(tile + q8_k_at(o, 8 * l)) = u32x2{bytes4(q[0], q[1], q[2], q[3]), bytes4(q[4], q[5], q[6], q[7])};
        if (l % 4 == 0) *(uint16_t *)(tile + q8_scale_at(D, l / 4, o)) = f2h(d);
      } else {
        *(uint32_t *)(tile + q4_k_at(D, o, 8 * l)) = q4_k_word(q);
        if (l % 4 == 0) *(uint16_t *)(tile + q4_scale_at(D, l / 4, o)) = f2h(d);
      }
    }
  }
}

// The first workgroups take V (a window of W tokens of one head each), the others a
// token each.
template <int TYPE, int D, int W>
__global__ void __launch_bounds__(KV_THREADS)
qkv_rope_axes_kernel(const float *__restrict__ qkv, int64_t n, int H, int Hkv, AxesRope r,
                     const float *__restrict__ q_norm, const float *__restrict__ k_norm, float eps,
                     uint8_t *__restrict__ kp, uint8_t *__restrict__ vp, int64_t n_cells,
                     const int64_t *__restrict__ cells, float *__restrict__ q_out, uint32_t v_groups) {
  __shared__ union {
    VTurn<TYPE, D, W> v;
    struct {
      alignas(16) float cs[D], rows[KV_THREADS / 64][512];
    } qk;
  } lds;
  if (blockIdx.x < v_groups) {
    const int h = blockIdx.x % (uint32_t)Hkv;
    const int64_t j0 = (int64_t)(blockIdx.x / (uint32_t)Hkv) * W, stride = (int64_t)(H + 2 * Hkv) * D;
    lds.v.store(qkv + j0 * stride + (int64_t)(H + Hkv + h) * D, stride, vp, h, Hkv, cells, j0, n, n_cells);
    return;
  }
  turn_heads<TYPE, D>(qkv, n, H, Hkv, r, q_norm, k_norm, eps, kp, n_cells, cells, q_out,
                      (int64_t)(blockIdx.x - v_groups), lds.qk.cs, lds.qk.rows);
}

}  // namespace lgmlh

using namespace lgmlh;

extern "C" int lgmlh_qkv_rope_store_axes(int kv_type, const float *qkv, int64_t n, int n_head, int n_head_kv,
                                         int head_dim, int n_rot, const int32_t *sections, int interleaved,
                                         float freq_base, const float *freq_factors, const float *q_norm,
                                         const float *k_norm, float eps, const int32_t *pos, void *kpool,
                                         void *vpool, int64_t n_cells, const int64_t *cells, float *q_out,
                                         void *stream) {
  const int D = head_dim;
  if ((kv_type != LGMLH_F16 && kv_type != LGMLH_Q8_0 && kv_type != LGMLH_Q4_0) || !qkv || !sections || !pos ||
      !kpool || !vpool || !cells || !q_out || n < 0 || n_head <= 0 || n_head_kv <= 0 || n_head_kv > 65535 ||
      n_head > 65535 || (D != 64 && D != 128 && D != 256) || n_rot <= 0 || n_rot > D || n_rot % 8 ||
      !(freq_base > 0.0f) || n_cells <= 0 || n_cells > CELLS_MAX || n_cells % KV_BLOCK) {
    set_error("qkv_rope_store_axes: bad arguments (pools of f16, Q8_0 or Q4_0, heads of 64, 128 or 256, n_rot a "
              "multiple of 8)");
    return LGMLH_EINVAL;
  }
  int64_t sum = 0;
  for (int a = 0; a < 4; a++) {
    sum += sections[a];
    if (sections[a] < 0 || sum > n_rot / 2) {
      sum = -1;
      break;
    }
  }
  if (sum != n_rot / 2 || (interleaved && sections[3])) {
    set_error("qkv_rope_store_axes: sections of %d %d %d %d pairs for n_rot %d%s", sections[0], sections[1],
              sections[2], sections[3], n_rot, interleaved ? " (interleaved: of three axes)" : "");
    return LGMLH_EINVAL;
  }
  if (((uintptr_t)kpool | (uintptr_t)vpool) & 15) {
    set_error("qkv_rope_store_axes: pools are 16-byte aligned");
    return LGMLH_EINVAL;
  }
  if (n >= ((int64_t)1 << 23) / n_head_kv) {  // fewer than 2^32 threads a launch
    set_error("qkv_rope_store_axes: %lld tokens in one call", (long long)n);
    return LGMLH_EINVAL;
  }
  if (n == 0) return LGMLH_OK;
  AxesRope r;
  r.n_rot = n_rot;
  r.interleaved = interleaved != 0;
  r.end[0] = sections[0];
  r.end[1] = r.end[0] + sections[1];
  r.end[2] = r.end[1] + sections[2];
  r.log2_step = -2.0 / n_rot * log2((double)freq_base);
  r.ff = freq_factors;
  r.pos = pos;
  // (V's tokens of a workgroup: 64 tokens of 32 / 8 heads of 128 take 5.3 us with
  // 16, 8.5 with 64; 4096 of 32 / 4 heads 29.2 and 28.4)
  const int big = D > 128 ? 32 : 64;
  const bool small = (n + big - 1) / big * n_head_kv < 256;
  const int w = small ? 16 : big;
  const uint32_t v_groups = (uint32_t)((n + w - 1) / w * n_head_kv);
  const dim3 grid((unsigned)(v_groups + n));
  auto launch = [&](auto kern) {
    hipLaunchKernelGGL(kern, grid, dim3(KV_THREADS), 0, as_stream(stream), qkv, n, n_head, n_head_kv, r, q_norm,
                       k_norm, eps, (uint8_t *)kpool, (uint8_t *)vpool, n_cells, cells, q_out, v_groups);
  };
  auto of = [&](auto type) {
    constexpr int T = decltype(type)::value;
    if (D == 64)
      small ? launch(qkv_rope_axes_kernel<T, 64, 16>) : launch(qkv_rope_axes_kernel<T, 64, 64>);
    else if (D == 128)
      small ? launch(qkv_rope_axes_kernel<T, 128, 16>) : launch(qkv_rope_axes_kernel<T, 128, 64>);
    else
      small ? launch(qkv_rope_axes_kernel<T, 256, 16>) : launch(qkv_rope_axes_kernel<T, 256, 32>);
  };
  if (kv_type == LGMLH_F16)
    of(std::integral_constant<int, LGMLH_F16>{});
  else if (kv_type == LGMLH_Q8_0)
    of(std::integral_constant<int, LGMLH_Q8_0>{});
  else
    of(std::integral_constant<int, LGMLH_Q4_0>{});
  return hip_check(hipGetLastError(), "qkv_rope_store_axes");
}
