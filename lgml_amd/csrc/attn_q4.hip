// Paged GQA attention over Q4_0 KV blocks (gfx950): the work items, rows and
// merge of attn.hip over the tiles of kvq4.hip.
//
// The arithmetic is attnq.h's, with n - 8 for the whole numbers. A 4-bit n becomes an f16
// by the mantissa: bits 0 .. 3 of a half word under the exponent of 1024 are 1024 + n, bits
// 4 .. 7 under that of 64 are 64 + n, and the differences to 1032 and 72 are exact: 9
// operations for 8 values. (Left as they are, the bits are n 2^-24 and 16 n 2^-24 and take
// 5; but the matrix unit aligns products by the exponents that subnormal numbers have in
// common, and loses 8 and 4 bits of sums over unlike terms: 2e-5 and 1e-6 of the largest.)
// q is multiplied by the scale before it is split, so that what makes scores of the sums
// is a power of two, exact in an fma with the maximum; P is 2^13 times as large by way of
// that maximum, so that small weights keep their bits.
//
// A run of blocks is taken in PARTS parts, part i its blocks i, i + 4, ... (of a ring by
// their own numbers), a wave each: a row's state (O, m, l) starts anew in each, and the
// states join in order.
//
// Sets of items over the same blocks (a chunk's) are taken one by one, too. Unpacked once
// for a set's eight waves in LDS, as Q8_0's are, they were slower at every size, in runs of
// 12 (28) and with what this kernel was then: heads of 128, 32 / 8, 512 tokens after 2048
// cells 110 us against 95 (90 since), 4096 from none 639 against 583 (561); heads of 256, 8 /
// 4, 133 against 55 (50) and 318 against 288 (277).
//
// Bounds. One token of 64 sequences at 128 to 4096 cells, 32 / 8 heads of 128, is 46 us in
// runs of 12 blocks and 42 in runs of 20 (968 workgroups), the merge's 5 with them: 159 MB,
// 3.9 and 4.3 TB/s in the first kernel (34 us with the loads alone). In runs of 12, a block
// of 64 cells is 650 vector operations a wave (288 of them the unpacking; a decode step's 4
// rows use a quarter of the columns of the others), which take the three waves of a SIMD
// 3.8 us, its bytes of all the waves 5.6 at the copy's rate; a workgroup of 12 blocks starts
// with 4 us until its first bytes are there, and the 1688 workgroups of the step are 2.2
// times what the card holds. A chunk of 512 tokens after 2048, 8 / 4 heads of 256, is 50
// us, half of them vector operations of its 2048 waves, two a SIMD; over 32 / 8 heads of
// 128, in runs of 20, 83. One sequence leaves most of the card idle, and the blocks of a
// wave go one after another: 8192 cells, 32 / 8 heads of 128, are 16 us in runs of 12 and
// 21 in runs of 20 (56 workgroups, five blocks a wave), 8 / 4 heads of 256 40 in runs of
// 28 (Q8_0 34 and 113, f16 20 and 55).
#include "attnq.h"
#include "kvq4.h"

namespace lgmlh {

// The masks and the exponents are made opaque, the former for scalar registers, the
// latter for vector ones: a mask and an exponent known as numbers are two operations, (w &
// m) | e of registers is one.
struct Nibbles {
  uint32_t low = 0x000f000f, high = 0x00f000f0, e1024 = 0x64006400, e64 = 0x54005400;
  __device__ __forceinline__ Nibbles() { asm("" : "+s"(low), "+s"(high), "+v"(e1024), "+v"(e64)); }
  __device__ __forceinline__ f16x2 low_pair(uint32_t w) const {
    return __builtin_bit_cast(f16x2, (w & low) | e1024) - f16x2{(f16)1032.0f, (f16)1032.0f};
  }
  __device__ __forceinline__ f16x2 high_pair(uint32_t w) const {
    return __builtin_bit_cast(f16x2, (w & high) | e64) - f16x2{(f16)72.0f, (f16)72.0f};
  }
  // K's word: 8 dims of a cell.
  __device__ __forceinline__ f16x8 k(uint32_t w) const {
    return join(low_pair(w), high_pair(w), low_pair(w >> 8), high_pair(w >> 8));
  }
  // V's two words: 8 cells of a dim r (their low halves) or r + 16.
  __device__ __forceinline__ f16x8 v(uint32_t w0, uint32_t w1, bool upper) const {
    return upper ? join(high_pair(w0), high_pair(w0 >> 8), high_pair(w1), high_pair(w1 >> 8))
                 : join(low_pair(w0), low_pair(w0 >> 8), low_pair(w1), low_pair(w1 >> 8));
  }
  __device__ __forceinline__ static f16x8 join(f16x2 a, f16x2 b, f16x2 c, f16x2 d) {
    return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
  }
};

constexpr int PARTS = 4;

template <int HEAD>
struct Q4Frag {
  static constexpr int D = HEAD, NB = D / 32, DT = D / 16;
  static constexpr int SCALES = 32 * D, TILE = q4_tile_bytes(D);
  static constexpr int DV = 1;          // V's scales of 2^-8 to 2^2 (largest values of 0.03 to 31) go packed
  static constexpr int U = q4_k_words(D);
  typedef uint32_t KUnit __attribute__((ext_vector_type(U)));  // a cell's dims 32 (U j + u) + 8 quad ..
  static constexpr int KJ = D / (32 * U), VJ = D / 32;
  __device__ __forceinline__ static f16x8 k_frag(Nibbles n, const KUnit (&k)[KJ], int b) { return n.k(k[b / U][b % U]); }
  __device__ __forceinline__ static f16x8 v_frag(Nibbles n, const u32x4 (&v)[VJ], int t, int kc) {
    return n.v(v[t / 2][2 * kc], v[t / 2][2 * kc + 1], t & 1);
  }
};

// A row's state: O^T, the largest score less 13 (in units of log2), the sum of P of the
// lane's own cells.
template <typename F>
struct Q4State {
  f32x4 o[F::DT];
  float m, l;
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < F::DT; i++) o[i] = f32x4{0, 0, 0, 0};
    m = -INFINITY;
    l = 0.0f;
  }
  // The end of a part: l of the whole row.
  __device__ __forceinline__ void finish() {
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
  }
  // Joined with a later part's. (Few tiles at a time: read all at once, they take registers.)
  template <typename O>
  __device__ __forceinline__ void join(float m1, float l1, O o1) {
    const float top = fmaxf(m, m1), use = top == -INFINITY ? 0.0f : top;
    const float w = __builtin_amdgcn_exp2f(m - use), w1 = __builtin_amdgcn_exp2f(m1 - use);
#pragma unroll
    for (int t = 0; t < F::DT; t++) {
      const f32x4 a = o1(t);
#pragma unroll
      for (int i = 0; i < 4; i++) o[t][i] = fmaf(o[t][i], w, a[i] * w1);
      if (t % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }
    l = fmaf(l, w, l1 * w1);
    m = top;
  }
};

// q row pieces -> B operands, hi and lo, of the row times the scale and 2^(15 - e), for the
// blocks of dims that are `mine` (the same for the wave); the power of two that undoes it.
template <int NB, typename P, typename M>
__device__ __forceinline__ float split_q4(f32x4 (&qa)[2 * NB], bool rvalid, float scale_log2, P put, M mine) {
  float mx = 0.0f;
#pragma unroll
  for (int i = 0; i < 2 * NB; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) {
      qa[i][j] *= scale_log2;
      mx = fmaxf(mx, fabsf(qa[i][j]));
    }
  mx = quads_max(mx);
  int e = __builtin_amdgcn_frexp_expf(mx);
  e = e < -110 ? -110 : e;
  const float up = rvalid ? pow2(15 - e) : 0.0f;
#pragma unroll
  for (int b = 0; b < NB; b++) {
    if (!mine(b)) continue;
    f16x8 hi, lo;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float x = rvalid ? qa[2 * b + (i >> 2)][i & 3] * up : 0.0f;
      hi[i] = (f16)x;
      lo[i] = (f16)(x - (float)hi[i]);
    }
    put(b, hi, lo);
  }
  return pow2(e - 15);
}

// Raw scores -> P (2^13 of the weight) in place, the running maximum and sum, the
// rescale of O^T. up: the power of two that makes scores of them, in units of log2.
// masked: cells without a bit in word are dropped.
template <typename F>
__device__ __forceinline__ void softmax_q4(f32x4 (&st)[4], float up, bool masked, uint64_t word, Q4State<F> &s) {
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
  mx = quads_max(mx) * up;
  // 13 below the largest, and no further by that sum's rounding: P is at most 2^13
  float below = mx - 13.0f;
  if (mx - below > 13.0f) below = mx;
  const float m = fmaxf(s.m, below), use = m == -INFINITY ? 0.0f : m;
  float sum = 0.0f;
#pragma unroll
  for (int ct = 0; ct < 4; ct++)
#pragma unroll
    for (int i = 0; i < 4; i++) {
      st[ct][i] = __builtin_amdgcn_exp2f(fmaf(st[ct][i], up, -use));  // exp2(-inf) = 0
      sum += st[ct][i];
    }
  if (__builtin_amdgcn_ballot_w64(m != s.m)) {
    const float alpha = __builtin_amdgcn_exp2f(s.m - use);
    s.l *= alpha;
#pragma unroll
    for (int t = 0; t < F::DT; t++) s.o[t] *= alpha;
  }
  s.l += sum;
  s.m = m;
  asm volatile("" : "+v"(s.l));  // (summed here: put off to the end of the block, P is held for it)
}

// P of the cells 32 h + 8 quad + e as f16 hi + lo.
__device__ __forceinline__ void split_ph(const f32x4 (&st)[4], int h, f16x8 &hi, f16x8 &lo) {
  float minus = -1.0f;  // (opaque: an fma of mixed types, not a conversion and a sum)
  asm("" : "+s"(minus));
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const f32x4 &s = st[2 * h + (e >> 2)];
    const f16x2 a = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_pkrtz(s[e & 3], s[(e & 3) + 1]));
    hi[e] = a[0];
    hi[e + 1] = a[1];
    lo[e] = (f16)fmaf((float)a[0], minus, s[e & 3]);
    lo[e + 1] = (f16)fmaf((float)a[1], minus, s[(e & 3) + 1]);
  }
}
// P dv of those cells times up, or of a plain row as the packed products make it. (What
// other calls make alike is not held for this one: the copy is opaque.)
__device__ __forceinline__ void weigh_ph(const f32x4 (&st)[4], int h, f16x8 dv, bool plain, float up, f16x8 &hi,
                                         f16x8 &lo) {
  asm volatile("" : "+v"(dv));
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const float p0 = st[2 * h + (e >> 2)][e & 3], p1 = st[2 * h + (e >> 2)][(e & 3) + 1];
    f16x2 a, b;
    split2(p0 * (float)dv[e] * up, p1 * (float)dv[e + 1] * up, a, b);
    f16x2 c, d, ph, pl;
    split2(p0, p1, ph, pl);
    packed_pdv(ph, pl, f16x2{dv[e], dv[e + 1]}, c, d);
    a = plain ? c : a;
    b = plain ? d : b;
    hi[e] = a[0];
    hi[e + 1] = a[1];
    lo[e] = b[0];
    lo[e + 1] = b[1];
  }
}

// P for the products with dv: scale(b, h) gives the lane's cells' dv of block b of dims.
// plain (the same for the wave): all scales go by the packed products, and P is split once,
// in its own registers. Else a row goes its own way by the scales of the cells it sees
// (word), and by nothing else, so that it has the same bits in any group of rows: true if
// that is the packed products' too.
template <typename F, typename S>
__device__ __forceinline__ bool ready_p(f32x4 (&st)[4], bool plain, uint64_t word, S scale) {
  bool row_plain = true;
  if (plain) {
    f16x8 hi[2], lo[2];
    split_ph(st, 0, hi[0], lo[0]);
    split_ph(st, 1, hi[1], lo[1]);
#pragma unroll
    for (int h = 0; h < 2; h++) {
      st[2 * h] = __builtin_bit_cast(f32x4, hi[h]);
      st[2 * h + 1] = __builtin_bit_cast(f32x4, lo[h]);
    }
  } else {
    float low = 65535.0f, high = 0.0f;
#pragma unroll 1
    for (int b = 0; b < F::NB; b++) {
      u32x4 s0 = scale(b, 0), s1 = scale(b, 1);
      seen_scales(s0, s1, word);
      low = fminf(low, fminf(low_bits(s0), low_bits(s1)));
      high = fmaxf(high, fmaxf(high_bits(s0), high_bits(s1)));
    }
    row_plain = plain_range<F>(-quads_max(-low), quads_max(high));
  }
#pragma unroll
  for (int i = 0; i < 4; i++) here(st[i]);  // (P or its halves, in the same registers)
  return row_plain;
}
// P dv of a block of dims as f16 hi + lo, from ready_p's P and the lane's cells' dv; what
// undoes its power of two.
__device__ __forceinline__ float times_dv_q4(const f32x4 (&st)[4], bool plain, bool row_plain, uint64_t word, u32x4 s0,
                                             u32x4 s1, f16x8 (&hi)[2], f16x8 (&lo)[2]) {
  float back = 1.0f;
  if (plain) {
    packed_pdv(__builtin_bit_cast(f16x8, st[0]), __builtin_bit_cast(f16x8, st[1]), __builtin_bit_cast(f16x8, s0), hi[0],
               lo[0]);
    packed_pdv(__builtin_bit_cast(f16x8, st[2]), __builtin_bit_cast(f16x8, st[3]), __builtin_bit_cast(f16x8, s1), hi[1],
               lo[1]);
  } else {
    seen_scales(s0, s1, word);
    const f16x8 dv[2] = {__builtin_bit_cast(f16x8, s0), __builtin_bit_cast(f16x8, s1)};
    const int ex = largest_pdv(st, dv);
    back = pow2(ex - 15);
    weigh_ph(st, 0, dv[0], row_plain, pow2(15 - ex), hi[0], lo[0]);
    weigh_ph(st, 1, dv[1], row_plain, pow2(15 - ex), hi[1], lo[1]);
  }
  return back;
}
// The accumulators of two tiles before and after those products.
__device__ __forceinline__ void begin_acc(f32x4 (&acc)[2], const f32x4 *o, bool plain, bool row_plain) {
#pragma unroll
  for (int t = 0; t < 2; t++) {
    acc[t] = o[t];
    if (!plain)
#pragma unroll
      for (int i = 0; i < 4; i++) acc[t][i] = row_plain ? acc[t][i] : 0.0f;
  }
}
__device__ __forceinline__ void end_acc(const f32x4 (&acc)[2], f32x4 *o, bool plain, bool row_plain, float back) {
#pragma unroll
  for (int t = 0; t < 2; t++) {
    if (plain)
      o[t] = acc[t];
    else
#pragma unroll
      for (int i = 0; i < 4; i++) o[t][i] = row_plain ? acc[t][i] : fmaf(acc[t][i], back, o[t][i]);
    here(o[t]);
  }
}

// O^T += V^T (P dv)^T over a block: frag(t, kc) is V's operand.
template <typename F, typename S, typename V>
__device__ __forceinline__ void values_q4(Q4State<F> &s, f32x4 (&st)[4], bool plain, uint64_t word, S scale, V frag) {
  const bool row_plain = ready_p<F>(st, plain, word, scale);
#pragma unroll
  for (int b = 0; b < F::NB; b++) {
    f16x8 hi[2], lo[2];
    f32x4 acc[2];
    const float back = times_dv_q4(st, plain, row_plain, word, scale(b, 0), scale(b, 1), hi, lo);
    begin_acc(acc, s.o + 2 * b, plain, row_plain);
#pragma unroll
    for (int kc = 0; kc < 2; kc++) {
      f16x8 v[2];
#pragma unroll
      for (int t = 0; t < 2; t++) {
        v[t] = frag(2 * b + t, kc);
        acc[t] = mfma16q(v[t], hi[kc], acc[t]);
      }
#pragma unroll
      for (int t = 0; t < 2; t++) acc[t] = mfma16q(v[t], lo[kc], acc[t]);
    }
    end_acc(acc, s.o + 2 * b, plain, row_plain, back);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// Whether a lane's 8 scales go by the packed products.
template <typename F>
__device__ __forceinline__ bool plain_lane(u32x4 sc) {
  return plain_range<F>(low_bits(sc), high_bits(sc));
}

// An item: a workgroup, a wave each part. Each wave reads its blocks from the pool into
// registers, the next one's K and scales while one is used; q's operands are in LDS, made
// once, and the states join there. ONCE (plans without shared sets): values are read past
// the caches. The step of 64 sequences, in runs of 12, takes 45 us so, 49 through them (77
// either way after a prefix of 4000 cells that all share); a chunk, whose items read the
// same blocks, 52 and 50.
template <int D, bool ONCE>
__global__ void __launch_bounds__(64 * PARTS, D == 256 ? 2 : 3)
paged_attn_q4_kernel(const float *__restrict__ q, int H, int Hkv, float scale_log2,
                     const uint8_t *__restrict__ kpool, const uint8_t *__restrict__ vpool,
                     const int32_t *__restrict__ items, const int32_t *__restrict__ seq_off,
                     const int32_t *__restrict__ seq_npast, const int32_t *__restrict__ block_tab,
                     int max_blocks, int ring, int window, float *__restrict__ out,
                     f16 *__restrict__ planes, int64_t npad, int xf, float *__restrict__ part,
                     const int32_t *__restrict__ order, int n_order, const uint64_t *__restrict__ vis) {
  typedef Q4Frag<D> F;
  constexpr int NB = F::NB, DT = F::DT;
  constexpr int SR = D > 128 ? 2 : 1;       // registers of a block's scales: K's and V's, or K's then V's
  constexpr int SL = D > 128 ? 64 : D / 4;  // lanes of K's
  __shared__ __align__(16) f16x8 qsh[NB * 64], qsl[NB * 64];
  __shared__ __align__(16) u32x4 scales[PARTS][2 * SL];  // of each wave's block
  __shared__ __align__(16) f32x4 parts[PARTS - 1][DT * 64];
  __shared__ float part_m[PARTS - 1][64], part_l[PARTS - 1][64];
  const int lane = threadIdx.x & 63, row = lane & 15, quad = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int slot = (int)(blockIdx.x / (uint32_t)Hkv), kvh = (int)(blockIdx.x % (uint32_t)Hkv);
  const int item = slot < n_order ? order[slot] : slot;
  const int seq = items[4 * item + 0], tok0 = items[4 * item + 1];
  const int ntok = items[4 * item + 2] & 31, mg = (items[4 * item + 2] >> 5) - 1;
  const int blo = items[4 * item + 3] & 0xffff, bhi = (items[4 * item + 3] >> 16) & 0xffff;
  const int G = H / Hkv;
  const Sight see(seq_off[seq], seq_npast[seq], tok0, ntok, G, ring, window, vis);
  const int32_t *bt = block_tab + (int64_t)seq * max_blocks;
  auto tile = [&](const uint8_t *pool, int blk) {
    const int64_t b = __builtin_amdgcn_readfirstlane(bt[ring > 0 ? blk % ring : blk]);
    return pool + (b * Hkv + kvh) * (int64_t)F::TILE;
  };
  typename F::KUnit kq[4][F::KJ];
  u32x4 vq[F::VJ], sreg[SR];
  constexpr int KC = 4 * sizeof(typename F::KUnit);  // bytes of a cell's units
  const uint32_t koff = (8 * (row >> 2) + (row & 3)) * KC + quad * (KC / 4), voff = row * 64 + quad * 16;
  auto read = [](auto *from) { return ONCE ? __builtin_nontemporal_load(from) : *from; };
  auto load_k = [&](int blk) {
    const uint8_t *t = tile(kpool, blk);
#pragma unroll
    for (int ct = 0; ct < 4; ct++)
#pragma unroll
      for (int j = 0; j < F::KJ; j++)
        kq[ct][j] = read((const typename F::KUnit *)(t + (j * 4096 + s_cell(ct, 0) * KC) + koff));
  };
  auto load_v = [&](int blk) {
    const uint8_t *t = tile(vpool, blk);
#pragma unroll
    for (int j = 0; j < F::VJ; j++) vq[j] = read((const u32x4 *)(t + j * 1024 + voff));
  };
  auto load_s = [&](int blk) {
    const uint8_t *k = tile(kpool, blk) + F::SCALES, *v = tile(vpool, blk) + F::SCALES;
    if constexpr (SR == 2) {
      sreg[0] = *(const u32x4 *)(k + lane * 16u);
      sreg[1] = *(const u32x4 *)(v + lane * 16u);
    } else {
      sreg[0] = *(const u32x4 *)((lane < SL ? k : v) + lane % SL * 16u);
    }
  };
  u32x4 *scl = scales[wave];
  auto scale_of = [&](int v, int b, int h) { return scl[v * SL + b * 8 + h * 4 + quad]; };
  // the wave's part: from lo on every PARTS-th block, to the last that a row sees
  const int seen_hi = see.p_last / KV_BLOCK + 1, hi = bhi < seen_hi ? bhi : seen_hi;
  const int org = ring > 0 ? 0 : blo, lo = blo + ((wave - (blo - org)) & (PARTS - 1));
  float up;
  {
    const RowOf r(lane, G, ntok);
    f32x4 qa[2 * NB];
    const float *qr = q + ((int64_t)(tok0 + (r.valid ? r.rtok : ntok - 1)) * H + kvh * G + r.head) * D;
#pragma unroll
    for (int b = 0; b < NB; b++) {
      qa[2 * b] = *(const f32x4 *)(qr + 32 * b + 8 * r.quad);
      qa[2 * b + 1] = *(const f32x4 *)(qr + 32 * b + 8 * r.quad + 4);
    }
    if (lo < hi) {
      load_s(lo);
      load_k(lo);
    }
    up = split_q4<NB>(qa, r.valid, scale_log2, [&](int b, f16x8 h, f16x8 l) {
      qsh[b * 64 + lane] = h;
      qsl[b * 64 + lane] = l;
    }, [&](int b) { return b % PARTS == wave; });
  }
  lds_sync();
  const Nibbles nib;
  Q4State<F> s;
  s.clear();
  for (int blk = lo; blk < hi; blk += PARTS) {
    const bool more = blk + PARTS < hi;
    f32x4 st[4];
    int ql_at = lane;
    asm volatile("" : "+v"(ql_at));  // Q's operands are read anew: held, they spill others
    // (the lanes of K's scales have no part in this)
    const bool plain = !__builtin_amdgcn_ballot_w64(!plain_lane<F>(sreg[SR - 1]) &&
                                                    (SR == 2 || (lane >= SL && lane < 2 * SL)));
    if (SR == 2) scl[lane] = sreg[0];
    if (SR == 2 || lane < 2 * SL) scl[(SR - 1) * 64 + lane] = sreg[SR - 1];
    load_v(blk);  // (a block ahead, it kept the next one's K waiting: 64 sequences' step 54 us, so 49)
    scores_q<NB>(
        st,
        [&](int b, int p, f16x8(&k)[2], f16x8 &d) {
#pragma unroll
          for (int t = 0; t < 2; t++) k[t] = F::k_frag(nib, kq[2 * p + t], b);
          d = __builtin_bit_cast(f16x8, scale_of(0, b, p));
        },
        [&](int b, f16x8 &h, f16x8 &l) {
          h = qsh[b * 64 + ql_at];
          l = qsl[b * 64 + ql_at];
        });
    if (more) load_s(blk + PARTS);
    if (more) load_k(blk + PARTS);
    uint64_t word = ~(uint64_t)0;
    const bool masked = see.masks(blk, word);
    softmax_q4<F>(st, up, masked, word, s);
    __builtin_amdgcn_sched_barrier(0);
    values_q4<F>(s, st, plain, word, [&](int b, int h) { return scale_of(1, b, h); },
                 [&](int t, int kc) { return F::v_frag(nib, vq, t, kc); });
  }
  s.finish();
  if (wave > 0) {
#pragma unroll
    for (int t = 0; t < DT; t++) parts[wave - 1][t * 64 + lane] = s.o[t];
    part_m[wave - 1][lane] = s.m;
    part_l[wave - 1][lane] = s.l;
  }
  lds_sync();
  if (wave) return;
#pragma unroll 1
  for (int i = 0; i < PARTS - 1; i++)
    s.join(part_m[i][lane], part_l[i][lane], [&](int t) { return parts[i][t * 64 + lane]; });
  const RowOf r(lane_anew(), G, ntok);
  finish_item<D>(s.o, s.m, s.l, mg, r.valid, tok0, r.rtok, kvh * G + r.head, ntok, G, r.row, r.quad, item, kvh,
                 Hkv, H, out, planes, npad, xf, part);
}

template <int D>
static void launch_attn_q4(const float *q, int H, int Hkv, float scale_log2, const void *kp, const void *vp,
                           const lgmlh_ubatch *ub, float *out, f16 *planes, int64_t npad, int xf,
                           float *part, hipStream_t st) {
  const uint64_t *vis = ub->ring == LGMLH_PLAN_TREE ? plan_vis(ub) : nullptr;
  const auto kern = ub->n_shared > 0 ? paged_attn_q4_kernel<D, false> : paged_attn_q4_kernel<D, true>;
  if (ub->n_items > 0)
    hipLaunchKernelGGL(kern, dim3((uint32_t)ub->n_items * Hkv), dim3(64 * PARTS), 0, st, q, H, Hkv,
                       scale_log2, (const uint8_t *)kp, (const uint8_t *)vp, ub->items, ub->seq_off, ub->seq_npast,
                       ub->block_tab, ub->max_blocks, ub->ring, ub->window, out, planes, npad, xf, part, ub->order,
                       ub->order ? ub->n_single : 0, vis);
  merge_slices_dev(D, ub, H, Hkv, part, out, planes, npad, xf, st);
}

// paged_attention_dev over Q4_0 pools.
int paged_attention_q4_dev(const float *q, int n_head, int n_head_kv, int head_dim, float scale,
                           const void *kpool, const void *vpool, const lgmlh_ubatch *ub, float *out,
                           f16 *planes, int64_t npad, void *workspace, size_t workspace_bytes,
                           hipStream_t st, int xf) {
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) {
    set_error("paged_attention_q4: head_dim %d not supported (64, 128, 256)", head_dim);
    return LGMLH_EINVAL;
  }
  if (((uintptr_t)kpool | (uintptr_t)vpool) & 15) {
    set_error("paged_attention_q4: pools are 16-byte aligned");
    return LGMLH_EINVAL;
  }
  int run = 0;
  LGMLH_TRY(attn_check("paged_attention_q4", q, n_head, n_head_kv, head_dim, kpool, vpool, ub, out,
                       planes, xf, workspace, workspace_bytes, &run));
  if (!run) return LGMLH_OK;
  if ((int64_t)ub->n_items * n_head_kv >= ((int64_t)1 << 32) / (64 * PARTS)) {  // fewer than 2^32 threads a launch
    set_error("paged_attention_q4: %d items x %d KV heads in one launch", ub->n_items, n_head_kv);
    return LGMLH_EINVAL;
  }
  const float sl = scale * LOG2E;
  float *part = (float *)workspace;
  switch (head_dim) {
    case 64: launch_attn_q4<64>(q, n_head, n_head_kv, sl, kpool, vpool, ub, out, planes, npad, xf, part, st); break;
    case 128: launch_attn_q4<128>(q, n_head, n_head_kv, sl, kpool, vpool, ub, out, planes, npad, xf, part, st); break;
    default: launch_attn_q4<256>(q, n_head, n_head_kv, sl, kpool, vpool, ub, out, planes, npad, xf, part, st); break;
  }
  return hip_check(hipGetLastError(), "paged_attention_q4");
}

}  // namespace lgmlh

using namespace lgmlh;

extern "C" int lgmlh_paged_attention_q4(const float *q, int n_head, int n_head_kv, int head_dim,
                                        float scale, const void *kpool, const void *vpool,
                                        const lgmlh_ubatch *ub, float *out, void *workspace,
                                        size_t workspace_bytes, void *stream) {
  if (!out) {
    set_error("paged_attention_q4: bad arguments");
    return LGMLH_EINVAL;
  }
  return paged_attention_q4_dev(q, n_head, n_head_kv, head_dim, scale, kpool, vpool, ub, out,
                                nullptr, 0, workspace, workspace_bytes, as_stream(stream), XF_SPLIT);
}
