// Paged GQA attention over 64-cell KV blocks (gfx950, wave64, MFMA).
//
// One wavefront per work item: (sequence, KV head, group of query tokens,
// split of KV blocks). The 16 MFMA rows are (token, query head) pairs of
// the group: row r = token (r / G) and head (r % G) of the KV head's G
// query heads, so decode (one token) uses G rows and a prefill chunk packs
// 16 / G tokens per wave.
//
// Per 64-cell block the wave computes S^T = K Q^T with 16x16x32 f16 MFMAs
// (K rows straight from the [cell][D] tile), an online softmax per row in
// f32 (each lane owns one row; reductions over 4 lanes with shuffles), and
// O^T += V^T P^T (V columns straight from the transposed [D][cell] tile, P
// from the lane's own S^T values: s_cell). K and V are exact f16; Q and P
// enter the MFMAs as f16 hi + lo pairs, P ATTN_P times as large (O with it, and
// l in the end: the factor cancels), so that a pair carries 22 bits of every P
// down to 2^-17 of the row's largest, and below is at most 2^-40 of that off.
// (Unscaled, P below 2^-25 was 0 in O but counted in l: one cell 16 above 2000
// others made 4% to 20% of the result wrong. 64 decoding sequences of 32 / 8
// heads of 128 take 106 us either way, a 512-token chunk beside 32 sequences
// 163 and 164.) The loads of block b + 1 are issued as soon as block b's
// registers are consumed (K after S, V after O), so they overlap block b's
// softmax and products.
// Items start longest run first (the plan's order): all of a launch's
// waves are resident at once, and the ones that share a SIMD with an older
// wave advance slowly until it ends, so those should be the shortest.
//
// The splits of a token group are merged by merge_kernel in a fixed order,
// so results are deterministic and, since the split points depend only on
// the sequence's own length, the same for a sequence alone or in any batch.
// (Merging inside the attention kernel by the last split to arrive needs a
// device-scope release per split, an L2 write-back on this multi-XCD part,
// which costs more than the second launch.)
#include <math.h>

#include <type_traits>

#include "attn.h"

namespace lgmlh {

// Scores of one block (scaled, in units of log2) -> P, the running max and
// sum, and the rescale of O^T: the online softmax of a row (a lane owns one;
// its quads hold the cells). masked: cells past p_row (RING: before the window)
// are dropped (TREE: cells whose bit of vis is off); rows past the group hold
// zeros and are never stored.
typedef float f32x2 __attribute__((ext_vector_type(2)));
template <int DT, bool TREE = false>
__device__ __forceinline__ void softmax_block(f32x4 (&st)[4], float scale_log2, bool full,
                                              int cbase, int quad, int p_row, int p_lo, bool rvalid,
                                              uint64_t vis, float &m, float &l, f32x4 (&o)[DT], f16x8 (&ph)[2],
                                              f16x8 (&pl)[2]) {
#pragma unroll
  for (int ct = 0; ct < 4; ct++) st[ct] *= scale_log2;
  if (!full) {  // wave-uniform
#pragma unroll
    for (int ct = 0; ct < 4; ct++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        if constexpr (TREE) {
          if (!(vis >> s_cell(ct, 4 * quad + i) & 1)) st[ct][i] = -INFINITY;
        } else {
          const int p = cbase + s_cell(ct, 4 * quad + i);
          if (!rvalid || p > p_row || p < p_lo) st[ct][i] = -INFINITY;
        }
      }
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
  // rescale only when some row's maximum moved
  if (__builtin_amdgcn_ballot_w64(m_new != m)) {
    const float alpha = __builtin_amdgcn_exp2f(m - m_use);  // 0 when m is -inf
    l *= alpha;
#pragma unroll
    for (int dt = 0; dt < DT; dt++) o[dt] *= alpha;
  }
  l += rs;
  m = m_new;
  // P as f16 hi + lo, cells 32 j + 8 quad + e
#pragma unroll
  for (int j = 0; j < 2; j++)
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const f32x2 p = {st[2 * j + (e >> 2)][e & 3] * ATTN_P,
                       st[2 * j + (e >> 2)][(e & 3) + 1] * ATTN_P};
      const f16x2 hi = __builtin_convertvector(p, f16x2);
      const f32x2 r = {fmaf((float)hi[0], -1.0f, p[0]), fmaf((float)hi[1], -1.0f, p[1])};
      const f16x2 lo = __builtin_convertvector(r, f16x2);
      ph[j][e] = hi[0];
      ph[j][e + 1] = hi[1];
      pl[j][e] = lo[0];
      pl[j][e + 1] = lo[1];
    }
}

// The second product of a block where rows see different cells of a tree's
// nodes and a node's V may be infinite or NaN: 0 times it would be NaN for the
// rows that do not see it. Row by row, with the V of the cells the row does not
// see as zeros, keeping that row's column only. Taken where a lane's V of the
// block is not finite.
__device__ __forceinline__ bool not_finite(f16x8 v) {
  const u32x4 w = __builtin_bit_cast(u32x4, v);
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; i++)
    bad |= (w[i] & 0x7c00u) == 0x7c00u || (w[i] & 0x7c000000u) == 0x7c000000u;
  return bad;
}
// The cells 32 kc + 8 quad .. + 7 of a V fragment that row r's word leaves.
__device__ __forceinline__ f16x8 seen_cells(f16x8 v, uint64_t word, int kc, int quad) {
  const uint32_t bits = (uint32_t)(word >> (32 * kc + 8 * quad)) & 0xff;
#pragma unroll
  for (int e = 0; e < 8; e++)
    if (!(bits >> e & 1)) v[e] = (f16)0.0f;
  return v;
}
template <int D, typename V>
__device__ __forceinline__ void product_by_rows(f32x4 (&o)[D / 16], const f16x8 (&ph)[2],
                                                const f16x8 (&pl)[2], uint64_t vis, int row,
                                                int quad, V frag) {
#pragma unroll
  for (int dt = 0; dt < D / 16; dt++) {
#pragma unroll 1
    for (int r = 0; r < ROWS; r++) {
      const uint64_t word = __shfl(vis, r);  // lane r holds row r's
      f32x4 acc = o[dt];
#pragma unroll
      for (int kc = 0; kc < 2; kc++) {
        const f16x8 v = seen_cells(frag(dt, kc), word, kc, quad);
        acc = mfma16(v, ph[kc], acc);
        acc = mfma16(v, pl[kc], acc);
      }
      if (row == r) o[dt] = acc;
    }
  }
}

// RING: a sliding-window plan. Items hold logical block ranges; logical
// block b of sequence s is ring entry b % ring, and row position p sees
// positions p - window + 1 .. p only. TREE: the plan of drafted trees
// (lgmlh_plan_tree). Blocks before npast / 64 are visible to every token; from
// there a token sees the cells of its words in vis (vis_words a token).
template <int D, bool RING, bool TREE = false>
__global__ void __launch_bounds__(64, D <= 128 ? 2 : 1)
paged_attn_kernel(const float *__restrict__ q, int H, int Hkv, float scale_log2,
                  const uint16_t *__restrict__ kpool, const uint16_t *__restrict__ vpool,
                  const int32_t *__restrict__ items, const int32_t *__restrict__ seq_off,
                  const int32_t *__restrict__ seq_npast, const int32_t *__restrict__ block_tab,
                  int max_blocks, int ring, int window, float *__restrict__ out,
                  f16 *__restrict__ planes, int64_t npad, int xf, float *__restrict__ part,
                  const int32_t *__restrict__ order, int n_order, const uint64_t *__restrict__ vis,
                  int vis_words) {
  // MFMA k-steps over D; a head of 16 takes one step of 32 whose upper
  // half is zero in K and Q (the lanes of quads 2 and 3 load nothing)
  constexpr int KS = D >= 32 ? D / 32 : 1;
  constexpr int DT = D / 16;   // d tiles of the output
  __shared__ __align__(16) f16x8 qsh[KS * 64], qsl[KS * 64];  // Q fragments, hi and lo

  const int lane = threadIdx.x;
  // a flat grid, KV heads fastest: workgroup w runs KV head w % Hkv of
  // slot w / Hkv, which is item order[slot] (slots past the order: item
  // slot)
  const int slot = (int)(blockIdx.x / (uint32_t)Hkv);
  const int kvh = (int)(blockIdx.x % (uint32_t)Hkv);
  const int item = order && slot < n_order ? order[slot] : slot;
  const int G = H / Hkv;
  const int s = items[4 * item + 0];
  const int tok0 = items[4 * item + 1];
  const int ntok = items[4 * item + 2] & 31;
  const int mg = (items[4 * item + 2] >> 5) - 1;  // merge group, -1: one split
  const int blo = items[4 * item + 3] & 0xffff;
  const int bhi = (items[4 * item + 3] >> 16) & 0xffff;

  const int row = lane & 15;       // the row this lane owns in S^T / O^T
  const int quad = lane >> 4;      // 0..3
  const int rtok = row / G;        // token of the row within the group
  const int rhead = kvh * G + row % G;
  const bool rvalid = rtok < ntok;
  const int p_first = seq_npast[s] + (tok0 - seq_off[s]);
  const int p_row = p_first + rtok;  // last visible position of the row

  const int b_tree = TREE ? seq_npast[s] / KV_BLOCK : 0;  // the first block that vis speaks of
  const uint64_t *vrow = TREE ? vis + (int64_t)(tok0 + (rvalid ? rtok : 0)) * vis_words : nullptr;

  const int32_t *bt = block_tab + (int64_t)s * max_blocks;
  auto phys = [&](int blk) -> int64_t { return RING ? bt[blk % ring] : bt[blk]; };
  auto ktile = [&](int blk) { return kpool + (phys(blk) * Hkv + kvh) * (int64_t)(64 * D); };
  auto vtile = [&](int blk) { return vpool + (phys(blk) * Hkv + kvh) * (int64_t)(64 * D); };
  // K rows (A operand of S^T = K Q^T) and V^T columns (A operand of
  // O^T += V^T P^T) of one block, straight from the pool tiles.
  f16x8 kf[4][KS], vf[DT][2];
  const bool kpart = D >= 32 || quad < 2;  // this lane's k range lies in the head
  auto load_k = [&](const uint16_t *kt) {
#pragma unroll
    for (int ct = 0; ct < 4; ct++)
#pragma unroll
      for (int ks = 0; ks < KS; ks++)
        kf[ct][ks] = kpart ? load_f16x8(kt + s_cell(ct, row) * D + ks * 32 + quad * 8)
                           : f16x8{0, 0, 0, 0, 0, 0, 0, 0};
  };
  auto load_v = [&](const uint16_t *vt) {
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
      for (int kc = 0; kc < 2; kc++) vf[dt][kc] = load_f16x8(vt + (dt * 16 + row) * 64 + kc * 32 + quad * 8);
  };
  // Q fragments (B operand): Q[row][ks*32 + quad*8 .. +7] as f16 hi + lo
  // (q = hi + lo to 22 bits; K is exact f16, so S^T is f32-accurate). Kept
  // in LDS to leave registers for the next block's tiles. Every lane
  // addresses a valid row (rows past the group read its last token and are
  // zeroed), so all pieces load together.
  {
    const int qt = rvalid ? rtok : ntok - 1;
    const float *qr = q + ((int64_t)(tok0 + qt) * H + rhead) * D;
    f32x4 qa[2 * KS];
#pragma unroll
    for (int ks = 0; ks < KS; ks++) {
      qa[2 * ks] = kpart ? *(const f32x4 *)(qr + ks * 32 + quad * 8) : f32x4{0, 0, 0, 0};
      qa[2 * ks + 1] = kpart ? *(const f32x4 *)(qr + ks * 32 + quad * 8 + 4) : f32x4{0, 0, 0, 0};
    }
    // The first block's tiles go out before the Q pieces are converted,
    // so the two loads overlap. Unconditional, so that the conversion waits
    // for the Q pieces only (a run always has a block; block 0 of every
    // planned sequence is a valid pool block).
    const int b_first = blo < bhi ? blo : 0;
    load_k(ktile(b_first));
    load_v(vtile(b_first));
#pragma unroll
    for (int ks = 0; ks < KS; ks++) {
      f16x8 h, lo;
      const f32x4 a = rvalid ? qa[2 * ks] : f32x4{0, 0, 0, 0};
      const f32x4 b = rvalid ? qa[2 * ks + 1] : f32x4{0, 0, 0, 0};
#pragma unroll
      for (int e = 0; e < 4; e++) {
        h[e] = (f16)a[e];
        lo[e] = (f16)(a[e] - (float)h[e]);
        h[4 + e] = (f16)b[e];
        lo[4 + e] = (f16)(b[e] - (float)h[4 + e]);
      }
      qsh[ks * 64 + lane] = h;
      qsl[ks * 64 + lane] = lo;
    }
  }

  f32x4 o[DT];
#pragma unroll
  for (int i = 0; i < DT; i++) o[i] = f32x4{0, 0, 0, 0};
  float m = -INFINITY, l = 0.0f;

  // One block; NEXT: the next block's tiles are loaded meanwhile
  // (straight-line code keeps the load counter waits exact, so the O
  // products do not wait for the next K). Heads of up to 128 run the last
  // block without NEXT, so no tile is loaded twice; heads of 256 (whose
  // registers are full) load the last block's tiles again, from L2. Their O
  // products stay behind the softmax: with the schedule free, tiles in flight
  // spilled, and a spill waits for them (214 -> 260 us at 32 sequences of
  // U[1024, 16384]); held in program order after S and after O too, a chain of
  // few blocks is longer (one sequence of 2386 cells 43.7 us, 38.6 so).
  constexpr bool PEEL = D <= 128;
  auto block = [&](int blk, auto next) __attribute__((always_inline)) {
    constexpr bool NEXT = decltype(next)::value;
    const int nxt = blk + 1 < bhi ? blk + 1 : blk;
    // S^T[cell][row] for 4 tiles of 16 cells.
    f32x4 st[4];
#pragma unroll
    for (int ct = 0; ct < 4; ct++) {
      f32x4 acc = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int ks = 0; ks < KS; ks++) {
        acc = mfma16(kf[ct][ks], qsh[ks * 64 + lane], acc);
        acc = mfma16(kf[ct][ks], qsl[ks * 64 + lane], acc);
      }
      st[ct] = acc;
    }
    if constexpr (NEXT) load_k(ktile(nxt));

    // A block that ends at or before the group's first position (and, with a
    // window, starts inside the window of its last) is visible to every
    // valid row.
    const int cbase = blk * 64;
    bool full = cbase + 63 <= p_first && (!RING || cbase > p_first + ntok - 1 - window);
    if constexpr (TREE) {
      // every block here; not known when compiled, so that the scores are rounded
      // before the maximum is taken off as in the other plans (a line of tokens
      // has the bits of the causal plan)
      int all = 1;
      asm volatile("" : "+s"(all));
      full = all != 0;
    }
    f16x8 pfh[2], pfl[2];
    softmax_block<DT>(st, scale_log2, full, cbase, quad, p_row, RING ? p_row - window + 1 : 0,
                      rvalid, 0, m, l, o, pfh, pfl);
    if constexpr (!PEEL) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
      for (int kc = 0; kc < 2; kc++) {
        o[dt] = mfma16(vf[dt][kc], pfh[kc], o[dt]);
        o[dt] = mfma16(vf[dt][kc], pfl[kc], o[dt]);
      }
    if constexpr (NEXT) load_v(vtile(nxt));
  };
  // A block with tokens of the pass (TREE), its tiles loaded: nothing is loaded
  // ahead, so that the tiles in flight and the rows of product_by_rows do not
  // want registers at once. A sequence has one or two.
  auto tree_block = [&](int blk) __attribute__((always_inline)) {
    f32x4 st[4];
#pragma unroll
    for (int ct = 0; ct < 4; ct++) {
      st[ct] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int ks = 0; ks < KS; ks++) {
        st[ct] = mfma16(kf[ct][ks], qsh[ks * 64 + lane], st[ct]);
        st[ct] = mfma16(kf[ct][ks], qsl[ks * 64 + lane], st[ct]);
      }
    }
    const uint64_t word = rvalid ? vrow[blk - b_tree] : 0;
    f16x8 pfh[2], pfl[2];
    softmax_block<DT, true>(st, scale_log2, false, blk * 64, quad, 0, 0, rvalid, word, m, l, o, pfh,
                            pfl);
    bool bad = false;
#pragma unroll
    for (int dt = 0; dt < DT; dt++) bad |= not_finite(vf[dt][0]) || not_finite(vf[dt][1]);
    if (__builtin_amdgcn_ballot_w64(bad)) {
      const uint16_t *vt = vtile(blk);  // read again: the fragments are addressed by row here
      product_by_rows<D>(o, pfh, pfl, word, row, quad, [&](int dt, int kc) {
        int at = (dt * 16 + row) * 64 + kc * 32 + quad * 8;
        asm volatile("" : "+v"(at));  // made here, not ahead of the loops for every dt and kc
        return load_f16x8(vt + at);
      });
    } else {
#pragma unroll
      for (int dt = 0; dt < DT; dt++)
#pragma unroll
        for (int kc = 0; kc < 2; kc++) {
          o[dt] = mfma16(vf[dt][kc], pfh[kc], o[dt]);
          o[dt] = mfma16(vf[dt][kc], pfl[kc], o[dt]);
        }
    }
  };
  const int bend = TREE && b_tree < bhi ? b_tree : bhi;  // blocks from here on are a tree's
  int blk = blo;
  for (; blk + (PEEL && bend == bhi ? 1 : 0) < bend; blk++) block(blk, std::true_type{});
  if constexpr (PEEL)
    if (blk < bend) block(blk, std::false_type{});
  if constexpr (TREE)
    for (blk = blo > b_tree ? blo : b_tree; blk < bhi; blk++) {
      tree_block(blk);
      if (blk + 1 < bhi) {
        load_k(ktile(blk + 1));
        load_v(vtile(blk + 1));
      }
    }

  finish_item<D>(o, m, l * ATTN_P, mg, rvalid, tok0, rtok, rhead, ntok, G, row, quad, item, kvh, Hkv, H,
                 out, planes, npad, xf, part);
}

// Shared runs (a prompt chunk's query groups in sets, lgmlh_plan): one
// workgroup of SHARED_WAVES waves per (run, KV head), wave w on item
// first + w (w < n). Each K / V block of the run is loaded once into LDS
// (global-to-LDS, the next block's loads in flight while this one is
// used) and every wave reads its MFMA fragments from there: the context
// of a chunk is read once per set instead of once per group. (W waves: a tree
// plan's sets of up to half as many items take workgroups of half as many
// waves, two to a CU; a larger set then takes two. Trees of 16 tokens of 32
// sequences at 128 to 4096 cells, 32 / 8 heads of 128: a pass 95 us in
// workgroups of eight waves, 76 so, with the merge's four loads below; 65 of them
// here, HBM's reads, 80 where the cells are in no cache.) The
// arithmetic of a wave is the per-item kernel's (same fragments, same
// order), so an item gives the same bits in either kernel. A block past a
// wave's last position is skipped (it would add nothing).
// LDS slots of 16 B: K slot (r, c) = row r (cell), chunk c of D / 8 holds
// the pool's chunk c ^ swk(r); V slot (r, c) = row r (d), chunk c of 8
// (cells) holds chunk c ^ swv(r): a 16-row fragment read touches every
// bank once.
constexpr int SHARED_WAVES = ATTN_SHARED;

template <int D, bool TREE = false, int W = SHARED_WAVES>
__global__ void __launch_bounds__(64 * W, 2)
paged_attn_shared_kernel(const float *__restrict__ q, int H, int Hkv, float scale_log2,
                         const uint16_t *__restrict__ kpool, const uint16_t *__restrict__ vpool,
                         const int32_t *__restrict__ items, const int32_t *__restrict__ shared,
                         const int32_t *__restrict__ seq_off, const int32_t *__restrict__ seq_npast,
                         const int32_t *__restrict__ block_tab, int max_blocks,
                         float *__restrict__ out, f16 *__restrict__ planes, int64_t npad,
                         int xf, float *__restrict__ part, const uint64_t *__restrict__ vis,
                         int vis_words) {
  constexpr int KS = D / 32, DT = D / 16;
  constexpr int TILE = 64 * D;             // f16 of one K (or V) tile
  constexpr int KC = D / 8;                // 16-byte chunks per K row
  constexpr int LOADS = TILE / 8 / (64 * W);  // per lane and tile
  __shared__ __align__(16) uint16_t kb0[TILE], kb1[TILE], vb0[TILE], vb1[TILE];
  typedef __attribute__((address_space(3))) void lds_t;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = W < SHARED_WAVES ? (int)blockIdx.z * W : 0;
  const int first = shared[2 * blockIdx.x] + half, n = shared[2 * blockIdx.x + 1] - half;
  if (W < SHARED_WAVES && n <= 0) return;  // a set of one half
  const int kvh = blockIdx.y;
  const int G = H / Hkv;
  const bool active = wave < n;
  const int item = first + (active ? wave : 0);
  const int s = items[4 * first + 0];
  const int blo = items[4 * first + 3] & 0xffff;
  const int bhi = (items[4 * first + 3] >> 16) & 0xffff;
  const int tok0 = items[4 * item + 1];
  const int ntok = items[4 * item + 2] & 31;
  const int mg = (items[4 * item + 2] >> 5) - 1;

  const int row = lane & 15, quad = lane >> 4;
  const int rtok = row / G;
  const int rhead = kvh * G + row % G;
  const bool rvalid = rtok < ntok;
  const int p_first = seq_npast[s] + (tok0 - seq_off[s]);
  const int p_row = p_first + rtok;
  const int p_last = p_first + ntok - 1;  // the wave's last position
  const int b_tree = TREE ? seq_npast[s] / KV_BLOCK : 0;
  const uint64_t *vrow = TREE ? vis + (int64_t)(tok0 + (rvalid ? rtok : 0)) * vis_words : nullptr;

  // Q fragments in registers: Q[row][ks*32 + quad*8 .. +7] as f16 hi + lo
  f16x8 qh[KS], ql[KS];
  {
    const int qt = rvalid ? rtok : ntok - 1;
    const float *qr = q + ((int64_t)(tok0 + qt) * H + rhead) * D;
#pragma unroll
    for (int ks = 0; ks < KS; ks++) {
      const f32x4 a = rvalid ? *(const f32x4 *)(qr + ks * 32 + quad * 8) : f32x4{0, 0, 0, 0};
      const f32x4 b = rvalid ? *(const f32x4 *)(qr + ks * 32 + quad * 8 + 4) : f32x4{0, 0, 0, 0};
#pragma unroll
      for (int e = 0; e < 4; e++) {
        qh[ks][e] = (f16)a[e];
        ql[ks][e] = (f16)(a[e] - (float)qh[ks][e]);
        qh[ks][4 + e] = (f16)b[e];
        ql[ks][4 + e] = (f16)(b[e] - (float)qh[ks][4 + e]);
      }
    }
  }

  f32x4 o[DT];
#pragma unroll
  for (int i = 0; i < DT; i++) o[i] = f32x4{0, 0, 0, 0};
  float m = -INFINITY, l = 0.0f;

  const int32_t *bt = block_tab + (int64_t)s * max_blocks;
  // Global-to-LDS loads of block blk into buffer buf: load j of this lane
  // fills slot (j * W + wave) * 64 + lane of each tile.
  auto load = [&](int blk, int buf) {
    const int64_t base = ((int64_t)bt[blk] * Hkv + kvh) * TILE;
    uint16_t *kd = buf ? kb1 : kb0, *vd = buf ? vb1 : vb0;
#pragma unroll
    for (int j = 0; j < LOADS; j++) {
      const int slot0 = (j * W + wave) * 64, sl = slot0 + lane;
      const int kr = sl / KC, kc = (sl % KC) ^ swk<D>(sl / KC);
      const int vr = sl / 8, vc = (sl % 8) ^ swv(sl / 8);
      __builtin_amdgcn_global_load_lds((const void *)(kpool + base + kr * D + kc * 8),
                                       (lds_t *)(kd + slot0 * 8), 16, 0, 0);
      __builtin_amdgcn_global_load_lds((const void *)(vpool + base + vr * 64 + vc * 8),
                                       (lds_t *)(vd + slot0 * 8), 16, 0, 0);
    }
  };
  if (blo < bhi) {
    load(blo, 0);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
  }
  for (int blk = blo; blk < bhi; blk++) {
    const int buf = (blk - blo) & 1;
    if (blk + 1 < bhi) load(blk + 1, buf ^ 1);  // into the buffer freed by the last barrier
    const int cbase = blk * 64;
    if (active && cbase <= p_last) {
      const uint16_t *kt = buf ? kb1 : kb0, *vt = buf ? vb1 : vb0;
      // S^T[cell][row] for 4 tiles of 16 cells; K fragments from LDS, the
      // next step's read while one multiplies
      f32x4 st[4];
      f16x8 kf[2][4];
      auto read_k = [&](int ks, f16x8(&f)[4]) __attribute__((always_inline)) {
#pragma unroll
        for (int ct = 0; ct < 4; ct++) {
          const int r = s_cell(ct, row);
          f[ct] = load_f16x8(kt + (r * KC + ((ks * 4 + quad) ^ swk<D>(r))) * 8);
        }
      };
      read_k(0, kf[0]);
#pragma unroll
      for (int ks = 0; ks < KS; ks++) {
        if (ks + 1 < KS) read_k(ks + 1, kf[(ks + 1) & 1]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int ct = 0; ct < 4; ct++)
          st[ct] = mfma16(kf[ks & 1][ct], qh[ks], ks ? st[ct] : f32x4{0, 0, 0, 0});
#pragma unroll
        for (int ct = 0; ct < 4; ct++) st[ct] = mfma16(kf[ks & 1][ct], ql[ks], st[ct]);
        __builtin_amdgcn_sched_barrier(0);
      }
      f16x8 pfh[2], pfl[2];
      const bool full = TREE ? blk < b_tree : cbase + 63 <= p_first;
      uint64_t word = 0;
      if (TREE && !full && rvalid) word = vrow[blk - b_tree];
      softmax_block<DT, TREE>(st, scale_log2, full, cbase, quad, p_row, 0, rvalid, word, m, l, o, pfh,
                              pfl);
      bool by_rows = false;
      if constexpr (TREE) {
        if (!full) {
          auto frag = [&](int dt, int kc) {
            const int r = dt * 16 + row;
            int at = (r * 8 + ((kc * 4 + quad) ^ swv(r))) * 8;
            asm volatile("" : "+v"(at));  // made here, not ahead of the loops
            return load_f16x8(vt + at);
          };
          bool bad = false;
#pragma unroll 1
          for (int dt = 0; dt < DT; dt++) bad |= not_finite(frag(dt, 0)) || not_finite(frag(dt, 1));
          by_rows = __builtin_amdgcn_ballot_w64(bad) != 0;
          if (by_rows) product_by_rows<D>(o, pfh, pfl, word, row, quad, frag);
        }
      }
      // O^T += V^T P^T, two d tiles at a time, the next two read meanwhile
      f16x8 vf[2][2][2];
      auto read_v = [&](int dt, f16x8(&f)[2][2]) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
          for (int kc = 0; kc < 2; kc++) {
            const int r = (dt + t) * 16 + row;
            f[t][kc] = load_f16x8(vt + (r * 8 + ((kc * 4 + quad) ^ swv(r))) * 8);
          }
      };
      if (!TREE || !by_rows) {
        read_v(0, vf[0]);
#pragma unroll
        for (int dt = 0; dt < DT; dt += 2) {
          const int b = dt >> 1 & 1;
          if (dt + 2 < DT) read_v(dt + 2, vf[b ^ 1]);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int kc = 0; kc < 2; kc++) {
            o[dt] = mfma16(vf[b][0][kc], pfh[kc], o[dt]);
            o[dt + 1] = mfma16(vf[b][1][kc], pfh[kc], o[dt + 1]);
            o[dt] = mfma16(vf[b][0][kc], pfl[kc], o[dt]);
            o[dt + 1] = mfma16(vf[b][1][kc], pfl[kc], o[dt + 1]);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
    __builtin_amdgcn_s_waitcnt(0);  // this wave's loads of blk + 1 have landed
    __syncthreads();                // ... and everyone's; buffer buf is free again
  }
  if (!active) return;
  finish_item<D>(o, m, l * ATTN_P, mg, rvalid, tok0, rtok, rhead, ntok, G, row, quad, item, kvh, Hkv, H,
                 out, planes, npad, xf, part);
}

// Fixed-order merge of the splits of one token group (merge group: first
// item, splits, first token, tokens), one workgroup of MERGE_THREADS per
// (group, KV head). Each thread holds a position of 4 output columns (up to
// 4 per round); for each it loads, in one go per SC splits, the split
// outputs with the m and l of the position's row, and finds the row's max
// M, the split weights w = exp2(m - M) and L = sum l w itself (the threads
// of a row agree), adding the outputs weighted, in split order. A merge of
// up to SC splits is one round trip; with 4 or fewer SC is 4, else 16 (the loads
// past the last split repeat it).
// SPREAD (Q4_0 pools): the positions are gridDim.z workgroups', one a thread; SLICES > 1
// (more than 16 splits): a wave's positions, their splits in as many runs, a wave each,
// with a maximum of its own as it goes (one round trip per SC splits), and the runs join
// in order. A step of 4 sequences at 32768 to 131072 cells, 32 / 4 heads of 128, 43 to 171
// splits: 9 us, where one workgroup for all positions and splits took 24.
constexpr int MERGE_THREADS = 256, MERGE_SLICES = 4;
template <int D, int SC, bool SPREAD = false, int SLICES = 1>
__device__ __forceinline__ void merge_group(const int32_t *__restrict__ merge, int H, int Hkv,
                                            const float *__restrict__ part, float *__restrict__ out,
                                            f16 *__restrict__ planes, int64_t npad, int xf) {
  constexpr int MT = MERGE_THREADS / SLICES, NJ = SPREAD ? 1 : 4;
  const int tid = SLICES > 1 ? threadIdx.x % MT : threadIdx.x, lane = tid & 63, mg = blockIdx.x, kvh = blockIdx.y;
  const int first = merge[4 * mg + 0], ns = merge[4 * mg + 1];
  const int tok0 = merge[4 * mg + 2], ntok = merge[4 * mg + 3] & 0xff;
  const int stride = merge[4 * mg + 3] >> 8;  // items from one split to the next
  const int G = H / Hkv, nrows = ntok * G;
  const float *p0 = part + ((int64_t)first * Hkv + kvh) * Partial<D>::floats;
  const int64_t pstride = (int64_t)stride * Hkv * Partial<D>::floats;
  const float *ml = p0 + ROWS * D;  // m of row r at ml[r], l at ml[ROWS + r]
  const int n4 = nrows * (D / 4);
  const int base0 = SPREAD ? blockIdx.z * MT : 0;
  for (int base = base0; base < n4; base += SPREAD ? gridDim.z * MT : NJ * MT) {
    const int nj = min(NJ, (n4 - base + MT - 1) / MT);  // workgroup-uniform
    int rr[NJ], dd[NJ];
    f32x4 acc[NJ];
    float M[NJ], L[NJ];
#pragma unroll
    for (int jj = 0; jj < NJ; jj++) {
      const int e4 = min(base + tid + MT * jj, n4 - 1);
      rr[jj] = e4 / (D / 4);
      dd[jj] = 4 * (e4 % (D / 4));
      acc[jj] = f32x4{0, 0, 0, 0};
      M[jj] = -INFINITY;
      L[jj] = 0.0f;
    }
    if constexpr (SLICES > 1) {
      __shared__ f32x4 slice_acc[SLICES - 1][MT];
      __shared__ float slice_m[SLICES - 1][MT], slice_l[SLICES - 1][MT];
      const int slice = threadIdx.x / MT, run = (ns + SLICES - 1) / SLICES;
      const int last = min(ns, (slice + 1) * run);
      for (int s0 = slice * run; s0 < last; s0 += SC) {
        f32x4 a[SC];
        float mv[SC], lv[SC];
#pragma unroll
        for (int i = 0; i < SC; i++) {
          const int64_t o = (int64_t)min(s0 + i, last - 1) * pstride;
          a[i] = *(const f32x4 *)(p0 + o + rr[0] * D + dd[0]);
          mv[i] = ml[o + rr[0]];
          lv[i] = ml[o + ROWS + rr[0]];
        }
        float top = M[0];
#pragma unroll
        for (int i = 0; i < SC; i++) top = fmaxf(top, mv[i]);
        if (top == -INFINITY) continue;  // splits that saw no cell
        const float w = exp2f(M[0] - top);
        L[0] *= w;
        acc[0] *= w;
#pragma unroll
        for (int i = 0; i < SC; i++)
          if (s0 + i < last) {
            const float w = exp2f(mv[i] - top);
            L[0] += lv[i] * w;
            acc[0] += a[i] * w;
          }
        M[0] = top;
      }
      if (base > base0) __syncthreads();  // the last positions' are read
      if (slice > 0) {
        slice_acc[slice - 1][tid] = acc[0];
        slice_m[slice - 1][tid] = M[0];
        slice_l[slice - 1][tid] = L[0];
      }
      __syncthreads();
      if (slice > 0) continue;
#pragma unroll
      for (int i = 0; i < SLICES - 1; i++) {
        const float m = slice_m[i][tid], top = fmaxf(M[0], m);
        if (top == -INFINITY) continue;
        const float w = exp2f(M[0] - top), w1 = exp2f(m - top);
        L[0] = L[0] * w + slice_l[i][tid] * w1;
        acc[0] = acc[0] * w + slice_acc[i][tid] * w1;
        M[0] = top;
      }
    } else {
      // More than SC splits: the maxima first, over every split's m.
      if (ns > SC)
        for (int s0 = 0; s0 < ns; s0 += SC) {
#pragma unroll
          for (int jj = 0; jj < NJ; jj++)
            if (jj < nj) {
              float mv[SC];
#pragma unroll
              for (int i = 0; i < SC; i++) mv[i] = ml[(int64_t)min(s0 + i, ns - 1) * pstride + rr[jj]];
#pragma unroll
              for (int i = 0; i < SC; i++) M[jj] = fmaxf(M[jj], mv[i]);  // repeats: same max
            }
        }
      for (int s0 = 0; s0 < ns; s0 += SC) {
#pragma unroll
        for (int jj = 0; jj < NJ; jj++)
          if (jj < nj) {
            f32x4 a[SC];
            float mv[SC], lv[SC];
#pragma unroll
            for (int i = 0; i < SC; i++) {
              const int64_t o = (int64_t)min(s0 + i, ns - 1) * pstride;
              a[i] = *(const f32x4 *)(p0 + o + rr[jj] * D + dd[jj]);
              mv[i] = ml[o + rr[jj]];
              lv[i] = ml[o + ROWS + rr[jj]];
            }
            if (ns <= SC)
#pragma unroll
              for (int i = 0; i < SC; i++) M[jj] = fmaxf(M[jj], mv[i]);
#pragma unroll
            for (int i = 0; i < SC; i++)
              if (s0 + i < ns) {
                const float w = exp2f(mv[i] - M[jj]);  // 0 for a split that saw no cell
                L[jj] += lv[i] * w;
                acc[jj] += a[i] * w;
              }
          }
      }
    }
#pragma unroll
    for (int jj = 0; jj < NJ; jj++) {
      const int e4 = base + tid + MT * jj;
      // groups of 8 lanes (D / 4 is a multiple of 8) leave together, and
      // whole waves where a wave holds a Q8_K block (n4 a multiple of 64)
      if (jj >= nj || e4 >= n4) continue;
      const int r = rr[jj], d0 = dd[jj];
      const f32x4 y = acc[jj] / L[jj];
      const int64_t n = tok0 + r / G, k = (int64_t)(kvh * G + r % G) * D + d0;
      if (planes && xf == XF_Q8K) {
        // the 64 lanes hold one Q8_K block (whole chunks: G D % 256 == 0),
        // value 4 lane + i of the block; the steps of finish_q8k
        const int64_t K = (int64_t)H * D;
        float amax = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; i++) amax = fmaxf(amax, fabsf(y[i]));
        amax = group_max<64>(amax);
        const float yv[4] = {y[0], y[1], y[2], y[3]};
        const float mx = group_first_abs<64, 4>(yv, amax);
        const float iscale = amax == 0.0f ? 0.0f : -127.0f / mx;
        float qv[4], s = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          qv[i] = amax == 0.0f ? 0.0f : fminf(127.0f, __builtin_rintf(iscale * y[i]));
          s += qv[i];
        }
        s += dpp_f<DPP_XOR1>(s);
        s += dpp_f<DPP_XOR2>(s);
        *(f16x4 *)(planes + n * K + k) = f16x4{(f16)qv[0], (f16)qv[1], (f16)qv[2], (f16)qv[3]};
        if ((lane & 3) == 0) planes[q8_bs_off(npad, K) + n * (K / 16) + (k >> 4)] = (f16)s;
        if (lane == 0) {
          float *dp = (float *)((char *)planes + q8_d_off(npad, K));
          dp[n * (K / 256) + (k >> 8)] = amax == 0.0f ? 0.0f : 1.0f / iscale;
        }
      } else if (planes && xf == XF_Q80) {
        // 8 lanes hold a Q8_0 block (32 values); the steps of q80_block8
        const int64_t K = (int64_t)H * D;
        float amax = fmaxf(fmaxf(fabsf(y[0]), fabsf(y[1])), fmaxf(fabsf(y[2]), fabsf(y[3])));
        amax = group_max<8>(amax);
        const float dd = amax / 127.0f;
        const float id = dd != 0.0f ? 1.0f / dd : 0.0f;
        *(f16x4 *)(planes + n * K + k) =
            f16x4{(f16)__builtin_roundf(y[0] * id), (f16)__builtin_roundf(y[1] * id),
                  (f16)__builtin_roundf(y[2] * id), (f16)__builtin_roundf(y[3] * id)};
        if ((e4 & 7) == 0) {
          float *dp = (float *)((char *)planes + q8_d_off(npad, K));
          dp[n * (K / 32) + (k >> 5)] = (float)(f16)dd;
        }
      } else if (planes) {
        // 8 lanes hold a 32-value group
        const int64_t K = (int64_t)H * D;
        const float v[4] = {y[0], y[1], y[2], y[3]};
        split_store4(planes, npad, K, n, k, v);
        float s = v[0] + v[1] + v[2] + v[3];
        s += dpp_f<DPP_XOR1>(s);
        s += dpp_f<DPP_XOR2>(s);
        s += __shfl_xor(s, 4);
        if ((e4 & 7) == 0) split_store_gsum(planes, npad, K, n, k >> 5, s);
      } else {
        *(f32x4 *)(out + n * H * D + k) = y;
      }
    }
  }
}

template <int D>
__global__ void __launch_bounds__(MERGE_THREADS)
merge_kernel(const int32_t *__restrict__ merge, int H, int Hkv, const float *__restrict__ part,
             float *__restrict__ out, f16 *__restrict__ planes, int64_t npad, int xf) {
  if (merge[4 * blockIdx.x + 1] <= 4)
    merge_group<D, 4>(merge, H, Hkv, part, out, planes, npad, xf);
  else
    merge_group<D, 16>(merge, H, Hkv, part, out, planes, npad, xf);
}
template <int D>
__global__ void __launch_bounds__(MERGE_THREADS)
merge_slices_kernel(const int32_t *__restrict__ merge, int H, int Hkv, const float *__restrict__ part,
                    float *__restrict__ out, f16 *__restrict__ planes, int64_t npad, int xf) {
  const int ns = merge[4 * blockIdx.x + 1];
  if (ns <= 4)
    merge_group<D, 4, true>(merge, H, Hkv, part, out, planes, npad, xf);
  else if (ns <= 16)
    merge_group<D, 16, true>(merge, H, Hkv, part, out, planes, npad, xf);
  else
    merge_group<D, 16, true, MERGE_SLICES>(merge, H, Hkv, part, out, planes, npad, xf);
}

}  // namespace lgmlh

using namespace lgmlh;

extern "C" size_t lgmlh_attention_workspace(const lgmlh_plan_info *info, int head_dim) {
  if (!info) return 0;
  return (size_t)info->n_items * info->n_head_kv * (ROWS * head_dim + 2 * ROWS) * sizeof(float);
}

template <int D>
static void launch_merge(const lgmlh_ubatch *ub, int H, int Hkv, const float *part, float *out,
                         f16 *planes, int64_t npad, int xf, hipStream_t st) {
  hipLaunchKernelGGL(merge_kernel<D>, dim3(ub->n_merge, Hkv), dim3(MERGE_THREADS), 0, st, ub->merge,
                     H, Hkv, part, out, planes, npad, xf);
}

void lgmlh::merge_slices_dev(int head_dim, const lgmlh_ubatch *ub, int H, int Hkv, const float *part,
                             float *out, f16 *planes, int64_t npad, int xf, hipStream_t st) {
  if (ub->n_merge <= 0) return;
  const auto kern = head_dim == 64 ? merge_slices_kernel<64> : head_dim == 128 ? merge_slices_kernel<128>
                                                                               : merge_slices_kernel<256>;
  // (for 8 rows' positions in slices in one turn; other groups' are a half of that)
  hipLaunchKernelGGL(kern, dim3(ub->n_merge, Hkv, head_dim / 32), dim3(MERGE_THREADS), 0, st, ub->merge, H, Hkv, part, out,
                     planes, npad, xf);
}

void lgmlh::merge_dev(int head_dim, const lgmlh_ubatch *ub, int H, int Hkv, const float *part,
                      float *out, f16 *planes, int64_t npad, int xf, hipStream_t st) {
  if (ub->n_merge <= 0) return;
  switch (head_dim) {
    case 16: launch_merge<16>(ub, H, Hkv, part, out, planes, npad, xf, st); break;
    case 32: launch_merge<32>(ub, H, Hkv, part, out, planes, npad, xf, st); break;
    case 64: launch_merge<64>(ub, H, Hkv, part, out, planes, npad, xf, st); break;
    case 128: launch_merge<128>(ub, H, Hkv, part, out, planes, npad, xf, st); break;
    case 256: launch_merge<256>(ub, H, Hkv, part, out, planes, npad, xf, st); break;
  }
}

template <int D>
static void launch_attn(const float *q, int H, int Hkv, float scale_log2, const void *kp,
                        const void *vp, const lgmlh_ubatch *ub, float *out, f16 *planes,
                        int64_t npad, int xf, float *part, hipStream_t st) {
  const bool tree = ub->ring == LGMLH_PLAN_TREE;
  const uint64_t *vis = tree ? plan_vis(ub) : nullptr;
  // one workgroup per (item, KV head), the items on their own in the
  // plan's order
  if (ub->ring > 0)
    hipLaunchKernelGGL((paged_attn_kernel<D, true>), dim3((uint32_t)ub->n_single * Hkv),
                       dim3(64), 0, st, q, H, Hkv, scale_log2, (const uint16_t *)kp,
                       (const uint16_t *)vp, ub->items, ub->seq_off, ub->seq_npast, ub->block_tab,
                       ub->max_blocks, ub->ring, ub->window, out, planes, npad, xf, part,
                       ub->order, ub->n_single, nullptr, 0);
  // heads of 256, and of 32 or less, run the shared runs' items with the
  // per-item kernel too
  else if (const int n1 = D <= 128 && D >= 64 ? ub->n_single : ub->n_items; n1 > 0) {
    const auto kern = tree ? paged_attn_kernel<D, false, true> : paged_attn_kernel<D, false, false>;
    hipLaunchKernelGGL(kern, dim3((uint32_t)n1 * Hkv), dim3(64), 0, st, q, H, Hkv, scale_log2,
                       (const uint16_t *)kp, (const uint16_t *)vp, ub->items, ub->seq_off,
                       ub->seq_npast, ub->block_tab, ub->max_blocks, 0, 0, out, planes, npad, xf,
                       part, ub->order, ub->n_single, vis, ub->window);
  }
  if (ub->ring <= 0 && ub->n_shared > 0) {
    if constexpr (D <= 128 && D >= 64) {
      constexpr int HALF = SHARED_WAVES / 2;
      const bool small = tree && ub->n_items - ub->n_single <= HALF * ub->n_shared;
      const auto kern = small  ? paged_attn_shared_kernel<D, true, HALF>
                        : tree ? paged_attn_shared_kernel<D, true>
                               : paged_attn_shared_kernel<D, false>;
      hipLaunchKernelGGL(kern, dim3(ub->n_shared, Hkv, small ? 2 : 1),
                         dim3(64 * (small ? HALF : SHARED_WAVES)), 0, st, q, H, Hkv, scale_log2,
                         (const uint16_t *)kp, (const uint16_t *)vp, ub->items, ub->shared,
                         ub->seq_off, ub->seq_npast, ub->block_tab, ub->max_blocks, out, planes,
                         npad, xf, part, vis, ub->window);
    }
  }
  merge_dev(D, ub, H, Hkv, part, out, planes, npad, xf, st);
}

namespace lgmlh {
// The attention output as f32 rows (out) or, with planes set, as the
// output product's X in the form xf (rows padded to npad): XF_SPLIT split
// planes or XF_Q80 blocks (heads of 32 or more), or XF_Q8K blocks when a
// block's 256 / D heads are of one KV head's group (heads of 64 or more,
// G % (256 / D) == 0: attn_q8k_fits).
bool attn_q8k_fits(int head_dim, int G) {
  return head_dim >= 64 && head_dim <= 256 && G % (256 / head_dim) == 0;
}

// The checks of an attention call (16 rows a wave); *run: there is work.
int attn_check(const char *what, const float *q, int n_head, int n_head_kv, int head_dim,
               const void *kpool, const void *vpool, const lgmlh_ubatch *ub, const float *out,
               const f16 *planes, int xf, const void *workspace, size_t workspace_bytes, int *run) {
  if (!q || !kpool || !vpool || !ub || !(out || planes) || n_head_kv <= 0 ||
      n_head <= 0 || n_head % n_head_kv) {
    set_error("%s: bad arguments", what);
    return LGMLH_EINVAL;
  }
  int G = n_head / n_head_kv;
  if (G > ROWS || ROWS % G || ub->rows != ROWS || ub->n_head_kv != n_head_kv) {
    set_error("%s: %d query heads per KV head does not match the plan", what, G);
    return LGMLH_EINVAL;
  }
  size_t need = (size_t)ub->n_items * n_head_kv * (ROWS * head_dim + 2 * ROWS) * sizeof(float);
  if (ub->n_merge > 0 && (!workspace || workspace_bytes < need)) {
    set_error("%s: workspace of %zu bytes, need %zu", what, workspace_bytes, need);
    return LGMLH_ENOMEM;
  }
  *run = ub->n_items > 0;
  if (!*run) return LGMLH_OK;
  if ((int64_t)ub->n_items * n_head_kv > (int64_t)1 << 25) {  // the per-item grid's threads
    set_error("%s: %d items x %d KV heads in one launch", what, ub->n_items, n_head_kv);
    return LGMLH_EINVAL;
  }
  if (planes && (xf == XF_Q8K ? !attn_q8k_fits(head_dim, G) : head_dim < 32)) {
    set_error("%s: heads of %d (%d per KV head) cannot write X form %d", what, head_dim,
              G, xf);
    return LGMLH_EINVAL;
  }
  return LGMLH_OK;
}

int paged_attention_dev(const float *q, int n_head, int n_head_kv, int head_dim, float scale,
                        const void *kpool, const void *vpool, const lgmlh_ubatch *ub, float *out,
                        f16 *planes, int64_t npad, void *workspace, size_t workspace_bytes,
                        hipStream_t st, int xf) {
  int run = 0;
  LGMLH_TRY(attn_check("paged_attention", q, n_head, n_head_kv, head_dim, kpool, vpool, ub, out,
                       planes, xf, workspace, workspace_bytes, &run));
  if (!run) return LGMLH_OK;
  float sl = scale * LOG2E;
  float *part = (float *)workspace;
  switch (head_dim) {
    case 16: launch_attn<16>(q, n_head, n_head_kv, sl, kpool, vpool, ub, out, planes, npad, xf, part, st); break;
    case 32: launch_attn<32>(q, n_head, n_head_kv, sl, kpool, vpool, ub, out, planes, npad, xf, part, st); break;
    case 64: launch_attn<64>(q, n_head, n_head_kv, sl, kpool, vpool, ub, out, planes, npad, xf, part, st); break;
    case 128: launch_attn<128>(q, n_head, n_head_kv, sl, kpool, vpool, ub, out, planes, npad, xf, part, st); break;
    case 256: launch_attn<256>(q, n_head, n_head_kv, sl, kpool, vpool, ub, out, planes, npad, xf, part, st); break;
    default:
      set_error("paged_attention: head_dim %d not supported (16, 32, 64, 128, 256)", head_dim);
      return LGMLH_EINVAL;
  }
  return hip_check(hipGetLastError(), "paged_attention");
}
}  // namespace lgmlh

extern "C" int lgmlh_paged_attention(const float *q, int n_head, int n_head_kv, int head_dim,
                                     float scale, const void *kpool, const void *vpool,
                                     const lgmlh_ubatch *ub, float *out, void *workspace,
                                     size_t workspace_bytes, void *stream) {
  if (!out) {
    set_error("paged_attention: bad arguments");
    return LGMLH_EINVAL;
  }
  return paged_attention_dev(q, n_head, n_head_kv, head_dim, scale, kpool, vpool, ub, out,
                             nullptr, 0, workspace, workspace_bytes, as_stream(stream), XF_SPLIT);
}
