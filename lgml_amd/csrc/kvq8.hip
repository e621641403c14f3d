// The KV pool in Q8_0 (8-bit values, an f16 scale per 32), and moves of cells
// within a pool of either type (gfx950).
#include <stdlib.h>
#include <string.h>

#include <memory>
#include <type_traits>

#include "kvq8.h"

namespace lgmlh {

// The places (kvq8.h) for a head size: K's dims 8 g8 .. + 7 are 8 bytes, V's cells 8 c
// .. + 7 of a dim too.
template <int D>
struct Q8Tile {
  static constexpr int bytes = q8_tile_bytes(D);
  __device__ static int k_at(int cell, int g8) { return q8_k_at(cell, 8 * g8); }
  __device__ static int v_at(int d, int cell) { return q8_v_at(d, cell); }
  __device__ static int scale_at(int b, int cell) { return q8_scale_at(D, b, cell); }
};

// A workgroup takes W consecutive tokens (64, or 16 of a call of few) of one head
// of K or V, 4 values a thread and step. V turns in LDS: 8 tokens whose cells are
// 8 in a row from a multiple of 8 on (a whole group) are 8 consecutive bytes of
// each dim, and 8 lanes take a dim's 64 bytes. Runs of cells start anywhere, so a
// group belongs to the workgroup that has its first token, which also takes the
// up to 7 of it that lie past its own; tokens in no whole group go byte by byte.
// 8192 tokens of 8 heads of 128, K and V: 67 MB of rows read, 18 MB written, 23 us
// with the rows in the memory-side cache (3.7 TB/s; with V's bytes one by one 39),
// 31 from HBM; 64 tokens of them 5.7 us, the time of one workgroup's reads, turn and
// writes after another.
constexpr int Q8_THREADS = 256, Q8_GROUP = 8, Q8_HALO = 7;
constexpr int64_t Q8_CELLS = (int64_t)1 << 36;  // a block's number has 31 bits

// The tile of cell c (>= 0) of one head: head is the first block's.
template <int D, typename P>
__device__ __forceinline__ P *tile_of(P *head, int64_t c, int Hkv) {
  return head + (uint64_t)(uint32_t)((uint64_t)c >> 6) * (uint32_t)(Hkv * Q8Tile<D>::bytes);
}

template <int W>
struct Q8Window {
  int64_t cells[W + 2 * Q8_HALO];  // of tokens j0 - 7 .. j0 + W + 6; -1: none
  int lead[W / Q8_GROUP];          // first tokens of the whole groups, 0 .. W - 1
  int lone[W];                     // tokens in no whole group
  int n_lead, n_lone;
  __device__ __forceinline__ int64_t cell(int t) const { return cells[t + Q8_HALO]; }
  __device__ __forceinline__ bool leads(int t) const {
    bool w = cell(t) >= 0 && cell(t) % 8 == 0;
#pragma unroll
    for (int i = 1; i < 8; i++) w &= cell(t + i) == cell(t) + i;
    return w;
  }
  // All threads; the lists are there for V only.
  __device__ __forceinline__ void fill(const int64_t *__restrict__ src, int64_t j0, int64_t n,
                                       int64_t n_cells, bool lists) {
    const int tid = threadIdx.x;
    if (tid < W + 2 * Q8_HALO) {
      const int64_t j = j0 + tid - Q8_HALO, c = j >= 0 && j < n ? src[j] : -1;
      cells[tid] = c < n_cells ? c : -1;
    }
    __syncthreads();
    if (lists && tid < 64) {
      const int t = tid < W ? tid : W - 1;
      const int64_t c = cell(t);
      const bool is_lead = tid < W && leads(t);
      const int back = c >= 0 ? (int)(c % 8) : 0;
      const bool is_lone = tid < W && c >= 0 && !leads(t - back);
      const uint64_t ml = __builtin_amdgcn_ballot_w64(is_lead), mo = __builtin_amdgcn_ballot_w64(is_lone);
      const uint64_t below = ((uint64_t)1 << tid) - 1;
      if (is_lead) lead[__builtin_popcountll(ml & below)] = t;
      if (is_lone) lone[__builtin_popcountll(mo & below)] = t;
      if (tid == 0) {
        n_lead = __builtin_popcountll(ml);
        n_lone = __builtin_popcountll(mo);
      }
    }
    if (lists) __syncthreads();
  }
};

// Threads for n lone tokens: the power of two that holds them, as bits.
__device__ __forceinline__ int lone_bits(int n) { return n > 1 ? 32 - __builtin_clz(n - 1) : 0; }

// x (n, Hkv D) f32 rows into their cells. Per 32 values (8 lanes), the format's
// steps in f32: d = amax / 127, q = round(x (1 / d)) with halves away from
// zero, d kept as f16.
template <int D, int W>
__global__ void __launch_bounds__(Q8_THREADS)
kv_store_q8_kernel(uint8_t *__restrict__ kp, uint8_t *__restrict__ vp, int64_t n_cells,
                   const float *__restrict__ ks, const float *__restrict__ vs,
                   const int64_t *__restrict__ cells, int64_t n, int Hkv) {
  typedef Q8Tile<D> T;
  constexpr int G4 = D / 4, STEP = Q8_THREADS / G4, PAD = D + 4;
  constexpr int ROWS = W + Q8_HALO, IT = (ROWS + STEP - 1) / STEP, GROUPS = W / Q8_GROUP;
  __shared__ Q8Window<W> win;
  __shared__ __align__(4) int8_t turn[ROWS * PAD];
  __shared__ uint16_t scale[D / 32 * W];
  const int tid = threadIdx.x, h = blockIdx.x % (uint32_t)Hkv, is_v = blockIdx.y;
  const int64_t j0 = (int64_t)(blockIdx.x / (uint32_t)Hkv) * W;
  const int g4 = tid % G4, t0 = tid / G4;
  const float *src = (is_v ? vs : ks) + (j0 * Hkv + h) * D + 4 * g4;
  uint8_t *pool = (is_v ? vp : kp) + (int64_t)h * T::bytes;
  const int64_t left = n - j0 < (is_v ? ROWS : W) ? n - j0 : is_v ? ROWS : W;
  f32x4 x[IT];
#pragma unroll
  for (int i = 0; i < IT; i++) {
    const int t = t0 + i * STEP;
    x[i] = t < left ? *(const f32x4_u *)(src + (int64_t)t * Hkv * D) : f32x4{0, 0, 0, 0};
  }
  win.fill(cells, j0, n, n_cells, is_v);
#pragma unroll
  for (int i = 0; i < IT; i++) {
    const int t = t0 + i * STEP;
    float amax = fmaxf(fmaxf(fabsf(x[i][0]), fabsf(x[i][1])), fmaxf(fabsf(x[i][2]), fabsf(x[i][3])));
    amax = group_max<8>(amax);  // the 8 lanes of a block
    const float d = amax / 127.0f, id = d != 0.0f ? 1.0f / d : 0.0f;
    uint32_t q = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) q |= (uint32_t)(round_away(x[i][e], id) & 0xff) << 8 * e;
    if (t >= left) continue;  // whole blocks of lanes leave together
    if (g4 % 8 == 0 && t < W) scale[g4 / 8 * W + t] = f2h(d);
    if (is_v) {
      *(uint32_t *)(turn + t * PAD + 4 * g4) = q;
    } else if (const int64_t c = win.cell(t); c >= 0) {
      *(uint32_t *)(tile_of<D>(pool, c, Hkv) + T::k_at((int)c & 63, g4 / 2) + 4 * (g4 & 1)) = q;
    }
  }
  __syncthreads();
  // the scales with tokens along the lanes, as a tile has them
  for (int i = tid; i < D / 32 * W; i += Q8_THREADS) {
    const int64_t c = win.cell(i % W);
    if (c >= 0) *(uint16_t *)(tile_of<D>(pool, c, Hkv) + T::scale_at(i / W, (int)c & 63)) = scale[i];
  }
  if (!is_v) return;
  // a thread's group or lone token is the same in every step
  if (const int g = tid % GROUPS; g < win.n_lead) {
    const int t = win.lead[g];
    const int64_t c = win.cell(t);
    uint8_t *tile = tile_of<D>(pool, c, Hkv) + T::v_at(0, (int)c & 63);
#pragma unroll 4
    for (int d = tid / GROUPS; d < D; d += Q8_THREADS / GROUPS) {
      const int8_t *s8 = turn + t * PAD + d;
      uint32_t q[2] = {0, 0};
#pragma unroll
      for (int e = 0; e < 8; e++) q[e >> 2] |= (uint32_t)(uint8_t)s8[e * PAD] << 8 * (e & 3);
      *(u32x2 *)(tile + 64 * d) = u32x2{q[0], q[1]};
    }
  }
  const int no = win.n_lone, sh = lone_bits(no);
  if (const int k = tid & ((1 << sh) - 1); k < no) {
    const int t = win.lone[k];
    const int64_t c = win.cell(t);
    uint8_t *tile = tile_of<D>(pool, c, Hkv) + T::v_at(0, (int)c & 63);
#pragma unroll 8
    for (int d = tid >> sh; d < D; d += Q8_THREADS >> sh) tile[64 * d] = (uint8_t)turn[t * PAD + d];
  }
}

// A value's four of a row: f32 or f16 of d q.
template <typename OutT>
__device__ __forceinline__ void put4(OutT *out, uint32_t q, float d) {
  typedef OutT o4 __attribute__((ext_vector_type(4), aligned(sizeof(OutT))));
  o4 y;
#pragma unroll
  for (int e = 0; e < 4; e++) y[e] = (OutT)(d * (float)(int8_t)(q >> 8 * e));
  *(o4 *)out = y;
}

// The scales of N tokens (cell(t), -1: none) into LDS, tokens along the lanes, as
// a tile has them: 64 cells' of 32 dims are a line. (By the lanes that use them
// they are 8 lines a wave and 64 tokens, twice the values'.)
template <int D, int N, typename C>
__device__ __forceinline__ void load_scales(uint16_t *lds, const uint8_t *head, int Hkv, C cell) {
#pragma unroll
  for (int k = 0; k < (D / 32 * N + Q8_THREADS - 1) / Q8_THREADS; k++) {
    const int i = threadIdx.x + k * Q8_THREADS;
    if (i >= D / 32 * N) break;
    const int64_t c = cell(i % N);
    lds[i] = c < 0 ? 0
                   : *(const uint16_t *)(tile_of<D>(head, c, Hkv) + Q8Tile<D>::scale_at(i / N, (int)c & 63));
  }
}

// Cells as rows (n, Hkv D) of f32 or f16, the store the other way round: the values
// into LDS as rows (K's 16 bytes a lane are 8 dims of two blocks), the scales too,
// then out 4 values a lane. (K's values straight from the tile, 4 bytes a lane,
// need each token's address in each lane: 32768 tokens of 8 heads of 128 54 us.)
// Bound by HBM's writes: those tokens' K are 35 MB read and 134 MB of f32 written
// in 36 us (4.7 TB/s), V as many in 39.
template <int D, int W, bool IS_V, typename OutT>
__global__ void __launch_bounds__(Q8_THREADS)
kv_gather_q8_kernel(const uint8_t *__restrict__ pool, int64_t n_cells,
                    const int64_t *__restrict__ cells, int64_t n, int Hkv,
                    OutT *__restrict__ out) {
  typedef Q8Tile<D> T;
  constexpr int G4 = D / 4, STEP = Q8_THREADS / G4, PAD = IS_V ? D + 4 : D + 8;
  constexpr int ROWS = IS_V ? W + Q8_HALO : W, NS = IS_V ? W + 8 : W, GROUPS = W / Q8_GROUP;
  __shared__ Q8Window<W> win;
  __shared__ __align__(8) int8_t turn[ROWS * PAD];
  __shared__ uint8_t mine[ROWS];  // the rows of turn that are this workgroup's
  __shared__ uint16_t scale[D / 32 * NS];
  const int tid = threadIdx.x, h = blockIdx.x % (uint32_t)Hkv;
  const int64_t j0 = (int64_t)(blockIdx.x / (uint32_t)Hkv) * W;
  const uint8_t *head = pool + (int64_t)h * T::bytes;
  win.fill(cells, j0, n, n_cells, IS_V);
  load_scales<D, NS>(scale, head, Hkv, [&](int t) { return t < ROWS ? win.cell(t) : -1; });
  if constexpr (IS_V) {
    const int ng = win.n_lead, no = win.n_lone;
    if (tid < ROWS) mine[tid] = tid < W && win.cell(tid) < 0;  // a cell outside: zeros
    constexpr int GI = (GROUPS * D + Q8_THREADS - 1) / Q8_THREADS;
    const int g = tid % GROUPS, lead = g < ng ? win.lead[g] : -1;
    u32x2 q8[GI];
    if (lead >= 0) {
      const int64_t c = win.cell(lead);
      const uint8_t *tile = tile_of<D>(head, c, Hkv) + T::v_at(0, (int)c & 63);
#pragma unroll
      for (int i = 0; i < GI; i++) {
        const int d = tid / GROUPS + i * (Q8_THREADS / GROUPS);
        if (d < D) q8[i] = *(const u32x2 *)(tile + 64 * d);
      }
    }
    __syncthreads();
    if (tid < 8 * ng) mine[win.lead[tid >> 3] + (tid & 7)] = 1;
    if (tid < no) mine[win.lone[tid]] = 1;
    if (lead >= 0) {
#pragma unroll
      for (int i = 0; i < GI; i++) {
        const int d = tid / GROUPS + i * (Q8_THREADS / GROUPS);
        int8_t *s8 = turn + lead * PAD + d;
        if (d < D)
#pragma unroll
          for (int e = 0; e < 8; e++) s8[e * PAD] = (int8_t)(q8[i][e >> 2] >> 8 * (e & 3));
      }
    }
    const int sh = lone_bits(no);
    if (const int k = tid & ((1 << sh) - 1); k < no) {
      const int t = win.lone[k];
      const int64_t c = win.cell(t);
      const uint8_t *tile = tile_of<D>(head, c, Hkv) + T::v_at(0, (int)c & 63);
#pragma unroll 8
      for (int d = tid >> sh; d < D; d += Q8_THREADS >> sh) turn[t * PAD + d] = (int8_t)tile[64 * d];
    }
  } else {
    constexpr int PI = (W * D / 16 + Q8_THREADS - 1) / Q8_THREADS;
#pragma unroll
    for (int i = 0; i < PI; i++) {  // (token, j, quad), tokens of 4 quads in a row
      const int k = tid + i * Q8_THREADS, t = k / 4 % W, j = k / (4 * W), quad = k % 4;
      if (k >= W * D / 16) break;
      const int64_t c = win.cell(t);
      if (c < 0) continue;
      const u32x4 q = *(const u32x4 *)(tile_of<D>(head, c, Hkv) + T::k_at((int)c & 63, 8 * j + quad));
      *(u32x2 *)(turn + t * PAD + 64 * j + 8 * quad) = u32x2{q[0], q[1]};
      *(u32x2 *)(turn + t * PAD + 64 * j + 32 + 8 * quad) = u32x2{q[2], q[3]};
    }
  }
  __syncthreads();
  const int g4 = tid % G4;
  const int left = n - j0 < ROWS ? (int)(n - j0) : ROWS;
#pragma unroll 8
  for (int t = tid / G4; t < left; t += STEP) {
    if (IS_V && !mine[t]) continue;
    const uint32_t q = win.cell(t) < 0 ? 0 : *(const uint32_t *)(turn + t * PAD + 4 * g4);
    put4(out + ((j0 + t) * Hkv + h) * (int64_t)D + 4 * g4, q, h2f(scale[g4 / 8 * NS + t]));
  }
}

// Tokens of a workgroup: 64 (32 of heads of 256), but 16 where that makes fewer
// than 256 workgroups.
constexpr int q8_tokens(int D) { return D > 128 ? 32 : 64; }
static bool q8_small(int64_t n, int n_head_kv, int kinds, int D) {
  return (n + q8_tokens(D) - 1) / q8_tokens(D) * n_head_kv * kinds < 256;
}

// Cells src -> dst of every pool tensor (K at even places, V at odd ones), each
// dst as its src was before the call: a workgroup takes rows of one head's tiles
// of one tensor (16-byte pieces of K's cells, V's dims, Q8_0's scales), reads all
// the moves' values of them into registers, then writes. It is bound by V, whose
// cells are 2 (or 1) bytes of a line each: 320 moves of 32 layers of 8 heads of
// 128 in f16 are 84 MB of values, but 2.1 million lines of V, 134 us with the pool
// in HBM (reads alone 58, writes alone, whose lines are fetched to be merged into,
// 106: 128 bytes each way are 540 MB at 4 to 5 TB/s; K's part 13) and 91 with its
// lines in the memory-side cache. Stores past the caches take those 91 where
// others take 104, reads past them 140; 512 threads of 8 values 91 and 256 of 16
// 95; a head's slices on all dies at once 129 (149 from HBM).
constexpr int MOVE_MAX = 1024, MOVE_THREADS = 512;

// The values (row r, move m), m fastest or (CELLS) r fastest, at base + off[m] +
// at(r): PER a thread, the rest of the index stepped without a division.
template <typename T, int PER, bool CELLS, typename At>
__device__ __forceinline__ void move_rows(uint8_t *base, const int64_t *from, const int64_t *to, int n,
                                          int rows, At at) {
  const int total = n * rows, inner = CELLS ? rows : n;
  int lo[PER], hi[PER];
  T v[PER];
  int b = (int)threadIdx.x / inner, a = (int)threadIdx.x % inner;
  const int db = MOVE_THREADS / inner, da = MOVE_THREADS % inner;
#pragma unroll
  for (int j = 0; j < PER; j++) {
    lo[j] = CELLS ? b : a;  // the move
    hi[j] = at(CELLS ? a : b);
    a += da;
    b += db;
    if (a >= inner) {
      a -= inner;
      b++;
    }
    if (j * MOVE_THREADS + (int)threadIdx.x < total && from[lo[j]] >= 0)
      v[j] = *(const T *)(base + from[lo[j]] + hi[j]);
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < PER; j++)
    if (j * MOVE_THREADS + (int)threadIdx.x < total && from[lo[j]] >= 0)
      __builtin_nontemporal_store(v[j], (T *)(base + to[lo[j]] + hi[j]));
}

// Rows of a workgroup: K's 16-byte pieces of a cell, V's dims.
struct MoveShape {
  int k_rows, v_rows;
};
template <bool Q8, int PER>
__global__ void __launch_bounds__(MOVE_THREADS)
kv_move_kernel(void *const *__restrict__ pools, int64_t n_cells, int Hkv, int D,
               const int64_t *__restrict__ src, const int64_t *__restrict__ dst, int n,
               MoveShape shape) {
  __shared__ int64_t from[MOVE_MAX], to[MOVE_MAX];
  const int p = blockIdx.y, is_v = p & 1;
  const int h = blockIdx.x % Hkv, s = blockIdx.x / Hkv;
  const int all = is_v ? D : Q8 ? D / 16 : D / 8, rows = is_v ? shape.v_rows : shape.k_rows;
  const bool scales = Q8 && s == (int)(gridDim.x / Hkv) - 1;
  if (!scales && s * rows >= all) return;
  uint8_t *pool = (uint8_t *)pools[p];
  const int64_t tile = Q8 ? 68 * (int64_t)D : 128 * (int64_t)D;
  // a cell's place in its tile, without the row
  auto place = [&](int64_t c) {
    const int o = (int)(c % KV_BLOCK);
    const int in = scales  ? 64 * D + 2 * o
                   : !is_v ? (Q8 ? o * 64 : o * D * 2)
                           : (Q8 ? o % 32 / 8 * 16 + o / 32 * 8 + o % 8 : 2 * o);
    return ((c / KV_BLOCK) * Hkv + h) * tile + in;
  };
  for (int m = threadIdx.x; m < n; m += MOVE_THREADS) {
    const int64_t a = src[m], b = dst[m];
    const bool good = (uint64_t)a < (uint64_t)n_cells && (uint64_t)b < (uint64_t)n_cells;
    from[m] = good ? place(a) : -1;
    to[m] = good ? place(b) : -1;
  }
  __syncthreads();
  const int r0 = s * rows, left = all - r0 < rows ? all - r0 : rows;
  if (scales)
    move_rows<uint16_t, PER, false>(pool, from, to, n, D / 32, [](int r) { return 128 * r; });
  else if (!is_v)
    move_rows<u32x4, PER, true>(pool, from, to, n, left, [&](int r) {
      return Q8 ? (r0 + r) / 4 * 4096 + (r0 + r) % 4 * 16 : 16 * (r0 + r);
    });
  else if (Q8)
    move_rows<uint8_t, PER, false>(pool, from, to, n, left, [&](int r) { return 64 * (r0 + r); });
  else
    move_rows<uint16_t, PER, false>(pool, from, to, n, left, [&](int r) { return 128 * (r0 + r); });
}

// Range and distinctness of cells that a call writes. Cells come in runs (c, c +
// 1, ...), cut at blocks: a table of (block, cells seen) takes one entry per
// piece, and is twice as long (on the stack up to 512 pieces). 65536 cells in
// a run take 0.1 ms of the host, each in a block of its own 0.6, 262144 of those
// 2.5.
static int check_write_cells(const int64_t *h, int64_t n, int64_t n_cells, const char *what) {
  if (!h) {
    set_error("%s: the host copy of the cells is required for the checks", what);
    return LGMLH_EINVAL;
  }
  int64_t pieces = 0;
  for (int64_t j = 0; j < n; j++) {
    if (h[j] < 0 || h[j] >= n_cells) {
      set_error("%s: cell %lld out of range [0, %lld)", what, (long long)h[j], (long long)n_cells);
      return LGMLH_ERANGE;
    }
    pieces += j == 0 || h[j] != h[j - 1] + 1 || h[j] % KV_BLOCK == 0;
  }
  constexpr int NEAR = 1024;
  struct Slot {
    int64_t block;  // + 1; 0: free
    uint64_t seen;
  } near_[NEAR];
  int bits = 4;
  while ((int64_t)1 << bits < 2 * pieces) bits++;
  const uint64_t slots = (uint64_t)1 << bits;
  std::unique_ptr<Slot, void (*)(void *)> far(nullptr, free);
  Slot *table = near_;
  if (slots > NEAR) {
    far.reset((Slot *)calloc(slots, sizeof(Slot)));
    if (!far) {
      set_error("%s: no host memory to check %lld cells", what, (long long)n);
      return LGMLH_ENOMEM;
    }
    table = far.get();
  } else {
    memset(near_, 0, slots * sizeof(Slot));
  }
  for (int64_t j = 0; j < n;) {
    const int64_t block = h[j] / KV_BLOCK;
    uint64_t seen = 0;
    do {
      seen |= (uint64_t)1 << h[j] % KV_BLOCK;
      j++;
    } while (j < n && h[j] == h[j - 1] + 1 && h[j] % KV_BLOCK);
    uint64_t at = (uint64_t)block * 0x9e3779b97f4a7c15ull >> (64 - bits);
    while (table[at].block && table[at].block != block + 1) at = (at + 1) & (slots - 1);
    table[at].block = block + 1;
    if (table[at].seen & seen) {
      set_error("%s: a cell of block %lld is written twice", what, (long long)block);
      return LGMLH_EINVAL;
    }
    table[at].seen |= seen;
  }
  return LGMLH_OK;
}

// Heads of cells in one call: a launch has fewer than 2^32 threads, 256 for 32 or
// more of them. KV heads: the bytes of a block, 68 D for each, are counted in 31
// bits (tile_of).
constexpr int64_t Q8_ROWS = int64_t(1) << 29;
constexpr int Q8_HEADS = 65535;
static_assert((int64_t)Q8_HEADS * q8_tile_bytes(256) < INT32_MAX, "tile_of");

static bool q8_head(int D) { return D == 64 || D == 128 || D == 256; }

}  // namespace lgmlh

using namespace lgmlh;

extern "C" int64_t lgmlh_kv_q8_layer_bytes(int64_t n_cells, int n_head_kv, int head_dim) {
  if (n_cells <= 0 || n_cells % KV_BLOCK || n_head_kv <= 0 || !q8_head(head_dim)) return -1;
  return n_cells / KV_BLOCK * n_head_kv * 68 * head_dim;
}

extern "C" int lgmlh_kv_store_q8(void *kpool, void *vpool, int64_t n_cells, int n_head_kv,
                                 int head_dim, const float *k_src, const float *v_src,
                                 const int64_t *cells, const int64_t *h_cells, int64_t n,
                                 void *stream) {
  if (!kpool || !vpool || !k_src || !v_src || !cells || n < 0 || n_cells <= 0 ||
      n_cells > Q8_CELLS || n_cells % KV_BLOCK || n_head_kv <= 0 || n_head_kv > Q8_HEADS ||
      n >= Q8_ROWS / n_head_kv || !q8_head(head_dim)) {
    set_error("kv_store_q8: bad arguments (heads of 64, 128 or 256)");
    return LGMLH_EINVAL;
  }
  if (((uintptr_t)kpool | (uintptr_t)vpool) & 15) {
    set_error("kv_store_q8: pools are 16-byte aligned");
    return LGMLH_EINVAL;
  }
  LGMLH_TRY(check_write_cells(h_cells, n, n_cells, "kv_store_q8"));
  if (n == 0) return LGMLH_OK;
  const bool small = q8_small(n, n_head_kv, 2, head_dim);
  const int w = small ? 16 : q8_tokens(head_dim);
  // heads fastest: those of the same rows run together
  const dim3 grid((unsigned)((n + w - 1) / w * n_head_kv), 2);
  hipStream_t st = as_stream(stream);
  const auto kern = head_dim == 64    ? (small ? kv_store_q8_kernel<64, 16> : kv_store_q8_kernel<64, 64>)
                    : head_dim == 128 ? (small ? kv_store_q8_kernel<128, 16> : kv_store_q8_kernel<128, 64>)
                                      : (small ? kv_store_q8_kernel<256, 16> : kv_store_q8_kernel<256, 32>);
  hipLaunchKernelGGL(kern, grid, dim3(Q8_THREADS), 0, st, (uint8_t *)kpool, (uint8_t *)vpool,
                     n_cells, k_src, v_src, cells, n, n_head_kv);
  return hip_check(hipGetLastError(), "kv_store_q8");
}

extern "C" int lgmlh_kv_gather_q8(const void *pool, int which, int64_t n_cells, int n_head_kv,
                                  int head_dim, const int64_t *cells, int64_t n, void *out,
                                  int out_type, void *stream) {
  if (!pool || !cells || !out || n < 0 || (which != 0 && which != 1) || n_cells <= 0 ||
      n_cells > Q8_CELLS || n_cells % KV_BLOCK || n_head_kv <= 0 || n_head_kv > Q8_HEADS ||
      n >= Q8_ROWS / n_head_kv || !q8_head(head_dim) ||
      (out_type != LGMLH_F32 && out_type != LGMLH_F16)) {
    set_error("kv_gather_q8: bad arguments (heads of 64, 128 or 256; out f32 or f16)");
    return LGMLH_EINVAL;
  }
  if ((uintptr_t)pool & 15) {
    set_error("kv_gather_q8: pools are 16-byte aligned");
    return LGMLH_EINVAL;
  }
  if (n == 0) return LGMLH_OK;
  const bool small = q8_small(n, n_head_kv, 1, head_dim);
  const int w = small ? 16 : q8_tokens(head_dim);
  const dim3 grid((unsigned)((n + w - 1) / w * n_head_kv));
  hipStream_t st = as_stream(stream);
  auto go = [&](auto out_t) {
    typedef decltype(out_t) T;
    auto launch = [&](auto kern) {
      hipLaunchKernelGGL(kern, grid, dim3(Q8_THREADS), 0, st, (const uint8_t *)pool, n_cells, cells, n,
                         n_head_kv, (T *)out);
    };
    auto of = [&](auto d) {
      constexpr int D = decltype(d)::value, big = q8_tokens(D);
      if (which)
        launch(small ? kv_gather_q8_kernel<D, 16, true, T> : kv_gather_q8_kernel<D, big, true, T>);
      else
        launch(small ? kv_gather_q8_kernel<D, 16, false, T> : kv_gather_q8_kernel<D, big, false, T>);
    };
    if (head_dim == 64)
      of(std::integral_constant<int, 64>{});
    else if (head_dim == 128)
      of(std::integral_constant<int, 128>{});
    else
      of(std::integral_constant<int, 256>{});
  };
  if (out_type == LGMLH_F32)
    go(float{});
  else
    go(f16{});
  return hip_check(hipGetLastError(), "kv_gather_q8");
}

extern "C" int lgmlh_kv_move(int type, void *const *pools, int n_pools, int64_t n_cells,
                             int n_head_kv, int head_dim, const int64_t *src, const int64_t *dst,
                             const int64_t *h_src, const int64_t *h_dst, int64_t n, void *stream) {
  const bool q8 = type == LGMLH_Q8_0;
  if ((!q8 && type != LGMLH_F16) || !pools || !src || !dst || n_pools <= 0 || n_pools > 65535 ||
      n_pools % 2 || n_cells <= 0 || n_cells % KV_BLOCK || n_head_kv <= 0 || n_head_kv > 65535 || n < 0 ||
      (q8 ? !q8_head(head_dim) : head_dim != 16 && (head_dim <= 0 || head_dim % 32))) {
    set_error("kv_move: bad arguments (K and V tensors in turn, of f16 or Q8_0)");
    return LGMLH_EINVAL;
  }
  if (n > MOVE_MAX) {
    set_error("kv_move: %lld cells in one call (at most %d)", (long long)n, MOVE_MAX);
    return LGMLH_EINVAL;
  }
  if (!h_src) {
    set_error("kv_move: the host copy of the cells is required for the checks");
    return LGMLH_EINVAL;
  }
  for (int64_t j = 0; j < n; j++)
    if (h_src[j] < 0 || h_src[j] >= n_cells) {
      set_error("kv_move: cell %lld out of range [0, %lld)", (long long)h_src[j], (long long)n_cells);
      return LGMLH_ERANGE;
    }
  LGMLH_TRY(check_write_cells(h_dst, n, n_cells, "kv_move"));
  if (n == 0) return LGMLH_OK;
  // as few values a thread as leave a workgroup 8 rows, a cache line's of K; then
  // as many rows as it holds
  const int per = n <= MOVE_THREADS ? 8 : 16;
  const int hold = per * MOVE_THREADS / (int)n;
  auto fit = [&](int all) {
    int r = all;
    while (r > hold) r = (r + 1) / 2;
    return r;
  };
  const int pieces = head_dim / (q8 ? 16 : 8);
  const MoveShape shape = {fit(pieces), fit(head_dim)};
  const int slices_k = (pieces + shape.k_rows - 1) / shape.k_rows,
            slices_v = (head_dim + shape.v_rows - 1) / shape.v_rows;
  const int slices = (slices_k > slices_v ? slices_k : slices_v) + (q8 ? 1 : 0);
  const auto kern = q8 ? (per == 8 ? kv_move_kernel<true, 8> : kv_move_kernel<true, 16>)
                       : (per == 8 ? kv_move_kernel<false, 8> : kv_move_kernel<false, 16>);
  hipLaunchKernelGGL(kern, dim3((unsigned)(n_head_kv * slices), (unsigned)n_pools), dim3(MOVE_THREADS),
                     0, as_stream(stream), pools, n_cells, n_head_kv, head_dim, src, dst, (int)n, shape);
  return hip_check(hipGetLastError(), "kv_move");
}
