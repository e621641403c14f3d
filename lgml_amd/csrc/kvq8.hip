// The KV pool in Q8_0 (8-bit values, an f16 scale per 32), and moves of cells
// within a pool of either type (gfx950).
//
// A (block, KV head) tile of K or V is 68 D bytes: 64 D int8 values, then the
// f16 scales [D / 32][64 cells]. Values are placed so that one 16-byte load a
// lane gives its part of two of the attention's 16x16x32 operands:
//   K: [D / 64][cell][4][2][8], dim 64 j + 32 b + 8 q + e at (j, cell, q, b, e)
//   V: [D][4][2][8], cell 32 b + 8 q + e at (d, q, b, e)
// The scales' order is the one in which a lane has 8 cells of a block of 32
// dims in 16 bytes.
#include <type_traits>

#include "common.h"

namespace lgmlh {

template <int D>
struct Q8Tile {
  static constexpr int bytes = 68 * D, scales = 64 * D;
  // byte of K's dims 8 g8 .. + 7 of a cell
  __device__ static int k_at(int cell, int g8) {
    return ((g8 / 8 * 64 + cell) * 4 + g8 % 4) * 16 + g8 % 8 / 4 * 8;
  }
  // byte of V's (d, cell); cells 8 c .. 8 c + 7 are consecutive
  __device__ static int v_at(int d, int cell) {
    return d * 64 + cell % 32 / 8 * 16 + cell / 32 * 8 + cell % 8;
  }
  // byte of the scale of dims 32 b .. + 31
  __device__ static int scale_at(int b, int cell) { return scales + 2 * (b * 64 + cell); }
};

constexpr int Q8_TOKENS = 32, Q8_THREADS = 256;  // of a workgroup, for one head of K or V

// The tokens of a workgroup start at a multiple of 8 cells when the call's
// tokens are one run of cells (a prompt chunk): then groups of 8 tokens are 8
// consecutive bytes of V.
__device__ __forceinline__ int64_t first_token(const int64_t *__restrict__ cells) {
  return (int64_t)blockIdx.x * Q8_TOKENS - cells[0] % 8;
}
// Whether tokens j .. j + 7 are 8 cells from a multiple of 8 on (lds: the
// workgroup's cells, -1 for none).
__device__ __forceinline__ bool whole_group(const int64_t *cell) {
  bool w = cell[0] >= 0 && cell[0] % 8 == 0;
#pragma unroll
  for (int i = 1; i < 8; i++) w &= cell[i] == cell[0] + i;
  return w;
}
__device__ __forceinline__ void load_cells(int64_t *lds, const int64_t *__restrict__ cells,
                                           int64_t j0, int64_t n, int64_t n_cells) {
  if (threadIdx.x < Q8_TOKENS) {
    const int64_t j = j0 + threadIdx.x, c = j >= 0 && j < n ? cells[j] : -1;
    lds[threadIdx.x] = c < n_cells ? c : -1;
  }
}

// x (n, Hkv D) f32 rows into their cells. Per 32 values, the steps of
// quantize_row_q8_0: d = amax / 127, q = round(x (1 / d)) with halves away from
// zero, d kept as f16. A thread has 8 values; K leaves as 8 bytes, V turns in
// LDS so that 8 cells leave as 8 bytes.
template <int D>
__global__ void __launch_bounds__(Q8_THREADS)
kv_store_q8_kernel(uint8_t *__restrict__ kp, uint8_t *__restrict__ vp, int64_t n_cells,
                   const float *__restrict__ ks, const float *__restrict__ vs,
                   const int64_t *__restrict__ cells, int64_t n, int Hkv) {
  typedef Q8Tile<D> T;
  constexpr int G8 = D / 8, STEP = Q8_THREADS / G8, PAD = D + 4;
  __shared__ int64_t cell[Q8_TOKENS];
  __shared__ __align__(8) int8_t turn[Q8_TOKENS * PAD];
  const int tid = threadIdx.x, h = blockIdx.y, is_v = blockIdx.z;
  const int64_t j0 = first_token(cells);
  load_cells(cell, cells, j0, n, n_cells);
  const int g8 = tid % G8, t0 = tid / G8;
  const float *src = (is_v ? vs : ks) + (int64_t)h * D + 8 * g8;
  uint8_t *pool = (is_v ? vp : kp) + (int64_t)h * T::bytes;
  f32x4 x[Q8_TOKENS / STEP][2];
#pragma unroll
  for (int i = 0; i < Q8_TOKENS / STEP; i++) {
    const int64_t j = j0 + t0 + i * STEP;
    const f32x4_u *p = (const f32x4_u *)(src + j * Hkv * D);
    const bool in = j >= 0 && j < n;
    x[i][0] = in ? p[0] : f32x4{0, 0, 0, 0};
    x[i][1] = in ? p[1] : f32x4{0, 0, 0, 0};
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < Q8_TOKENS / STEP; i++) {
    const int t = t0 + i * STEP;
    float amax = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; e++) amax = fmaxf(amax, fabsf(x[i][e >> 2][e & 3]));
    amax = group_max<4>(amax);  // the 4 lanes of a block
    const float d = amax / 127.0f, id = d != 0.0f ? 1.0f / d : 0.0f;
    uint32_t q[2] = {0, 0};
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const int v = (int)__builtin_roundf(x[i][e >> 2][e & 3] * id);
      q[e >> 2] |= (uint32_t)(v & 0xff) << 8 * (e & 3);
    }
    const int64_t c = cell[t];
    if (is_v) {
      uint32_t *dst = (uint32_t *)(turn + t * PAD + 8 * g8);
      dst[0] = q[0];
      dst[1] = q[1];
    }
    if (c < 0) continue;  // groups of 4 lanes leave together
    uint8_t *tile = pool + (c / KV_BLOCK) * Hkv * T::bytes;
    const int o = (int)(c % KV_BLOCK);
    if (!is_v) *(u32x2 *)(tile + T::k_at(o, g8)) = u32x2{q[0], q[1]};
    if (g8 % 4 == 0) *(uint16_t *)(tile + T::scale_at(g8 / 4, o)) = f2h(d);
  }
  if (!is_v) return;
  __syncthreads();
  for (int i = tid; i < Q8_TOKENS / 8 * D; i += Q8_THREADS) {
    const int g = i / D, d = i % D;
    const int64_t *cg = cell + 8 * g;
    const int8_t *src8 = turn + 8 * g * PAD + d;
    if (whole_group(cg)) {  // the same for a wave's lanes
      uint8_t *tile = pool + (cg[0] / KV_BLOCK) * Hkv * T::bytes;
      uint32_t q[2] = {0, 0};
#pragma unroll
      for (int e = 0; e < 8; e++) q[e >> 2] |= (uint32_t)(uint8_t)src8[e * PAD] << 8 * (e & 3);
      *(u32x2 *)(tile + T::v_at(d, (int)(cg[0] % KV_BLOCK))) = u32x2{q[0], q[1]};
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const int64_t c = cg[e];
        if (c < 0) continue;
        uint8_t *tile = pool + (c / KV_BLOCK) * Hkv * T::bytes;
        tile[T::v_at(d, (int)(c % KV_BLOCK))] = (uint8_t)src8[e * PAD];
      }
    }
  }
}

// Cells as rows (n, Hkv D) of f32 or f16: the same shape the other way round.
template <int D, typename OutT>
__global__ void __launch_bounds__(Q8_THREADS)
kv_gather_q8_kernel(const uint8_t *__restrict__ pool, int which, int64_t n_cells,
                    const int64_t *__restrict__ cells, int64_t n, int Hkv,
                    OutT *__restrict__ out) {
  typedef Q8Tile<D> T;
  constexpr int G8 = D / 8, STEP = Q8_THREADS / G8, PAD = D + 4;
  __shared__ int64_t cell[Q8_TOKENS];
  __shared__ __align__(8) int8_t turn[Q8_TOKENS * PAD];
  const int tid = threadIdx.x, h = blockIdx.y;
  const int64_t j0 = first_token(cells);
  load_cells(cell, cells, j0, n, n_cells);
  __syncthreads();
  const uint8_t *head = pool + (int64_t)h * T::bytes;
  if (which) {
    for (int i = tid; i < Q8_TOKENS / 8 * D; i += Q8_THREADS) {
      const int g = i / D, d = i % D;
      const int64_t *cg = cell + 8 * g;
      int8_t *dst = turn + 8 * g * PAD + d;
      if (whole_group(cg)) {
        const uint8_t *tile = head + (cg[0] / KV_BLOCK) * Hkv * T::bytes;
        const u32x2 q = *(const u32x2 *)(tile + T::v_at(d, (int)(cg[0] % KV_BLOCK)));
#pragma unroll
        for (int e = 0; e < 8; e++) dst[e * PAD] = (int8_t)(q[e >> 2] >> 8 * (e & 3));
      } else {
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const int64_t c = cg[e];
          const uint8_t *tile = head + (c / KV_BLOCK) * Hkv * T::bytes;
          dst[e * PAD] = c < 0 ? (int8_t)0 : (int8_t)tile[T::v_at(d, (int)(c % KV_BLOCK))];
        }
      }
    }
    __syncthreads();
  }
  const int g8 = tid % G8, t0 = tid / G8;
#pragma unroll
  for (int i = 0; i < Q8_TOKENS / STEP; i++) {
    const int t = t0 + i * STEP;
    const int64_t j = j0 + t, c = cell[t];
    if (j < 0 || j >= n) continue;
    u32x2 q = {0, 0};
    float d = 0.0f;
    if (c >= 0) {
      const uint8_t *tile = head + (c / KV_BLOCK) * Hkv * T::bytes;
      const int o = (int)(c % KV_BLOCK);
      d = h2f(*(const uint16_t *)(tile + T::scale_at(g8 / 4, o)));
      if (which) {
        const uint32_t *s = (const uint32_t *)(turn + t * PAD + 8 * g8);
        q = u32x2{s[0], s[1]};
      } else {
        q = *(const u32x2 *)(tile + T::k_at(o, g8));
      }
    }
    typedef OutT o4 __attribute__((ext_vector_type(4), aligned(sizeof(OutT))));
    OutT *dst = out + (j * Hkv + h) * (int64_t)D + 8 * g8;
#pragma unroll
    for (int v = 0; v < 2; v++) {
      o4 y;
#pragma unroll
      for (int e = 0; e < 4; e++) y[e] = (OutT)(d * (float)(int8_t)(q[v] >> 8 * e));
      *(o4 *)(dst + 4 * v) = y;
    }
  }
}

// Cells src -> dst of every pool tensor (K at even places, V at odd ones), each
// dst as its src was before the call: a workgroup takes rows of one head's tiles
// of one tensor (16-byte pieces of K's cells, V's dims, Q8_0's scales), reads all
// the moves' values of them into registers, then writes. It is bound by V, whose
// cells are 2 (or 1) bytes of a line each.
constexpr int MOVE_MAX = 1024, MOVE_THREADS = 256;

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
      *(T *)(base + to[lo[j]] + hi[j]) = v[j];
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
// piece. Several passes, each over a share of the blocks, where the pieces are
// more than the table holds.
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
  constexpr int SLOTS = 1024, FILL = SLOTS / 2;
  struct Slot {
    int64_t block;
    uint64_t seen;
  } table[SLOTS];
  const uint64_t shares = (uint64_t)((pieces + FILL - 1) / FILL);
  for (uint64_t share = 0; share < shares; share++) {
    for (Slot &s : table) s.block = -1;
    int used = 0;
    for (int64_t j = 0; j < n;) {
      const int64_t block = h[j] / KV_BLOCK;
      uint64_t seen = 0;
      do {
        seen |= (uint64_t)1 << h[j] % KV_BLOCK;
        j++;
      } while (j < n && h[j] == h[j - 1] + 1 && h[j] % KV_BLOCK);
      const uint64_t key = (uint64_t)block * 0x9e3779b97f4a7c15ull;
      if (shares > 1 && (key >> 32) % shares != share) continue;
      int at = (int)(key >> 54);
      while (table[at].block >= 0 && table[at].block != block) at = (at + 1) % SLOTS;
      if (table[at].block < 0) {
        if (++used == SLOTS) {  // a share far above its part: cannot be told
          set_error("%s: too many blocks in one call", what);
          return LGMLH_EINVAL;
        }
        table[at] = Slot{block, 0};
      }
      if (table[at].seen & seen) {
        set_error("%s: a cell of block %lld is written twice", what, (long long)block);
        return LGMLH_EINVAL;
      }
      table[at].seen |= seen;
    }
  }
  return LGMLH_OK;
}

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
      n_cells % KV_BLOCK || n_head_kv <= 0 || n_head_kv > 65535 || !q8_head(head_dim)) {
    set_error("kv_store_q8: bad arguments (heads of 64, 128 or 256)");
    return LGMLH_EINVAL;
  }
  LGMLH_TRY(check_write_cells(h_cells, n, n_cells, "kv_store_q8"));
  if (n == 0) return LGMLH_OK;
  const dim3 grid((unsigned)((n + 7 + Q8_TOKENS - 1) / Q8_TOKENS), (unsigned)n_head_kv, 2);
  hipStream_t st = as_stream(stream);
  const auto kern = head_dim == 64    ? kv_store_q8_kernel<64>
                    : head_dim == 128 ? kv_store_q8_kernel<128>
                                      : kv_store_q8_kernel<256>;
  hipLaunchKernelGGL(kern, grid, dim3(Q8_THREADS), 0, st, (uint8_t *)kpool, (uint8_t *)vpool,
                     n_cells, k_src, v_src, cells, n, n_head_kv);
  return hip_check(hipGetLastError(), "kv_store_q8");
}

extern "C" int lgmlh_kv_gather_q8(const void *pool, int which, int64_t n_cells, int n_head_kv,
                                  int head_dim, const int64_t *cells, int64_t n, void *out,
                                  int out_type, void *stream) {
  if (!pool || !cells || !out || n < 0 || (which != 0 && which != 1) || n_cells <= 0 ||
      n_cells % KV_BLOCK || n_head_kv <= 0 || n_head_kv > 65535 || !q8_head(head_dim) ||
      (out_type != LGMLH_F32 && out_type != LGMLH_F16)) {
    set_error("kv_gather_q8: bad arguments (heads of 64, 128 or 256; out f32 or f16)");
    return LGMLH_EINVAL;
  }
  if (n == 0) return LGMLH_OK;
  const dim3 grid((unsigned)((n + 7 + Q8_TOKENS - 1) / Q8_TOKENS), (unsigned)n_head_kv);
  hipStream_t st = as_stream(stream);
  auto go = [&](auto out_t) {
    typedef decltype(out_t) OutT;
    const auto kern = head_dim == 64    ? kv_gather_q8_kernel<64, OutT>
                      : head_dim == 128 ? kv_gather_q8_kernel<128, OutT>
                                        : kv_gather_q8_kernel<256, OutT>;
    hipLaunchKernelGGL(kern, grid, dim3(Q8_THREADS), 0, st, (const uint8_t *)pool, which, n_cells,
                       cells, n, n_head_kv, (OutT *)out);
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
      n_pools % 2 || n_cells <= 0 || n_cells % KV_BLOCK || n_head_kv <= 0 || n < 0 ||
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
  // as few values a thread (8, 16, 32) as leave a workgroup 8 rows, a cache line's
  // of K; then as many rows as it holds
  const int per = n <= MOVE_THREADS ? 8 : n <= 2 * MOVE_THREADS ? 16 : 32;
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
  const auto kern = q8 ? (per == 8    ? kv_move_kernel<true, 8>
                          : per == 16 ? kv_move_kernel<true, 16>
                                      : kv_move_kernel<true, 32>)
                       : (per == 8    ? kv_move_kernel<false, 8>
                          : per == 16 ? kv_move_kernel<false, 16>
                                      : kv_move_kernel<false, 32>);
  hipLaunchKernelGGL(kern, dim3((unsigned)(n_head_kv * slices), (unsigned)n_pools), dim3(MOVE_THREADS),
                     0, as_stream(stream), pools, n_cells, n_head_kv, head_dim, src, dst, (int)n, shape);
  return hip_check(hipGetLastError(), "kv_move");
}
