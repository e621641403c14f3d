// The KV pool in Q4_0: 4-bit values and an f16 scale per 32 (gfx950).
#include <type_traits>

#include "kvstore.h"

namespace lgmlh {

// A workgroup takes W consecutive tokens (64, or 16 of a call of few) of one head
// of K or V, 8 values a thread and step: K's are the word they are stored as, V's
// turn in LDS (kvstore.h), or of few tokens go byte by byte. Bound by the rows: 8192 of 8
// heads of 128, 76 MB, take 18 us; 64 rows 3.7 us, dependent reads.
constexpr int Q4_THREADS = KV_THREADS;
constexpr int Q4_FEW = 16;  // W of a call of few tokens, whose V goes byte by byte, without a turn
// KV heads: the bytes of a block, 36 D for each, are counted in 31 bits.
constexpr int Q4_HEADS = 65535;
static_assert((int64_t)Q4_HEADS * q4_tile_bytes(256) < INT32_MAX, "tile_of");

template <int D, typename P>
__device__ __forceinline__ P *q4_tile(P *head, int64_t c, int Hkv) {
  return kv_tile<LGMLH_Q4_0, D>(head, c, Hkv);
}

// x (n, Hkv D) f32 rows into their cells, in the format's steps (quant8).
template <int D, int W>
__global__ void __launch_bounds__(Q4_THREADS)
kv_store_q4_kernel(uint8_t *__restrict__ kp, uint8_t *__restrict__ vp, int64_t n_cells,
                   const float *__restrict__ ks, const float *__restrict__ vs,
                   const int64_t *__restrict__ cells, int64_t n, int Hkv) {
  const int h = blockIdx.x % (uint32_t)Hkv;
  const int64_t j0 = (int64_t)(blockIdx.x / (uint32_t)Hkv) * W;
  const float *src = (blockIdx.y ? vs : ks) + (j0 * Hkv + h) * D;
  const bool is_v = blockIdx.y;
  if constexpr (W > Q4_FEW) {
    if (is_v) {
      __shared__ VTurn<LGMLH_Q4_0, D, W> turn;
      turn.store(src, (int64_t)Hkv * D, vp, h, Hkv, cells, j0, n, n_cells);
      return;
    }
  }
  constexpr int G8 = D / 8, STEP = Q4_THREADS / G8, IT = (W + STEP - 1) / STEP;
  __shared__ uint16_t scale[D / 32 * W];
  __shared__ int64_t cell[W];
  const int tid = threadIdx.x, g8 = tid % G8, t0 = tid / G8;
  const int left = (int)(n - j0 < W ? n - j0 : W);
  uint8_t *pool = (is_v ? vp : kp) + (int64_t)h * q4_tile_bytes(D);
  f32x4 x[IT][2];
#pragma unroll
  for (int i = 0; i < IT; i++) {
    const int t = t0 + i * STEP;
    const float *row = src + (int64_t)t * Hkv * D + 8 * g8;
    x[i][0] = t < left ? *(const f32x4_u *)row : f32x4{0, 0, 0, 0};
    x[i][1] = t < left ? *(const f32x4_u *)(row + 4) : f32x4{0, 0, 0, 0};
  }
  if (tid < W) {
    const int64_t c = tid < left ? cells[j0 + tid] : -1;
    cell[tid] = c < n_cells ? c : -1;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < IT; i++) {
    const int t = t0 + i * STEP;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = x[i][e >> 2][e & 3];
    uint32_t q[8];
    const float d = quant8<LGMLH_Q4_0>(v, q);
    if (t >= left) continue;  // whole blocks of lanes leave together
    if (g8 % 4 == 0) scale[g8 / 4 * W + t] = f2h(d);
    const int64_t c = cell[t];
    if (W > Q4_FEW || !is_v) {
      if (c >= 0) *(uint32_t *)(q4_tile<D>(pool, c, Hkv) + q4_k_at(D, (int)c & 63, 8 * g8)) = q4_k_word(q);
      continue;
    }
    // dims r and r + 16 share a byte: of the eight of a lane and the one two on, each writes four
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) w |= q[e] << 4 * e;
    const uint32_t other = __shfl_xor(w, 2);
    const int high = g8 & 2, r = 8 * (g8 & 1) + 2 * high;
    const uint32_t lo = (high ? other : w) >> 8 * high, hi = (high ? w : other) >> 8 * high;
    uint8_t *to = q4_tile<D>(pool, c < 0 ? 0 : c, Hkv) + q4_v_at(16 * (g8 / 4) + r, (int)c & 63);
    if (c >= 0)
#pragma unroll
      for (int e = 0; e < 4; e++) to[64 * e] = (uint8_t)((lo >> 4 * e & 15) | (hi >> 4 * e & 15) << 4);
  }
  __syncthreads();
  // the scales with tokens along the lanes, as a tile has them
  for (int i = tid; i < D / 32 * W; i += Q4_THREADS) {
    const int64_t c = cell[i % W];
    if (c >= 0) *(uint16_t *)(q4_tile<D>(pool, c, Hkv) + q4_scale_at(D, i / W, (int)c & 63)) = scale[i];
  }
}

// 16 bytes of a row, f32 or f16 of (n - 8) d, n the low halves of the bytes of one or two
// words.
template <typename OutT>
struct RowPiece {
  static constexpr int N = 16 / sizeof(OutT);
  typedef OutT T __attribute__((ext_vector_type(N), aligned(sizeof(OutT))));
  T y;
  __device__ __forceinline__ RowPiece(uint32_t n0, uint32_t n1, float d) {
#pragma unroll
    for (int e = 0; e < N; e++) y[e] = (OutT)(d * ((float)((e < 4 ? n0 : n1) >> 8 * (e & 3) & 15) - 8.0f));
  }
};

// Threads of a cell in the read back of K: 16 bytes of a row's in each of U blocks of 32
// dims, or of f16 in every other one, so that eight write a line's 128 bytes.
template <typename OutT>
__host__ __device__ constexpr int q4_k_threads(int D) {
  return D * sizeof(OutT) / 16 / q4_k_words(D) * (4 / sizeof(OutT));
}

// K's cells as rows (n, Hkv D), from a load's U words (of f32 the low or the high ones'
// half). The rows pass the caches by, whole 128-byte lines a store. The context of 8
// sequences of 4096 tokens, 8 heads of 128, as f16 rows of K and V: 31 us, 5.5 TB/s (64
// bytes of a line at a time 37; cached stores of 8 bytes a thread 49).
template <int D, typename OutT>
__global__ void __launch_bounds__(Q4_THREADS)
kv_gather_q4_k_kernel(const uint8_t *__restrict__ pool, int64_t n_cells,
                      const int64_t *__restrict__ cells, int64_t n, int Hkv, OutT *__restrict__ out) {
  typedef RowPiece<OutT> Piece;
  constexpr int N = Piece::N, U = q4_k_words(D), L = 32 / N, S = N / 4, PER = q4_k_threads<OutT>(D);
  const int h = blockIdx.x % (uint32_t)Hkv;
  const int64_t t = (int64_t)(blockIdx.x / (uint32_t)Hkv) * (Q4_THREADS / PER) + threadIdx.x / PER;
  const int k = threadIdx.x % PER, j = k / (L * S), odd = k / L % S, dim = k % L * N;
  if (t >= n) return;
  const int64_t c = cells[t];
  const bool in = (uint64_t)c < (uint64_t)n_cells;
  const int cell = (int)c & 63;
  uint32_t w[U / S];
  float d[U / S];
#pragma unroll
  for (int i = 0; i < U / S; i++) {
    w[i] = 0;
    d[i] = 0.0f;
  }
  if (in) {
    const uint8_t *tile = q4_tile<D>(pool + (int64_t)h * q4_tile_bytes(D), c, Hkv);
    typedef uint32_t uU __attribute__((ext_vector_type(U)));
    const uU r = *(const uU *)(tile + q4_k_at(D, cell, 32 * U * j + dim / 8 * 8));
#pragma unroll
    for (int i = 0; i < U / S; i++) {
      w[i] = odd ? r[S * i + S - 1] : r[S * i];
      d[i] = h2f(*(const uint16_t *)(tile + q4_scale_at(D, U * j + S * i + odd, cell)));
    }
  }
  OutT *row = out + (t * Hkv + h) * (int64_t)D + 32 * (U * j + odd) + dim;
#pragma unroll
  for (int i = 0; i < U / S; i++) {
    // dim e at bits 4 (e / 2) + 16 (e % 2): in order, a byte each
    uint32_t v[N / 4];
#pragma unroll
    for (int b = 0; b < N / 4; b++) {
      const uint32_t s = w[i] >> (8 * b + 2 * (dim % 8));
      v[b] = (s & 15) | (s >> 16 & 15) << 8 | (s >> 4 & 15) << 16 | (s >> 20 & 15) << 24;
    }
    const Piece y(v[0], v[N / 4 - 1], d[i]);
    __builtin_nontemporal_store(y.y, (typename Piece::T *)(row + 32 * S * i));
  }
}

// V's cells as rows, of few tokens: each value from its own byte, behind nothing but the
// cell's number.
template <int D, typename OutT>
__global__ void __launch_bounds__(Q4_THREADS)
kv_gather_q4_v_few_kernel(const uint8_t *__restrict__ pool, int64_t n_cells,
                          const int64_t *__restrict__ cells, int64_t n, int Hkv, OutT *__restrict__ out) {
  typedef RowPiece<OutT> Piece;
  constexpr int N = Piece::N, PER = D / N;
  const int h = blockIdx.x % (uint32_t)Hkv;
  const int64_t t = (int64_t)(blockIdx.x / (uint32_t)Hkv) * (Q4_THREADS / PER) + threadIdx.x / PER;
  const int dim = threadIdx.x % PER * N;
  if (t >= n) return;
  const int64_t c = cells[t];
  uint32_t v[2] = {0, 0};
  float d = 0.0f;
  if ((uint64_t)c < (uint64_t)n_cells) {
    const int cell = (int)c & 63;
    const uint8_t *tile = q4_tile<D>(pool + (int64_t)h * q4_tile_bytes(D), c, Hkv);
    const uint8_t *from = tile + q4_v_at(dim / 32 * 16 + dim % 16, cell);
    d = h2f(*(const uint16_t *)(tile + q4_scale_at(D, dim / 32, cell)));
#pragma unroll
    for (int e = 0; e < N; e++) v[e / 4] |= (uint32_t)(from[64 * e] >> dim % 32 / 16 * 4) << 8 * (e % 4);
  }
  *(typename Piece::T *)(out + (t * Hkv + h) * (int64_t)D + dim) = Piece(v[0], v[1], d).y;
}

// V's cells as rows: whole groups of 8 cells through LDS, as the store the other way
// round.
template <int D, int W, typename OutT>
__global__ void __launch_bounds__(Q4_THREADS)
kv_gather_q4_v_kernel(const uint8_t *__restrict__ pool, int64_t n_cells,
                      const int64_t *__restrict__ cells, int64_t n, int Hkv, OutT *__restrict__ out) {
  typedef RowPiece<OutT> Piece;  // of a thread and step, the halves of N bytes
  constexpr int N = Piece::N, GN = D / N, STEP = Q4_THREADS / GN, PAD = D / 2 + 4;
  constexpr int ROWS = W + CELL_HALO, NS = W + 8, GROUPS = W / CELL_GROUP;
  __shared__ CellWindow<W> win;
  __shared__ __align__(4) uint8_t turn[ROWS * PAD];
  __shared__ uint8_t mine[ROWS];  // the rows of turn that are this workgroup's
  __shared__ uint16_t scale[D / 32 * NS];
  const int tid = threadIdx.x, h = blockIdx.x % (uint32_t)Hkv;
  const int64_t j0 = (int64_t)(blockIdx.x / (uint32_t)Hkv) * W;
  const uint8_t *head = pool + (int64_t)h * q4_tile_bytes(D);
  win.fill(cells, j0, n, n_cells, true);
#pragma unroll
  for (int k = 0; k < (D / 32 * NS + Q4_THREADS - 1) / Q4_THREADS; k++) {
    const int i = tid + k * Q4_THREADS, t = i % NS;
    if (i >= D / 32 * NS) break;
    const int64_t c = t < ROWS ? win.cell(t) : -1;
    scale[i] = c < 0 ? 0 : *(const uint16_t *)(q4_tile<D>(head, c, Hkv) + q4_scale_at(D, i / NS, (int)c & 63));
  }
  const int ng = win.n_lead, no = win.n_lone;
  if (tid < ROWS) mine[tid] = tid < W && win.cell(tid) < 0;  // a cell outside: zeros
  constexpr int GI = (GROUPS * D / 2 + Q4_THREADS - 1) / Q4_THREADS;
  const int g = tid % GROUPS, lead = g < ng ? win.lead[g] : -1;
  u32x2 q8[GI];
  if (lead >= 0) {
    const int64_t c = win.cell(lead);
    const uint8_t *tile = q4_tile<D>(head, c, Hkv) + q4_v_at(0, (int)c & 63);
#pragma unroll
    for (int i = 0; i < GI; i++) {
      const int p = tid / GROUPS + i * (Q4_THREADS / GROUPS);
      if (p < D / 2) q8[i] = *(const u32x2 *)(tile + 64 * p);
    }
  }
  __syncthreads();
  if (tid < 8 * ng) mine[win.lead[tid >> 3] + (tid & 7)] = 1;
  if (tid < no) mine[win.lone[tid]] = 1;
  if (lead >= 0) {
#pragma unroll
    for (int i = 0; i < GI; i++) {
      const int p = tid / GROUPS + i * (Q4_THREADS / GROUPS);
      uint8_t *s8 = turn + lead * PAD + p;
      if (p < D / 2)
#pragma unroll
        for (int e = 0; e < 8; e++) s8[e * PAD] = (uint8_t)(q8[i][e >> 2] >> 8 * (q4_v_byte(e) & 3));
    }
  }
  const int sh = lone_bits(no);
  if (const int k = tid & ((1 << sh) - 1); k < no) {
    const int t = win.lone[k];
    const int64_t c = win.cell(t);
    const uint8_t *tile = q4_tile<D>(head, c, Hkv) + q4_v_at(0, (int)c & 63);
#pragma unroll 8
    for (int p = tid >> sh; p < D / 2; p += Q4_THREADS >> sh) turn[t * PAD + p] = tile[64 * p];
  }
  __syncthreads();
  const int dim = tid % GN * N, j = dim / 32, high = dim / 16 % 2 * 4;  // dims 32 j + 16 of the bytes' high halves
  const int left = n - j0 < ROWS ? (int)(n - j0) : ROWS;
#pragma unroll 4
  for (int t = tid / GN; t < left; t += STEP) {
    if (!mine[t]) continue;
    const bool in = win.cell(t) >= 0;
    const uint32_t *w = (const uint32_t *)(turn + t * PAD + 16 * j + dim % 16);
    const float d = in ? h2f(scale[j * NS + t]) : 0.0f;
    const Piece y(in ? w[0] >> high : 0, in && N == 8 ? w[N / 8] >> high : 0, d);
    __builtin_nontemporal_store(y.y, (typename Piece::T *)(out + ((j0 + t) * Hkv + h) * (int64_t)D + dim));
  }
}

// Tokens of a workgroup: 64 (32 of heads of 256), but 16 where that makes fewer than 256
// workgroups, whose V goes without a turn in LDS. 64 rows of 8 heads of 128: 3.7 us stored, V
// read back in 2.7 (16 tokens with turns 4.7 and 4.5, 64 7.9 and 7.6); with turns 8192 rows
// stored and read back took 39 us with 16, 35 with 64; 32768 as f16 rows 47 and 37 (before K's
// lines went whole).
constexpr int q4_tokens(int D) { return D > 128 ? 32 : 64; }
static bool q4_small(int64_t n, int n_head_kv, int kinds, int D) {
  return (n + q4_tokens(D) - 1) / q4_tokens(D) * n_head_kv * kinds < 256;
}
static bool q4_head(int D) { return D == 64 || D == 128 || D == 256; }

}  // namespace lgmlh

using namespace lgmlh;

extern "C" int64_t lgmlh_kv_q4_layer_bytes(int64_t n_cells, int n_head_kv, int head_dim) {
  if (n_cells <= 0 || n_cells % KV_BLOCK || n_head_kv <= 0 || !q4_head(head_dim)) return -1;
  return n_cells / KV_BLOCK * n_head_kv * q4_tile_bytes(head_dim);
}

extern "C" int lgmlh_kv_store_q4(void *kpool, void *vpool, int64_t n_cells, int n_head_kv,
                                 int head_dim, const float *k_src, const float *v_src,
                                 const int64_t *cells, const int64_t *h_cells, int64_t n,
                                 void *stream) {
  if (!kpool || !vpool || !k_src || !v_src || !cells || n < 0 || n_cells <= 0 ||
      n_cells > CELLS_MAX || n_cells % KV_BLOCK || n_head_kv <= 0 || n_head_kv > Q4_HEADS ||
      n >= CELL_ROWS / n_head_kv || !q4_head(head_dim)) {
    set_error("kv_store_q4: bad arguments (heads of 64, 128 or 256)");
    return LGMLH_EINVAL;
  }
  if (((uintptr_t)kpool | (uintptr_t)vpool) & 15) {
    set_error("kv_store_q4: pools are 16-byte aligned");
    return LGMLH_EINVAL;
  }
  const bool small = q4_small(n, n_head_kv, 2, head_dim);
  const int w = small ? Q4_FEW : q4_tokens(head_dim);
  const int64_t groups = (n + w - 1) / w * n_head_kv;
  LGMLH_TRY(check_groups(groups, "kv_store_q4"));
  LGMLH_TRY(check_write_cells(h_cells, n, n_cells, "kv_store_q4"));
  if (n == 0) return LGMLH_OK;
  // heads fastest: those of the same rows run together
  const dim3 grid((unsigned)groups, 2);
  const auto kern = head_dim == 64    ? (small ? kv_store_q4_kernel<64, Q4_FEW> : kv_store_q4_kernel<64, 64>)
                    : head_dim == 128 ? (small ? kv_store_q4_kernel<128, Q4_FEW> : kv_store_q4_kernel<128, 64>)
                                      : (small ? kv_store_q4_kernel<256, Q4_FEW> : kv_store_q4_kernel<256, 32>);
  hipLaunchKernelGGL(kern, grid, dim3(Q4_THREADS), 0, as_stream(stream), (uint8_t *)kpool,
                     (uint8_t *)vpool, n_cells, k_src, v_src, cells, n, n_head_kv);
  return hip_check(hipGetLastError(), "kv_store_q4");
}

extern "C" int lgmlh_kv_gather_q4(const void *pool, int which, int64_t n_cells, int n_head_kv,
                                  int head_dim, const int64_t *cells, int64_t n, void *out,
                                  int out_type, void *stream) {
  if (!pool || !cells || !out || n < 0 || (which != 0 && which != 1) || n_cells <= 0 ||
      n_cells > CELLS_MAX || n_cells % KV_BLOCK || n_head_kv <= 0 || n_head_kv > Q4_HEADS ||
      n >= CELL_ROWS / (head_dim == 256 ? 2 : 1) / n_head_kv || !q4_head(head_dim) ||
      (out_type != LGMLH_F32 && out_type != LGMLH_F16)) {
    set_error("kv_gather_q4: bad arguments (heads of 64, 128 or 256; out f32 or f16)");
    return LGMLH_EINVAL;
  }
  if ((uintptr_t)pool & 15) {
    set_error("kv_gather_q4: pools are 16-byte aligned");
    return LGMLH_EINVAL;
  }
  if (n == 0) return LGMLH_OK;
  const bool small = q4_small(n, n_head_kv, 1, head_dim);
  hipStream_t st = as_stream(stream);
  int rc = LGMLH_OK;
  auto go = [&](auto out_t) {
    typedef decltype(out_t) T;
    auto launch = [&](auto kern, int w) {
      const int64_t groups = (n + w - 1) / w * n_head_kv;
      rc = check_groups(groups, "kv_gather_q4");
      if (rc == LGMLH_OK)
        hipLaunchKernelGGL(kern, dim3((unsigned)groups), dim3(Q4_THREADS), 0, st, (const uint8_t *)pool, n_cells,
                           cells, n, n_head_kv, (T *)out);
    };
    auto of = [&](auto d) {
      constexpr int D = decltype(d)::value, big = q4_tokens(D);
      if (which)
        small ? launch(kv_gather_q4_v_few_kernel<D, T>, Q4_THREADS * (16 / (int)sizeof(T)) / D)
              : launch(kv_gather_q4_v_kernel<D, big, T>, big);
      else
        launch(kv_gather_q4_k_kernel<D, T>, Q4_THREADS / q4_k_threads<T>(D));
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
  LGMLH_TRY(rc);
  return hip_check(hipGetLastError(), "kv_gather_q4");
}
