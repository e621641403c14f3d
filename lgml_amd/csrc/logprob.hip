// Log probabilities of given tokens, entropy and the most likely tokens of rows
// of logits (gfx950).
//
// log p(i) = x_i - M - log Z, Z = sum e^(x - M); H = log Z - (1 / Z) sum e^(x -
// M) (x - M). A row is read once: a workgroup takes a slice of it into
// registers, finds its largest value m, and leaves C (how many are equal to m), S
// = sum over the others of e^(x - m) and T = sum e^(x - m) (x - m). Z = C + S is
// kept apart until the end, log Z = log C + log1p(S / C), so that a row whose
// mass is all in one token keeps the digits of its -log p = log1p(S), which 1 + S
// in f32 loses: relative to it they are off by 6e-8 where the next token is as
// likely, 8e-7 where it is e^-20 as likely, 2e-6 at e^-60 (d = x - M and its
// product are rounded), until the terms e^d come below 2^-126, where they are 0.
// It also leaves the largest value of every 64 tokens.
//
// The k most likely tokens are in the k groups of 64 with the largest (value,
// first index) keys: a token of another group is behind k tokens, one of each
// of those. So a second launch, a workgroup per row, joins the slices, selects k
// of the groups' maxima and then k of those groups' 64 k values.
//
// 1000 rows of 151936 and their 20 first: the slices take 119 us, 608 MB at 5.1
// TB/s, a large read's rate being 6.2; the rows 19. One row of 128256 takes 3.2 +
// 7.8 us: two launches' reads one after another, in the second one the maxima,
// then the chosen groups.
#include <math.h>

#include "common.h"

namespace lgmlh {

constexpr int LP_THREADS = 256, LP_GROUP = 64, LP_TOP = 64, LP_IDS = 64;
constexpr int64_t LP_COLS = 1 << 20;  // the largest row: 64 groups a thread, 64 x 64 candidates
constexpr float LP_LOG2E = 1.4426950408889634f;
// Vectors of 4 a thread holds: a slice of 8192, or of 2048 where the larger ones
// make few workgroups (one row of 128256: 16 of them, and 63 of the smaller).
constexpr int LP_WIDE = 8, LP_SLIM = 2;

struct Slice {
  float m, c, s, t;
};

// A value's order as an integer (-0 and 0 the same, NaN as -inf); never 0.
__device__ __forceinline__ uint32_t order_of(float x) {
  x = x != x ? -INFINITY : x + 0.0f;
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t order) {
  return __builtin_bit_cast(float, order & 0x80000000u ? order ^ 0x80000000u : ~order);
}
// e^d for d <= 0 or NaN
__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(d * LP_LOG2E); }

__device__ __forceinline__ float wave_sum(float v) {
  for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o);
  return v;
}

template <int LOADS>
__global__ void __launch_bounds__(LP_THREADS)
lp_slice_kernel(const float *__restrict__ x, int64_t n, int slices, Slice *__restrict__ part,
                float *__restrict__ groups, int64_t n_groups) {
  __shared__ float red[4][LP_THREADS / 64];
  const int tid = threadIdx.x, wave = tid >> 6;
  const int64_t r = blockIdx.x / (uint32_t)slices, slice = blockIdx.x % (uint32_t)slices;
  const int64_t c0 = slice * (4 * LP_THREADS * LOADS) + 4 * tid;
  const float *row = x + r * n;
  f32x4 v[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; i++) {
    const int64_t c = c0 + 4 * LP_THREADS * i;
    if (c + 4 <= n) {
      v[i] = *(const f32x4_u *)(row + c);
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++) v[i][e] = c + e < n ? row[c + e] : -INFINITY;
    }
  }
  float m = -INFINITY;  // fmaxf passes NaN by; it comes back in the sums
#pragma unroll
  for (int i = 0; i < LOADS; i++) {
    float g = fmaxf(fmaxf(v[i][0], v[i][1]), fmaxf(v[i][2], v[i][3]));
    g = fmaxf(g, -INFINITY);
    if (groups) {
      g = group_max<16>(g);  // 16 lanes hold a group of 64
      const int64_t c = c0 + 4 * LP_THREADS * i;
      if ((tid & 15) == 0 && c < n) groups[r * n_groups + c / LP_GROUP] = g;
    }
    m = fmaxf(m, g);
  }
  m = group_max<64>(m);
  if ((tid & 63) == 0) red[0][wave] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < LP_THREADS / 64; w++) m = fmaxf(m, red[0][w]);
  __syncthreads();
  float s = 0.0f, t = 0.0f;
  int nc = 0;
#pragma unroll
  for (int i = 0; i < LOADS; i++)
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const bool top = v[i][e] == m;
      nc += __builtin_popcountll(__builtin_amdgcn_ballot_w64(top));  // the wave's
      const float d = v[i][e] - m, p = top ? 0.0f : exp_of(d);
      s += p;
      t += p * fmaxf(d, -200.0f);  // (0 x -inf, 0 x NaN of inf - inf; p is 0 long before)
    }
  float c = (float)nc;
  s = wave_sum(s);
  t = wave_sum(t);
  if ((tid & 63) == 0) {
    red[1][wave] = c;
    red[2][wave] = s;
    red[3][wave] = t;
  }
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < LP_THREADS / 64; w++) {
      c += red[1][w];
      s += red[2][w];
      t += red[3][w];
    }
    part[blockIdx.x] = Slice{m, c, s, t};
  }
}

// b into a: two parts of a row. Parts of the same maximum add up, else the
// smaller one's C joins its S.
__device__ __forceinline__ Slice join(Slice a, Slice b) {
  if (b.m > a.m) {
    const Slice o = a;
    a = b;
    b = o;
  }
  if (b.m == a.m) return Slice{a.m, a.c + b.c, a.s + b.s, a.t + b.t};
  const float d = fmaxf(b.m - a.m, -200.0f), w = exp_of(d);
  return Slice{a.m, a.c, a.s + w * (b.c + b.s), a.t + w * (b.t + d * (b.c + b.s))};
}

constexpr int LP_HELD = 16;  // groups' values a thread holds (rows of up to 262144)
constexpr int LP_LIST = LP_TOP * LP_GROUP;  // the most candidates

// The k largest of keys (value, then ~index: all different, none 0) are found by
// cuts: a thread takes every 256th key, and where at least k threads' maxima are at
// or above a cut, so are the k largest keys. The cut grows bit by bit from the top;
// each wave holds all 256 maxima, 4 a lane, and counts by ballots, so the waves
// agree without a barrier. It stops at the first cut that k to `most` maxima reach
// (most >= k; with all 64 bits set exactly k do). 0 where fewer than k threads have
// a key.
__device__ __forceinline__ uint64_t cut_of(const uint64_t *tmax, int k, int most) {
  const int lane = threadIdx.x & 63;
  uint64_t key[LP_THREADS / 64];
#pragma unroll
  for (int i = 0; i < LP_THREADS / 64; i++) key[i] = tmax[64 * i + lane];
  uint64_t cut = 0;
  for (int bit = 63; bit >= 0; bit--) {
    const uint64_t c = cut | (uint64_t)1 << bit;
    int n = 0;
#pragma unroll
    for (int i = 0; i < LP_THREADS / 64; i++)
      n += __builtin_popcountll(__builtin_amdgcn_ballot_w64(key[i] >= c));
    if (n < k) continue;
    cut = c;
    if (n <= most) break;
  }
  return cut;
}

struct Select {
  uint64_t tmax[LP_THREADS];
  int count;
};
// The number of list's n keys left, at most 256, the k largest among them.
__device__ __forceinline__ int narrow(Select &sh, uint64_t *list, int n, int k) {
  const int tid = threadIdx.x;
  while (n > LP_THREADS) {  // n falls: at most k threads' keys stay, of 4 k or more
    uint64_t kept[LP_LIST / LP_THREADS], best = 0;  // a thread's keys
#pragma unroll
    for (int j = 0; j < LP_LIST / LP_THREADS; j++) {
      const int i = tid + j * LP_THREADS;
      kept[j] = i < n ? list[i] : 0;
      best = kept[j] > best ? kept[j] : best;
    }
    sh.tmax[tid] = best;
    if (tid == 0) sh.count = 0;
    __syncthreads();
    const uint64_t cut = cut_of(sh.tmax, k, k);
#pragma unroll
    for (int j = 0; j < LP_LIST / LP_THREADS; j++)
      if (kept[j] && kept[j] >= cut) list[atomicAdd(&sh.count, 1)] = kept[j];
    __syncthreads();
    n = sh.count;
    __syncthreads();
  }
  return n;
}

// How many of list's m keys (m <= 256) are above a thread's own; the keys after
// the last are zeros up to a multiple of 8, so that 8 reads are in flight.
__device__ __forceinline__ int rank_of(const uint64_t *list, int m, uint64_t key) {
  int above = 0;
  for (int j = 0; j < m; j += 8)
#pragma unroll
    for (int i = 0; i < 8; i++) above += list[j + i] > key;
  return above;
}

// One workgroup per row.
__global__ void __launch_bounds__(LP_THREADS)
lp_row_kernel(const float *__restrict__ x, int64_t n, int slices, const Slice *__restrict__ part,
              const float *__restrict__ groups, int n_groups, const int32_t *__restrict__ ids,
              int n_ids, float *__restrict__ id_lp, float *__restrict__ entropy, int k,
              int32_t *__restrict__ top_ids, float *__restrict__ top_lp) {
  __shared__ Slice red[LP_THREADS / 64];
  __shared__ Select sh;
  __shared__ uint64_t list[LP_LIST + 8];
  __shared__ int chosen[LP_TOP];
  __shared__ uint32_t last;  // the least of the chosen groups' values
  const int tid = threadIdx.x;
  const int64_t r = blockIdx.x;
  const float *row = x + r * n;
  // the groups' keys: (largest value, first)
  const float *grow = groups ? groups + r * n_groups : nullptr;
  if (k == 0) n_groups = 0;
  auto key_of = [](float v, uint32_t i) { return (uint64_t)order_of(v) << 32 | (uint32_t)~i; };
  if (tid == 0) sh.count = 0;
  // a thread's values stay in registers (all their loads at once) up to 16
  float held[LP_HELD];
#pragma unroll
  for (int j = 0; j < LP_HELD; j++) {
    const int i = tid + j * LP_THREADS;
    held[j] = i < n_groups ? grow[i] : 0.0f;
  }
  // a given token's logit, on its way meanwhile
  const int32_t id = tid < n_ids ? ids[r * n_ids + tid] : -1;
  const float given = id >= 0 && id < n ? row[id] : -INFINITY;
  // the parts of the row join while the values come
  Slice a = {-INFINITY, 0.0f, 0.0f, 0.0f};
  for (int i = tid; i < slices; i += LP_THREADS) a = join(a, part[r * slices + i]);
  for (int o = 1; o < 64; o <<= 1)
    a = join(a, Slice{__shfl_xor(a.m, o), __shfl_xor(a.c, o), __shfl_xor(a.s, o), __shfl_xor(a.t, o)});
  if ((tid & 63) == 0) red[tid >> 6] = a;
  uint64_t best = 0;
#pragma unroll
  for (int j = 0; j < LP_HELD; j++) {
    if (j * LP_THREADS >= n_groups) break;
    const int i = tid + j * LP_THREADS;
    const uint64_t key = i < n_groups ? key_of(held[j], i) : 0;
    best = key > best ? key : best;
  }
  for (int i = tid + LP_HELD * LP_THREADS; i < n_groups; i += LP_THREADS) {
    const uint64_t key = key_of(grow[i], i);
    best = key > best ? key : best;
  }
  sh.tmax[tid] = best;
  __syncthreads();
  a = red[0];
  for (int w = 1; w < LP_THREADS / 64; w++) a = join(a, red[w]);
  // a row of -inf alone has no distribution: log p is -inf, H 0
  const bool none = a.m == -INFINITY && a.s == a.s;
  const float log_z = a.c == 1.0f ? log1pf(a.s) : logf(a.c) + log1pf(a.s / a.c);
  auto log_p = [&](float v) {
    if (none) return -INFINITY;
    return v == a.m ? -log_z : (v - a.m) - log_z;  // (+inf, or equal: no inf - inf)
  };
  if (entropy && tid == 0) entropy[r] = none ? 0.0f : log_z - a.t / (a.c + a.s);
  if (tid < n_ids) id_lp[r * n_ids + tid] = id >= 0 && id < n ? log_p(given) : -INFINITY;
  if (k == 0) return;
  // the groups at or above the cut; a few more than k may stay, as many as the
  // list holds
  const int per = (n_groups + LP_THREADS - 1) / LP_THREADS, hold = LP_LIST / per;
  const uint64_t cut = cut_of(sh.tmax, k, 2 * k < hold ? 2 * k : hold);
#pragma unroll
  for (int j = 0; j < LP_HELD; j++) {
    if (j * LP_THREADS >= n_groups) break;
    const int i = tid + j * LP_THREADS;
    const uint64_t key = i < n_groups ? key_of(held[j], i) : 0;
    if (key && key >= cut) list[atomicAdd(&sh.count, 1)] = key;
  }
  for (int i = tid + LP_HELD * LP_THREADS; i < n_groups; i += LP_THREADS) {
    const uint64_t key = key_of(grow[i], i);
    if (key >= cut) list[atomicAdd(&sh.count, 1)] = key;
  }
  __syncthreads();
  int m = sh.count;
  __syncthreads();
  m = narrow(sh, list, m, k);
  const int kg = k < n_groups ? k : n_groups;
  if (tid < 8) list[m + tid] = 0;
  __syncthreads();
  if (tid < m) {
    const uint64_t key = list[tid];
    const int above = rank_of(list, m, key);
    if (above < kg) chosen[above] = (int)~(uint32_t)key;
    if (above == kg - 1) last = (uint32_t)(key >> 32);
  }
  if (tid == 0) sh.count = 0;
  __syncthreads();
  // their tokens: at or above the last chosen group's largest value
  const uint32_t floor_v = last;
  constexpr int IT = LP_LIST / LP_THREADS;
  float x_of[IT];
#pragma unroll
  for (int j = 0; j < IT; j++) {
    const int i = tid + j * LP_THREADS;
    const int64_t c = i < kg * LP_GROUP ? (int64_t)chosen[i / LP_GROUP] * LP_GROUP + i % LP_GROUP : n;
    x_of[j] = c < n ? row[c] : 0.0f;
  }
#pragma unroll
  for (int j = 0; j < IT; j++) {
    if (j * LP_THREADS >= kg * LP_GROUP) break;
    const int i = tid + j * LP_THREADS;
    const int64_t c = i < kg * LP_GROUP ? (int64_t)chosen[i / LP_GROUP] * LP_GROUP + i % LP_GROUP : n;
    const uint64_t key = key_of(x_of[j], (uint32_t)c);
    if (c < n && ((uint32_t)(key >> 32) >= floor_v || kg < k)) list[atomicAdd(&sh.count, 1)] = key;
  }
  __syncthreads();
  m = sh.count;
  __syncthreads();
  m = narrow(sh, list, m, k);
  if (tid < 8) list[m + tid] = 0;
  __syncthreads();
  if (tid < m) {
    const uint64_t key = list[tid];
    const int above = rank_of(list, m, key);
    if (above < k) {
      const uint32_t id = ~(uint32_t)key;
      if (top_ids) top_ids[r * k + above] = (int32_t)id;
      // (a NaN is back as -inf, but then log Z is NaN)
      if (top_lp) top_lp[r * k + above] = log_p(value_of((uint32_t)(key >> 32)));
    }
  }
}

static bool lp_wide(int64_t n_rows, int64_t n_cols) {
  return n_rows * (n_cols / (4 * LP_THREADS * LP_WIDE)) >= 512;
}
static int lp_slices(int64_t n_rows, int64_t n_cols) {
  const int64_t per = 4 * LP_THREADS * (lp_wide(n_rows, n_cols) ? LP_WIDE : LP_SLIM);
  return (int)((n_cols + per - 1) / per);
}

}  // namespace lgmlh

using namespace lgmlh;

extern "C" size_t lgmlh_log_probs_workspace(int64_t n_rows, int64_t n_cols, int n_top) {
  if (n_rows <= 0 || n_cols <= 0 || n_cols > LP_COLS || n_top < 0 || n_top > LP_TOP) return 0;
  const int64_t most = (n_cols + 4 * LP_THREADS * LP_SLIM - 1) / (4 * LP_THREADS * LP_SLIM);
  const int64_t groups = n_top ? (n_cols + LP_GROUP - 1) / LP_GROUP : 0;
  return (size_t)n_rows * ((size_t)most * sizeof(Slice) + (size_t)groups * sizeof(float));
}

extern "C" int lgmlh_log_probs(const float *logits, int64_t n_rows, int64_t n_cols,
                               const int32_t *ids, int n_ids, float *id_lp, float *entropy,
                               int n_top, int32_t *top_ids, float *top_lp, void *workspace,
                               size_t ws_bytes, void *stream) {
  if (!logits || n_rows < 0 || n_rows > INT32_MAX || n_cols <= 0 || n_ids < 0 || n_top < 0 ||
      (n_ids > 0 && (!ids || !id_lp)) || (n_top > 0 && !top_ids && !top_lp)) {
    set_error("log_probs: bad arguments");
    return LGMLH_EINVAL;
  }
  if (n_cols > LP_COLS || n_ids > LP_IDS || n_top > LP_TOP || n_top > n_cols) {
    set_error("log_probs: rows of %lld, %d given, %d alternatives (at most %lld, %d, %d and the row)",
              (long long)n_cols, n_ids, n_top, (long long)LP_COLS, LP_IDS, LP_TOP);
    return LGMLH_EINVAL;
  }
  if (n_rows == 0) return LGMLH_OK;
  const size_t need = lgmlh_log_probs_workspace(n_rows, n_cols, n_top);
  if (!workspace || ws_bytes < need || ((uintptr_t)workspace & 15)) {
    set_error("log_probs: workspace of %zu bytes, need %zu (16-byte aligned)", ws_bytes, need);
    return LGMLH_ENOMEM;
  }
  const int slices = lp_slices(n_rows, n_cols);
  const int n_groups = (int)((n_cols + LP_GROUP - 1) / LP_GROUP);
  Slice *part = (Slice *)workspace;
  float *groups = n_top ? (float *)(part + n_rows * slices) : nullptr;
  if (n_rows * slices >= (int64_t)1 << 24) {  // a launch has fewer than 2^32 threads
    set_error("log_probs: %lld rows of %lld in one call", (long long)n_rows, (long long)n_cols);
    return LGMLH_EINVAL;
  }
  hipStream_t st = as_stream(stream);
  const auto kern = lp_wide(n_rows, n_cols) ? lp_slice_kernel<LP_WIDE> : lp_slice_kernel<LP_SLIM>;
  hipLaunchKernelGGL(kern, dim3((unsigned)(n_rows * slices)), dim3(LP_THREADS), 0, st, logits, n_cols,
                     slices, part, groups, (int64_t)n_groups);
  hipLaunchKernelGGL(lp_row_kernel, dim3((unsigned)n_rows), dim3(LP_THREADS), 0, st, logits, n_cols,
                     slices, part, groups, n_groups, ids, n_ids, id_lp, entropy, n_top, top_ids,
                     top_lp);
  return hip_check(hipGetLastError(), "log_probs");
}
