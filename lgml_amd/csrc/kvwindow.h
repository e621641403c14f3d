// The cells of a workgroup's tokens in the quantised KV pools, and the checks of
// cells that a call writes.
#pragma once

#include "common.h"

namespace lgmlh {

constexpr int CELL_GROUP = 8, CELL_HALO = 7;
constexpr int64_t CELLS_MAX = (int64_t)1 << 36;  // a block's number has 31 bits
// Heads of cells in one call, and its workgroups of 256: a launch has fewer than 2^32
// threads. (CELL_ROWS of 32 a workgroup are as many; a last one in part for each head may
// be one too many.)
constexpr int64_t CELL_ROWS = int64_t(1) << 29, CELL_GROUPS = int64_t(1) << 24;
inline int check_groups(int64_t groups, const char *what) {
  if (groups < CELL_GROUPS) return LGMLH_OK;
  set_error("%s: %lld workgroups in one launch", what, (long long)groups);
  return LGMLH_EINVAL;
}

// Range and distinctness of cells that a call writes (kvq8.hip).
int check_write_cells(const int64_t *h, int64_t n, int64_t n_cells, const char *what);

// W consecutive tokens from j0 on, and the whole groups among them: 8 tokens whose
// cells are 8 in a row from a multiple of 8 on. A group belongs to the window that
// has its first token, up to 7 of it lie past the window's own.
template <int W>
struct CellWindow {
  int64_t cells[W + 2 * CELL_HALO];  // of tokens j0 - 7 .. j0 + W + 6; -1: none
  int lead[W / CELL_GROUP];            // first tokens of the whole groups, 0 .. W - 1
  int lone[W];                         // tokens in no whole group
  int n_lead, n_lone;
  __device__ __forceinline__ int64_t cell(int t) const { return cells[t + CELL_HALO]; }
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
    if (tid < W + 2 * CELL_HALO) {
      const int64_t j = j0 + tid - CELL_HALO, c = j >= 0 && j < n ? src[j] : -1;
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

}  // namespace lgmlh
