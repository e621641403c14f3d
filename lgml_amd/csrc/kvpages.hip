// Copies of blocks within the pool tensors of every layer at once (gfx950).
#include <stdlib.h>
#include <string.h>

#include <memory>

#include "kvq4.h"
#include "kvq8.h"

namespace lgmlh {

// A copy {src, dst, n}: the first n cells of block dst become those of block src (src
// -1: zeros) in every tensor (K at even places, V at odd ones). A thread takes a 16-byte
// unit of one block of one tensor. A unit holds one cell (K's values), eight cells of 2
// bytes (V of f16, scales) or twice eight cells of 1 byte (V of Q8_0 and Q4_0, cells 8 q ..
// and 32 + 8 q ..): one with cells of both sides of n is blended with the target's. So
// are the others of V's lines then, each of which has such cells: lines written in part
// are read and written again behind the caches. Nothing is read again here, so the
// stores pass the caches by. 64 blocks of 32 layers of K and V of 128 KB, 1.07 GB: 171 us
// (4 units a thread 203, cached stores 175); 32 copies of 37 cells on average from 4
// blocks 78 us (written in pieces 102). Over Q8_0 and Q4_0 such 32 copies take 45 and 22 us, whole
// blocks 50 and 22 (f16 88).
constexpr int PAGE_THREADS = 256;

// The cells of a unit at byte `at` of a tile: the first of its one or eight (W cells of
// 16 / W bytes; of W = 16 the second eight are 32 cells on).
struct Unit {
  int first, width;
};
template <int TYPE>
__device__ __forceinline__ Unit unit_at(int at, int is_v, int D) {
  const int values = TYPE == LGMLH_F16 ? 128 * D : TYPE == LGMLH_Q8_0 ? 64 * D : 32 * D;
  if (at >= values) return {(at - values) % 128 / 16 * 8, 8};  // scales [D / 32][64 cells]
  if (TYPE == LGMLH_F16) return is_v ? Unit{at % 128 / 16 * 8, 8} : Unit{at / (2 * D), 1};
  if (is_v) return {at % 64 / 16 * 8, 16};
  return {TYPE == LGMLH_Q4_0 && D == 64 ? at / 32 : at / 64 % 64, 1};
}

template <int TYPE>
__global__ void __launch_bounds__(PAGE_THREADS)
kv_copy_blocks_kernel(void *const *__restrict__ pools, int32_t n_blocks, int tile, int Hkv, int D,
                      const int32_t *__restrict__ copies, uint32_t slices) {
  const uint32_t i = blockIdx.x / slices, s = blockIdx.x % slices;
  const int p = blockIdx.y, is_v = p & 1;
  const int32_t src = copies[3 * (int64_t)i], dst = copies[3 * (int64_t)i + 1], n = copies[3 * (int64_t)i + 2];
  if (src < -1 || src >= n_blocks || dst < 0 || dst >= n_blocks || src == dst || n <= 0) return;
  const int64_t bytes = (int64_t)tile * Hkv;
  uint8_t *pool = (uint8_t *)pools[p];
  const uint8_t *from = pool + src * bytes;
  uint8_t *to = pool + dst * bytes;
  const int64_t o = 16 * ((int64_t)s * PAGE_THREADS + threadIdx.x);
  if (o >= bytes) return;
  const bool blend = n < KV_BLOCK && is_v;
  Unit u = {0, 1};
  bool all = true;
  if (n < KV_BLOCK) {
    u = unit_at<TYPE>((int)(o % tile), is_v, D);
    all = (u.width == 1 ? u.first : u.first + (u.width == 16 ? 39 : 7)) < n;
  }
  if (u.first >= n && !blend) return;
  u32x4 v = {0, 0, 0, 0};
  if (src >= 0 && u.first < n) v = *(const u32x4 *)(from + o);
  if (!all) {
    const u32x4 was = *(const u32x4 *)(to + o);
#pragma unroll
    for (int w = 0; w < 4; w++) {
      uint32_t keep = 0;  // the bits of cells from n on
      if (u.width == 8) {
#pragma unroll
        for (int e = 0; e < 2; e++)
          if (u.first + 2 * w + e >= n) keep |= 0xffffu << 16 * e;
      } else {
#pragma unroll
        for (int x = 0; x < 4; x++) {  // the byte's cell
          const int e = 4 * w + x, in = TYPE == LGMLH_Q4_0 ? (e & 4) | (e & 1) << 1 | (e >> 1 & 1) : e & 7;
          if (u.first + 32 * (e >> 3) + in >= n) keep |= 0xffu << 8 * x;
        }
      }
      v[w] = (v[w] & ~keep) | (was[w] & keep);
    }
  }
  __builtin_nontemporal_store(v, (u32x4 *)(to + o));
}

// Ranges of copies, no target twice, no target that is a source: a table of blocks
// with what each is, twice as long as the blocks named.
static int check_copies(const int32_t *h, int64_t n, int64_t n_blocks) {
  constexpr int NEAR = 1024;
  constexpr uint8_t SRC = 1, DST = 2;
  struct Slot {
    int32_t block;  // + 1; 0: free
    uint32_t is;
  } near_[NEAR];
  for (int64_t i = 0; i < n; i++) {
    const int32_t src = h[3 * i], dst = h[3 * i + 1], cells = h[3 * i + 2];
    if (src < -1 || src >= n_blocks || dst < 0 || dst >= n_blocks) {
      set_error("kv_copy_blocks: block %d to %d out of range [0, %lld)", src, dst, (long long)n_blocks);
      return LGMLH_ERANGE;
    }
    if (cells < 0 || cells > KV_BLOCK) {
      set_error("kv_copy_blocks: %d cells of a block", cells);
      return LGMLH_EINVAL;
    }
  }
  int bits = 4;
  while ((int64_t)1 << bits < 4 * n) bits++;
  const uint64_t slots = (uint64_t)1 << bits;
  std::unique_ptr<Slot, void (*)(void *)> far(nullptr, free);
  Slot *table = near_;
  if (slots > NEAR) {
    far.reset((Slot *)calloc(slots, sizeof(Slot)));
    if (!far) {
      set_error("kv_copy_blocks: no host memory to check %lld copies", (long long)n);
      return LGMLH_ENOMEM;
    }
    table = far.get();
  } else {
    memset(near_, 0, slots * sizeof(Slot));
  }
  for (int64_t i = 0; i < 2 * n; i++) {
    const int32_t block = h[3 * (i / 2) + i % 2];
    if (block < 0) continue;
    uint64_t at = (uint64_t)block * 0x9e3779b97f4a7c15ull >> (64 - bits);
    while (table[at].block && table[at].block != block + 1) at = (at + 1) & (slots - 1);
    Slot &t = table[at];
    const uint32_t is = i % 2 ? DST : SRC;
    if (t.is & DST || (t.is && is == DST)) {
      set_error("kv_copy_blocks: block %d is a target and %s", block, t.is & is ? "one again" : "a source");
      return LGMLH_EINVAL;
    }
    t.block = block + 1;
    t.is |= is;
  }
  return LGMLH_OK;
}

}  // namespace lgmlh

using namespace lgmlh;

extern "C" int lgmlh_kv_copy_blocks(int type, void *const *pools, int n_pools, int64_t n_cells,
                                    int n_head_kv, int head_dim, const int32_t *copies,
                                    const int32_t *h_copies, int64_t n, void *stream) {
  const bool quant = type == LGMLH_Q8_0 || type == LGMLH_Q4_0;
  if ((!quant && type != LGMLH_F16) || !pools || !copies || !h_copies || n_pools <= 0 || n_pools > 65535 ||
      n_pools % 2 || n_cells <= 0 || n_cells % KV_BLOCK || n_cells / KV_BLOCK > INT32_MAX || n_head_kv <= 0 ||
      n_head_kv > 65535 || n < 0 ||
      (quant ? head_dim != 64 && head_dim != 128 && head_dim != 256
             : head_dim <= 0 || head_dim % 8 || head_dim > 1024)) {
    set_error("kv_copy_blocks: bad arguments (K and V tensors in turn, of f16, Q8_0 or Q4_0)");
    return LGMLH_EINVAL;
  }
  const int tile = (type == LGMLH_Q8_0 ? 68 : type == LGMLH_Q4_0 ? 36 : 128) * head_dim;
  const int64_t slice = 16 * PAGE_THREADS, slices = ((int64_t)tile * n_head_kv + slice - 1) / slice;
  if (n > ((int64_t)1 << 24) / slices - 1) {  // fewer than 2^32 threads a launch
    set_error("kv_copy_blocks: %lld copies in one call", (long long)n);
    return LGMLH_EINVAL;
  }
  LGMLH_TRY(check_copies(h_copies, n, n_cells / KV_BLOCK));
  if (n == 0) return LGMLH_OK;
  const auto kern = type == LGMLH_Q8_0   ? kv_copy_blocks_kernel<LGMLH_Q8_0>
                    : type == LGMLH_Q4_0 ? kv_copy_blocks_kernel<LGMLH_Q4_0>
                                         : kv_copy_blocks_kernel<LGMLH_F16>;
  hipLaunchKernelGGL(kern, dim3((unsigned)(n * slices), (unsigned)n_pools), dim3(PAGE_THREADS), 0,
                     as_stream(stream), pools, (int32_t)(n_cells / KV_BLOCK), tile, n_head_kv, head_dim, copies,
                     (uint32_t)slices);
  return hip_check(hipGetLastError(), "kv_copy_blocks");
}
