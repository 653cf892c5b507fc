// Eviction: every sequence longer than `keep` is cut back to `keep` tokens, per head: the tokens of the last `recent` positions stay, then
// those with the largest accumulated weights (ties: the lowest slot); without weights the newest positions.
//
// Attention does not depend on the order of the slots, so nothing is shifted: a survivor in a slot behind `keep` moves into one of the holes
// that the others leave below it, the k-th survivor into the k-th hole.  Sources and destinations never overlap, every move is independent of
// the others, and a call that evicts a few tokens moves a few rows.
//
// Two kernels: the selection (a CTA per (sequence, head): 8 bytes per token read, the rest in shared memory) writes a list of moves, the
// second one carries them out, spread over all SMs whatever the number of heads is.
#pragma once
#include "cache.cuh"

namespace da {

struct EvictArgs {
  CacheArgs c;
  int keep, recent;
  int most;                          // moves that a (sequence, head) can have: min(keep, slots - keep)
  int* count;                        // [b * h] moves
  int2* moves;                       // [b * h][most] {from, to}
  int cached_keys;                   // the selection keeps all keys in shared memory
};

constexpr int SELECT_THREADS = 512, SELECT_WARPS = SELECT_THREADS / 32;
constexpr int SELECT_MOST_KEYS = 48 * 1024;      // that fit in shared memory

// Order of a slot: whole numbers, larger = rather kept.  NaN counts as larger than every number, -0 as 0.
__device__ __forceinline__ uint32_t evict_key(const EvictArgs& a, long long at, int newest_from) {
  const int pos = a.c.positions[at];
  if (pos >= newest_from) return 0xffffffffu;
  if (!a.c.weights) return uint32_t(max(pos, 0));
  const float w = a.c.weights[at];
  const uint32_t u = w != w ? 0x7fc00000u : __float_as_uint(w + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// sum of `x` over the threads before this one; `total`: over all.  `buf`: SELECT_WARPS ints, free again after the call's second barrier
__device__ __forceinline__ int block_before(int x, int* buf, int& total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int incl = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  if (lane == 31) buf[warp] = incl;
  __syncthreads();
  int s = lane < SELECT_WARPS ? buf[lane] : 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += y;
  }
  total = __shfl_sync(0xffffffffu, s, 31);
  const int before = __shfl_sync(0xffffffffu, s, max(warp - 1, 0));
  __syncthreads();
  return (warp ? before : 0) + incl - x;
}

__global__ void __launch_bounds__(SELECT_THREADS) diffattn_cache_select_kernel(const EvictArgs a) {
  extern __shared__ uint32_t keys[];
  __shared__ int hist[256], buf[SELECT_WARPS], found[2];
  const CacheArgs& c = a.c;
  griddep_launch();
  const int bh = blockIdx.x, b = bh / c.h, tid = threadIdx.x;
  const int len = cache_length(c, b);
  if (len <= a.keep) {
    if (tid == 0) a.count[bh] = 0;
    return;
  }
  const long long base = (long long)bh * c.slots;
  const int newest_from = c.next_position[b] - a.recent;
  if (a.cached_keys)
    for (int i = tid; i < len; i += SELECT_THREADS) keys[i] = evict_key(a, base + i, newest_from);
  auto key = [&](int i) { return a.cached_keys ? keys[i] : evict_key(a, base + i, newest_from); };      // (each thread reads its own)
  // the keep-th largest key, eight bits at a time: how many keys that agree with the bits so far have each next digit
  uint32_t prefix = 0;
  int want = a.keep;                 // of the keys that agree with `prefix`, this many stay
#pragma unroll 1
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += SELECT_THREADS) hist[i] = 0;
    __syncthreads();
    for (int i = tid; i < len; i += SELECT_THREADS) {
      const uint32_t k = key(i);
      if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255], 1);
    }
    __syncthreads();
    // digits from the largest down: thread t has digit 255 - t
    const int mine = tid < 256 ? hist[255 - tid] : 0;
    int total;
    const int above = block_before(mine, buf, total);
    if (mine && above < want && above + mine >= want) {
      found[0] = 255 - tid;
      found[1] = above;
    }
    __syncthreads();
    prefix |= uint32_t(found[0]) << shift;
    want -= found[1];
  }
  // keys above `prefix` stay, and the first `want` of those equal to it; survivors behind `keep` and holes below it in slot order
  int equal = 0, survivors = 0, holes = 0;
  for (int i0 = 0; i0 < len; i0 += SELECT_THREADS) {
    const int i = i0 + tid;
    const uint32_t k = i < len ? key(i) : 0;
    const bool eq = i < len && k == prefix;
    int total;
    const int rank = equal + block_before(eq, buf, total);
    equal += total;
    const bool kept = i < len && (k > prefix || (eq && rank < want));
    const bool moves = kept && i >= a.keep, hole = i < a.keep && !kept;
    const int at = block_before((moves ? 1 : 0) | (hole ? 0x10000 : 0), buf, total);      // both counts at once: at most SELECT_THREADS each
    int2* list = a.moves + (long long)bh * a.most;
    if (moves) list[survivors + (at & 0xffff)].x = i;
    if (hole) list[holes + (at >> 16)].y = i;
    survivors += total & 0xffff;
    holes += total >> 16;
  }
  if (tid == 0) a.count[bh] = survivors;
}

constexpr int MOVE_THREADS = 256, MOVE_UNROLL = 2;

template <int D>
__global__ void __launch_bounds__(MOVE_THREADS) diffattn_cache_move_kernel(const EvictArgs a) {
  constexpr int PARTS = D / 2, ROWS = MOVE_THREADS / PARTS;
  const CacheArgs& c = a.c;
  griddep_wait();
  const int part = threadIdx.x % PARTS;
  for (int bh = blockIdx.y; bh < c.b * c.h; bh += gridDim.y) {
    const int b = bh / c.h, head = bh - b * c.h, count = a.count[bh];
    const int2* list = a.moves + (long long)bh * a.most;
    for (int r0 = blockIdx.x * (ROWS * MOVE_UNROLL) + threadIdx.x / PARTS; r0 < count; r0 += gridDim.x * (ROWS * MOVE_UNROLL)) {
      uint4 x[MOVE_UNROLL];
      int2 mv[MOVE_UNROLL];
      bool ok[MOVE_UNROLL];
#pragma unroll
      for (int i = 0; i < MOVE_UNROLL; ++i) {
        const int r = r0 + i * ROWS;
        ok[i] = r < count;
        if (!ok[i]) continue;
        mv[i] = list[r];
        const int p = cache_page(c, mv[i].x), page = cache_page_id(c, b, p);
        ok[i] = page >= 0;
        if (ok[i]) x[i] = *cache_piece<D>(c, page, head, mv[i].x - p * c.page_size, part);
      }
#pragma unroll
      for (int i = 0; i < MOVE_UNROLL; ++i) {
        if (!ok[i]) continue;
        const int p = cache_page(c, mv[i].y), page = cache_page_id(c, b, p);
        if (page >= 0) *cache_piece<D>(c, page, head, mv[i].y - p * c.page_size, part) = x[i];
        if (part == 0) {
          const long long base = (long long)bh * c.slots;
          c.positions[base + mv[i].y] = c.positions[base + mv[i].x];
          if (c.weights) c.weights[base + mv[i].y] = c.weights[base + mv[i].x];
        }
      }
    }
    if (blockIdx.x == 0 && head == 0 && threadIdx.x == 0 && c.lengths[b] > a.keep) c.lengths[b] = a.keep;
  }
}

}  // namespace da
