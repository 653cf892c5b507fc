// Eviction: every sequence longer than `keep` is cut back to `keep` tokens, per head: the tokens of the last `recent` positions stay, then
// those with the largest accumulated weights (ties: the lowest slot); without weights the newest positions.
//
// Attention does not depend on the order of the slots, so nothing is shifted: a survivor in a slot behind `keep` moves into one of the holes
// that the others leave below it, the k-th survivor into the k-th hole.  Sources and destinations never overlap, every move is independent of
// the others, and a call that evicts a few tokens moves a few rows.
//
// The selection takes a CTA per (sequence, head): 8 bytes per token read, the rest in shared memory.  Where its moves are few, or the CTAs enough
// to fill the GPU, it carries them out too; else it writes them down for a second kernel that spreads them over all SMs.  Either way the
// lengths change in a kernel behind it, when every head has read them.
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
  int moves_at_once;                 // the selection carries its moves out
};

constexpr int SELECT_THREADS = 512, SELECT_WARPS = SELECT_THREADS / 32;
constexpr int SELECT_MOST_KEYS = 48 * 1024;      // that fit in shared memory
constexpr int SELECT_AHEAD = 8;                  // slots whose loads a thread has under way together

// Order of a slot: whole numbers, larger = rather kept.  NaN counts as larger than every number, -0 as 0.
__device__ __forceinline__ uint32_t evict_key(const EvictArgs& a, int pos, float w, int newest_from) {
  if (pos >= newest_from) return 0xffffffffu;
  if (!a.c.weights) return uint32_t(max(pos, 0));
  const uint32_t u = w != w ? 0x7fc00000u : __float_as_uint(w + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint32_t evict_key(const EvictArgs& a, long long at, int newest_from) {
  return evict_key(a, a.c.positions[at], a.c.weights ? a.c.weights[at] : 0.f, newest_from);
}

// sums of x and y over the threads before this one, in place; `total`: of y over all.  `buf`: SELECT_WARPS places of this call's own
__device__ __forceinline__ void block_before(int& x, int& y, int2* buf, int& total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, x0 = x, y0 = y;
  auto scan = [&](int& v) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
  };
  scan(x);
  scan(y);
  if (lane == 31) buf[warp] = make_int2(x, y);
  __syncthreads();
  const int2 all = lane < SELECT_WARPS ? buf[lane] : make_int2(0, 0);
  int sx = all.x, sy = all.y;
  scan(sx);
  scan(sy);
  total = __shfl_sync(0xffffffffu, sy, 31);
  sx = __shfl_sync(0xffffffffu, sx - all.x, warp);
  sy = __shfl_sync(0xffffffffu, sy - all.y, warp);
  x += sx - x0;
  y += sy - y0;
}

// A list of moves, by one block of `blocks`; all its threads call it.  Thread: one 16-byte piece of a row, UNROLL rows under way together.
constexpr int MOVE_UNROLL = 4;
template <int D, int THREADS>
struct MovePlaces {
  static constexpr int PARTS = D / 2, ROWS = THREADS / PARTS, BLOCK = ROWS * MOVE_UNROLL;
  RowPlaces<BLOCK> from, to;
};
template <int D, int THREADS>
__device__ __forceinline__ void move_rows(const EvictArgs& a, MovePlaces<D, THREADS>& places, int bh, const int2* list, int count, int block, int blocks) {
  using P = MovePlaces<D, THREADS>;
  const CacheArgs& c = a.c;
  const int b = bh / c.h, head = bh - b * c.h, row = threadIdx.x / P::PARTS;
  const Piece<D> piece(c, threadIdx.x % P::PARTS);
  for (int first = block * P::BLOCK; first < count; first += blocks * P::BLOCK) {
    if (threadIdx.x < P::BLOCK) {
      places.from.k[threadIdx.x] = -1;
      if (first + threadIdx.x < count) {
        const int2 mv = list[first + threadIdx.x];
        const long long base = (long long)bh * c.slots;
        const int pos = c.positions[base + mv.x];
        const float w = c.weights ? c.weights[base + mv.x] : 0.f;
        const int ef = cache_page(c, mv.x), et = cache_page(c, mv.y);
        const int idf = cache_page_load(c, b, ef), idt = cache_page_load(c, b, et);
        place_row(c, places.from, threadIdx.x, b, head, mv.x, ef, idf);
        place_row(c, places.to, threadIdx.x, b, head, mv.y, et, idt);
        if (places.to.k[threadIdx.x] < 0) places.from.k[threadIdx.x] = -1;
        c.positions[base + mv.y] = pos;
        if (c.weights) c.weights[base + mv.y] = w;
      }
    }
    __syncthreads();
    uint4 x[MOVE_UNROLL];
#pragma unroll
    for (int i = 0; i < MOVE_UNROLL; ++i)
      if (places.from.k[row + i * P::ROWS] >= 0) x[i] = *piece.at(places.from, row + i * P::ROWS);
#pragma unroll
    for (int i = 0; i < MOVE_UNROLL; ++i)
      if (places.from.k[row + i * P::ROWS] >= 0) *piece.at(places.to, row + i * P::ROWS) = x[i];
    __syncthreads();
  }
}

constexpr int SELECT_LIST = 512;                 // moves that the selection keeps in shared memory

template <int D>
__global__ void __launch_bounds__(SELECT_THREADS, 4) diffattn_cache_select_kernel(const EvictArgs a) {
  extern __shared__ uint32_t keys[];
  __shared__ int hist[4][256];
  __shared__ int2 buf[2][SELECT_WARPS];
  __shared__ int2 near_list[SELECT_LIST];
  __shared__ MovePlaces<D, SELECT_THREADS> places;
  const CacheArgs& c = a.c;
  griddep_launch();
  const int bh = blockIdx.x, b = bh / c.h, tid = threadIdx.x, lane = tid & 31;
  const int newest_from = c.next_position[b] - a.recent;
  const int len = cache_length(c, b);
  if (len <= a.keep) {
    if (tid == 0) a.count[bh] = 0;
    return;
  }
  for (int i = tid; i < 4 * 256; i += SELECT_THREADS) hist[0][i] = 0;
  __syncthreads();
  const long long base = (long long)bh * c.slots;
  // the keep-th largest key, eight bits at a time: how many keys that agree with the bits so far have each next digit
  auto key = [&](int i) { return a.cached_keys ? keys[i] : evict_key(a, base + i, newest_from); };
  for (int i0 = tid; i0 < len; i0 += SELECT_THREADS * SELECT_AHEAD) {
    int pos[SELECT_AHEAD];
    float w[SELECT_AHEAD];
#pragma unroll
    for (int x = 0; x < SELECT_AHEAD; ++x) {
      const int i = min(i0 + x * SELECT_THREADS, len - 1);
      pos[x] = c.positions[base + i];
      w[x] = c.weights ? c.weights[base + i] : 0.f;
    }
#pragma unroll
    for (int x = 0; x < SELECT_AHEAD; ++x) {
      const int i = i0 + x * SELECT_THREADS;
      if (i >= len) break;
      const uint32_t k = evict_key(a, pos[x], w[x], newest_from);
      if (a.cached_keys) keys[i] = k;
      atomicAdd(&hist[0][k >> 24], 1);
    }
  }
  uint32_t prefix = 0;
  int want = a.keep, alike = 0;      // of the `alike` keys that agree with `prefix`, `want` stay
#pragma unroll 1
  for (int digit = 0; digit < 4; ++digit) {
    const int shift = 24 - 8 * digit;
    if (digit > 0) {
      for (int i = tid; i < len; i += SELECT_THREADS) {
        const uint32_t k = key(i);
        if (k >> (shift + 8) == prefix >> (shift + 8)) atomicAdd(&hist[digit][(k >> shift) & 255], 1);
      }
    }
    __syncthreads();
    // every warp by itself: lane l has digits 255 - 8 l down to 248 - 8 l
    int n[8], sum = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) sum += n[k] = hist[digit][255 - 8 * lane - k];
    int above = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, above, o);
      if (lane >= o) above += y;
    }
    const int owner = __ffs(__ballot_sync(0xffffffffu, above >= want)) - 1;      // the lane whose digits hold the want-th key
    above -= sum;
    int d = 0, left = 0, size = 0;
    bool found = false;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (!found && above + n[k] >= want) {
        found = true;
        d = 255 - 8 * lane - k; left = want - above; size = n[k];
      }
      above += n[k];
    }
    prefix |= uint32_t(__shfl_sync(0xffffffffu, d, owner)) << shift;
    want = __shfl_sync(0xffffffffu, left, owner);
    alike = __shfl_sync(0xffffffffu, size, owner);
    if (alike == want) break;        // all of them stay: whatever their lower bits are
  }
  // Keys above `prefix` stay, and of those that agree with it the first `want`.  Survivors behind `keep` and holes below it in slot order: a
  // thread has a run of slots (an odd number, so that a warp's reads fall into different banks)
  const int run = ((len + SELECT_THREADS - 1) / SELECT_THREADS) | 1;
  const int i0 = min(tid * run, len), i1 = min(i0 + run, len);
  int rank = 0, total;
  if (alike != want) {               // (all 32 bits of `prefix` are known)
    int none = 0;
    for (int i = i0; i < i1; ++i) rank += key(i) == prefix;
    block_before(rank, none, buf[0], total);
  }
  auto stays = [&](uint32_t k, int& r) {
    if (alike == want) return k >= prefix;
    if (k != prefix) return k > prefix;
    return r++ < want;
  };
  int moves = 0, holes = 0, r = rank;
  for (int i = i0; i < i1; ++i) {
    const bool kept = stays(key(i), r);
    moves += kept && i >= a.keep;
    holes += !kept && i < a.keep;
  }
  int2* list = a.most <= SELECT_LIST ? near_list : a.moves + (long long)bh * a.most;
  block_before(holes, moves, buf[1], total);
  int at = moves, to = holes;
  r = rank;
  for (int i = i0; i < i1; ++i) {
    const bool kept = stays(key(i), r);
    if (kept && i >= a.keep) list[at++].x = i;
    if (!kept && i < a.keep) list[to++].y = i;
  }
  __syncthreads();
  if (a.moves_at_once) {
    move_rows<D, SELECT_THREADS>(a, places, bh, list, total, 0, 1);
    total = 0;
  } else if (list == near_list) {
    for (int i = tid; i < total; i += SELECT_THREADS) a.moves[(long long)bh * a.most + i] = list[i];
  }
  if (tid == 0) a.count[bh] = total;
}

constexpr int MOVE_THREADS = 256;

// Grid (wide, b * h): the moves that the selection wrote down.
template <int D>
__global__ void __launch_bounds__(MOVE_THREADS) diffattn_cache_move_kernel(const EvictArgs a) {
  __shared__ MovePlaces<D, MOVE_THREADS> places;
  griddep_wait();
  const int bh = blockIdx.y, b = bh / a.c.h;
  move_rows<D, MOVE_THREADS>(a, places, bh, a.moves + (long long)bh * a.most, a.count[bh], blockIdx.x, gridDim.x);
  if (blockIdx.x == 0 && bh == b * a.c.h && threadIdx.x == 0 && a.c.lengths[b] > a.keep) a.c.lengths[b] = a.keep;
}

// The lengths alone, where the selection has moved everything.
__global__ void __launch_bounds__(MOVE_THREADS) diffattn_cache_shorten_kernel(const EvictArgs a) {
  griddep_wait();
  const int b = blockIdx.x * MOVE_THREADS + threadIdx.x;
  if (b < a.c.b && a.c.lengths[b] > a.keep) a.c.lengths[b] = a.keep;
}

}  // namespace da
