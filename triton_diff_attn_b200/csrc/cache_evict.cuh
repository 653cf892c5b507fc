// Eviction: every sequence longer than `keep` is cut back to `keep` tokens, per head: the tokens of the last `recent` positions stay, then
// those with the largest accumulated weights (ties: the lowest slot); without weights the newest positions.
//
// Attention does not depend on the order of the slots, so nothing is shifted: a survivor in a slot behind `keep` moves into one of the holes
// that the others leave below it, the k-th survivor into the k-th hole.  Sources and destinations never overlap, every move is independent of
// the others, and a call that evicts a few tokens moves a few rows.
//
// The selection takes a CTA per (sequence, head): 8 bytes per token read, the rest in shared memory.  Where its moves are few, or the CTAs enough
// to fill the GPU, it carries them out too; else it writes them down for a second kernel that spreads them over all SMs.
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

// (256 threads: the chain of loads and barriers counts, not the arithmetic; 512 select no faster, and fewer CTAs are resident: a step of B32 H16 N2048
// 116 us with 512, 110 with 256)
constexpr int SELECT_THREADS = 256, SELECT_WARPS = SELECT_THREADS / 32;
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

// sums of x and y over the threads before this one, in place; `all`: over all of them.  `buf`: SELECT_WARPS places, free again after the next barrier
__device__ __forceinline__ void block_before(int& x, int& y, int2* buf, int2& all) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, x0 = x, y0 = y;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, x, o), v = __shfl_up_sync(0xffffffffu, y, o);
    if (lane >= o) { x += u; y += v; }
  }
  if (lane == 31) buf[warp] = make_int2(x, y);
  __syncthreads();
  x -= x0;
  y -= y0;
  all = make_int2(0, 0);
#pragma unroll
  for (int w = 0; w < SELECT_WARPS; ++w) {
    const int2 v = buf[w];
    if (w < warp) { x += v.x; y += v.y; }
    all.x += v.x;
    all.y += v.y;
  }
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
__global__ void __launch_bounds__(SELECT_THREADS) diffattn_cache_select_kernel(const EvictArgs a) {
  extern __shared__ uint32_t keys[];
  __shared__ int hist[4][256];
  __shared__ int2 buf[2][SELECT_WARPS];
  __shared__ int2 near_list[SELECT_LIST];
  __shared__ MovePlaces<D, SELECT_THREADS> places;
  const CacheArgs& c = a.c;
  griddep_wait();
  griddep_launch();
  const int bh = blockIdx.x, b = bh / c.h, tid = threadIdx.x, lane = tid & 31;
  const int newest_from = c.next_position[b] - a.recent;
  const int len = cache_length(c, b);
  if (a.moves_at_once) {
    __syncthreads();
    if (tid >= SELECT_THREADS - 32 && cache_last_block(c))
      for (int s = lane; s < c.b; s += 32)
        if (c.lengths[s] > a.keep) c.lengths[s] = a.keep;
  }
  if (len <= a.keep) {
    if (tid == 0 && !a.moves_at_once) a.count[bh] = 0;
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
  // Keys above `prefix` stay, and of those that agree with it the first `want`.  Survivors behind `keep` and holes below it in slot order: a thread
  // has a run of at most 31 neighbours (an odd number, so that a warp's reads fall into different banks) and keeps in a mask which of them
  // are one or the other.
  const bool ties = alike != want;   // (then all 32 bits of `prefix` are known)
  int2* list = a.most <= SELECT_LIST ? near_list : a.moves + (long long)bh * a.most;
  int equal = 0, holes = 0, moves = 0;           // before the current round
  for (int c0 = 0; c0 < len; c0 += 31 * SELECT_THREADS) {
    const int left = min(len - c0, 31 * SELECT_THREADS), run = min((left + SELECT_THREADS - 1) / SELECT_THREADS | 1, 31);
    const int i0 = min(c0 + tid * run, c0 + left), i1 = min(i0 + run, c0 + left);
    uint32_t same = 0, kept = 0;
    for (int i = i0; i < i1; ++i) {
      const uint32_t k = key(i);
      kept |= uint32_t(k >= prefix) << (i - i0);
      same |= uint32_t(k == prefix) << (i - i0);
    }
    int2 all;
    if (ties) {
      int rank = __popc(same), none = 0;
      block_before(rank, none, buf[0], all);
      rank += equal;
      for (uint32_t m = same; m; m &= m - 1)      // those behind the first `want` go
        if (rank++ >= want) kept &= ~(m & -m);
      equal += all.x;
    }
    const int low = min(max(a.keep - i0, 0), i1 - i0);      // slots of the run below `keep`
    const uint32_t mask_low = low >= 32 ? 0xffffffffu : (1u << low) - 1;
    uint32_t hole = ~kept & mask_low, moved = kept & ~mask_low;
    int x = __popc(hole), y = __popc(moved);
    block_before(x, y, buf[1], all);
    x += holes;
    y += moves;
    // (as many survivors as holes, and no more than `most`, as long as nobody writes positions or weights meanwhile)
    for (; hole && x < a.most; hole &= hole - 1) list[x++].y = i0 + __ffs(hole) - 1;
    for (; moved && y < a.most; moved &= moved - 1) list[y++].x = i0 + __ffs(moved) - 1;
    holes += all.x;
    moves += all.y;
    if (c0 + 31 * SELECT_THREADS < len) __syncthreads();      // (the next round writes buf)
  }
  int total = min(min(holes, moves), a.most);
  __syncthreads();
  if (a.moves_at_once) {
    move_rows<D, SELECT_THREADS>(a, places, bh, list, total, 0, 1);
    return;
  }
  if (list == near_list)
    for (int i = tid; i < total; i += SELECT_THREADS) a.moves[(long long)bh * a.most + i] = list[i];
  if (tid == 0) a.count[bh] = total;
}

constexpr int MOVE_THREADS = 256;

// Grid (wide, b * h): the moves that the selection wrote down, and the lengths.
template <int D>
__global__ void __launch_bounds__(MOVE_THREADS) diffattn_cache_move_kernel(const EvictArgs a) {
  __shared__ MovePlaces<D, MOVE_THREADS> places;
  griddep_wait();
  griddep_launch();
  const int bh = blockIdx.y, b = bh / a.c.h;
  move_rows<D, MOVE_THREADS>(a, places, bh, a.moves + (long long)bh * a.most, a.count[bh], blockIdx.x, gridDim.x);
  if (blockIdx.x == 0 && bh == b * a.c.h && threadIdx.x == 0 && a.c.lengths[b] > a.keep) a.c.lengths[b] = a.keep;
}

}  // namespace da
