// Paged key-value cache of differential attention: what its kernels share, and the kernels that store new tokens.
//
// A sequence's token j lies in slot j % page_size of page page_table[b][j / page_size]; a page holds the rows of all heads.  Rows: K1, K2 of
// D, V of 2D 16-bit elements, 8 D bytes a token and head.  Nothing about a sequence is known on the host but the table's width, so lengths
// and pages are checked here: a length outside [0, slots] counts as the nearest bound, a page outside the pool is not touched, and
// both are reported through a status word of the cache's.
#pragma once
#include "sm100.cuh"

namespace da {

// A cache whose contents make no sense: what, sequence, where (the first report since diffattn_status last took one).  A word apart from g_status: a
// full cache is the caller's doing and nothing unusual, and must not stand in the way of a wait that gives up later, in whatever kernel.
__device__ int g_cache_status[3];
constexpr int kCacheBadLength = 1, kCacheBadPage = 2, kCacheFull = 3;

__device__ __noinline__ void cache_fault(int what, int b, int at) {
  if (atomicCAS(&g_cache_status[0], 0, what) == 0) {
    g_cache_status[1] = b;
    g_cache_status[2] = at;
  }
}

// All kernels of the cache are launched with the attribute for dependent launches, behind each other and behind whatever the caller put on the
// stream, and every thread waits for the grid ahead before it touches global memory: only the launch itself and the barriers' set-up overlap
// what comes before (about 1.5 us a call in a stream).  Loads are plain ones: the read-only path may keep what it read before the wait.
struct CacheArgs {
  int b, h;
  int page_size, max_pages, num_pages;
  int slots;                         // page_size * max_pages: what a sequence can hold
  uint32_t page_magic;               // ceil(2^32 / page_size); 0: pages of one slot
  const int* page_table;             // [b][max_pages], rows table_stride apart
  long long table_stride;
  int* lengths;                      // [b]
  int* next_position;                // [b] or null: tokens that the sequence has had, with those evicted
  int* counter;                      // one, 0 between calls: see cache_last_block
  int* positions;                    // [b][h][slots] or null: the position of the token in each slot
  float* weights;                    // [b][h][slots] or null: accumulated attention weights
  uint4* k1; uint4* k2; uint4* v;    // the pools; strides in 16-byte pieces
  long long k_page, k_head, k_slot;
  long long v_page, v_head, v_slot;
};

__device__ __forceinline__ int cache_length(const CacheArgs& c, int b) {
  const int n = c.lengths[b];
  if (n >= 0 && n <= c.slots) return n;
  cache_fault(kCacheBadLength, b, n);
  return n < 0 ? 0 : c.slots;
}
// slot / page_size: slot < 2^31 and page_magic - 2^32 / page_size < 1, so the product is at most one quotient too high
__device__ __forceinline__ int cache_page(const CacheArgs& c, int slot) {
  int p = c.page_magic ? int(__umulhi(uint32_t(slot), c.page_magic)) : slot;
  if ((long long)p * c.page_size > slot) --p;
  return p;
}
// the page behind entry `i` of sequence b's table, or -1
__device__ __forceinline__ int cache_page_load(const CacheArgs& c, int b, int i) { return c.page_table[b * c.table_stride + i]; }
__device__ __forceinline__ int cache_page_check(const CacheArgs& c, int b, int i, int id) {
  if (uint32_t(id) < uint32_t(c.num_pages)) return id;
  cache_fault(kCacheBadPage, b, i);
  return -1;
}
__device__ __forceinline__ int cache_page_id(const CacheArgs& c, int b, int i) { return cache_page_check(c, b, i, cache_page_load(c, b, i)); }

// The 16-byte piece `part` (of D / 2: K1, then K2, then V) of a cached row.
template <int D>
__device__ __forceinline__ uint4* cache_piece(const CacheArgs& c, int page, int head, int in_page, int part) {
  constexpr int KP = D / 8;
  if (part < 2 * KP) return (part < KP ? c.k1 : c.k2) + page * c.k_page + head * c.k_head + in_page * c.k_slot + (part & (KP - 1));
  return c.v + page * c.v_page + head * c.v_head + in_page * c.v_slot + (part - 2 * KP);
}

// The lengths change when every CTA has read them.  One warp of each takes a ticket once its CTA has (behind a barrier), and where it is the last
// one this returns true, to the whole warp: it changes them.  The counter is 0 again then.  Writing calls on a cache are ordered, so one counter does.
// A second kernel instead costs 2.7 us on the host and 1.5 on the GPU; where many CTAs come and go the ticket costs more than that (4096 of them, B4
// H16 N2048 D64: 30 us instead of 26), so large appends have the second kernel.
__device__ __forceinline__ bool cache_last_block(const CacheArgs& c) {
  int ticket = 0;
  if ((threadIdx.x & 31) == 0) {
    __threadfence();
    ticket = atomicAdd(c.counter, 1);
  }
  const bool last = __shfl_sync(0xffffffffu, ticket, 0) == int(gridDim.x * gridDim.y) - 1;
  if (last) {
    __threadfence();
    if ((threadIdx.x & 31) == 0) *c.counter = 0;
  }
  return last;
}

struct CacheAppendArgs {
  CacheArgs c;
  int t;                             // rows given per (sequence, head)
  int take_tickets;                  // the storing kernel moves the lengths on itself
  const int* counts;                 // [b] or null (all t): how many of them sequence b gets
  const uint4* k1; const uint4* k2; const uint4* v;
  long long k_b, k_h, k_t, v_b, v_h, v_t;      // in 16-byte pieces
};

__device__ __forceinline__ int append_count(const CacheAppendArgs& a, int b) {
  return a.counts ? min(max(a.counts[b], 0), a.t) : a.t;
}
__device__ __forceinline__ void append_advance(const CacheAppendArgs& a, int b) {
  const int len = cache_length(a.c, b), stored = min(append_count(a, b), a.c.slots - len);
  a.c.lengths[b] = len + stored;
  if (a.c.next_position) a.c.next_position[b] += stored;
}

// Where the rows of one block's round lie: found by one thread a row (two divisions' worth of arithmetic, a page, 64-bit products), read by
// the D / 2 threads that move its pieces.  With every thread finding its own address the kernels here were bound by that: 213 instructions a warp for
// 512 bytes, 27 us instead of 13 for 65536 rows of D = 64.
template <int ROWS>
struct RowPlaces {
  long long k[ROWS], v[ROWS];        // 16-byte pieces from the pools' bases; k -1: no row
};
// (`id`: what the page table holds for the slot; the caller has loaded it, so that two of them are under way together)
template <int ROWS>
__device__ __forceinline__ void place_row(const CacheArgs& c, RowPlaces<ROWS>& p, int row, int b, int head, int slot, int entry, int id) {
  const int page = cache_page_check(c, b, entry, id), in_page = slot - entry * c.page_size;
  p.k[row] = page < 0 ? -1 : page * c.k_page + head * c.k_head + in_page * c.k_slot;
  p.v[row] = page * c.v_page + head * c.v_head + in_page * c.v_slot;
}
// a thread's piece of a row (of D / 2: K1, K2, V): the pool's base with the piece's offset, and which of the two places counts
template <int D>
struct Piece {
  uint4* base;
  bool is_v;
  __device__ __forceinline__ Piece(const CacheArgs& c, int part) {
    is_v = part >= D / 4;
    base = is_v ? c.v + (part - D / 4) : (part < D / 8 ? c.k1 : c.k2) + (part & (D / 8 - 1));
  }
  template <int ROWS>
  __device__ __forceinline__ uint4* at(const RowPlaces<ROWS>& p, int row) const {
    return base + (is_v ? p.v[row] : p.k[row]);
  }
};

// Stores new rows behind each sequence's last one.  Bound by HBM: 8 D bytes in and out per row.  A thread moves 16-byte pieces, neighbours
// along a row, two rows under way together (four: B8 H16 N2048 D32 28.5 us instead of 25.5, eight 27.1); grid (rows, b * h).
constexpr int APPEND_THREADS = 256, APPEND_UNROLL = 2;

template <int D>
__global__ void __launch_bounds__(APPEND_THREADS) diffattn_cache_append_kernel(const CacheAppendArgs a) {
  constexpr int PARTS = D / 2, ROWS = APPEND_THREADS / PARTS, BLOCK = ROWS * APPEND_UNROLL;
  __shared__ RowPlaces<BLOCK> places;
  const CacheArgs& c = a.c;
  griddep_wait();
  griddep_launch();
  const int head = blockIdx.y % c.h, b = blockIdx.y / c.h;
  const int part = threadIdx.x % PARTS;
  const int first = blockIdx.x * BLOCK, row = threadIdx.x / PARTS;
  const int count = append_count(a, b);
  const uint4* src;
  long long step;
  if (part < D / 4) {
    src = (part < D / 8 ? a.k1 : a.k2) + b * a.k_b + head * a.k_h + (part & (D / 8 - 1));
    step = a.k_t;
  } else {
    src = a.v + b * a.v_b + head * a.v_h + (part - D / 4);
    step = a.v_t;
  }
  src += (first + row) * step;
  uint4 x[APPEND_UNROLL];
#pragma unroll
  for (int i = 0; i < APPEND_UNROLL; ++i)
    if (first + row + i * ROWS < count) x[i] = src[i * ROWS * step];
  if (threadIdx.x < BLOCK) {
    const int t = first + threadIdx.x, len = cache_length(c, b);
    places.k[threadIdx.x] = -1;
    if (t < count && t < c.slots - len) {
      const int entry = cache_page(c, len + t);
      place_row(c, places, threadIdx.x, b, head, len + t, entry, cache_page_load(c, b, entry));
      const long long at = (long long)blockIdx.y * c.slots + len + t;
      if (c.positions) c.positions[at] = c.next_position[b] + t;
      if (c.weights) c.weights[at] = 0.f;
    } else if (t < count) {
      cache_fault(kCacheFull, b, len);
    }
  }
  __syncthreads();
  if (a.take_tickets && threadIdx.x >= APPEND_THREADS - 32 && cache_last_block(c))
    for (int s = threadIdx.x & 31; s < c.b; s += 32) append_advance(a, s);
  const Piece<D> piece(c, part);
#pragma unroll
  for (int i = 0; i < APPEND_UNROLL; ++i)
    if (places.k[row + i * ROWS] >= 0) *piece.at(places, row + i * ROWS) = x[i];
}

__global__ void __launch_bounds__(APPEND_THREADS) diffattn_cache_advance_kernel(const CacheAppendArgs a) {
  griddep_wait();
  griddep_launch();
  const int b = blockIdx.x * APPEND_THREADS + threadIdx.x;
  if (b < a.c.b) append_advance(a, b);
}

__global__ void __launch_bounds__(APPEND_THREADS) diffattn_cache_reset_kernel(int* lengths, int* next_position, int n) {
  griddep_wait();
  griddep_launch();
  const int b = blockIdx.x * APPEND_THREADS + threadIdx.x;
  if (b >= n) return;
  lengths[b] = 0;
  if (next_position) next_position[b] = 0;
}

}  // namespace da
