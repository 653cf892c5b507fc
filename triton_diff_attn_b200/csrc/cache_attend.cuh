// Differential attention of one new token per (sequence, head) over a paged cache.
//
//   s_b[j] = q_b . k_b[j] / sqrt(D),  P_b = softmax(s_b),  A = P_1 V - lambda P_2 V,  y = A * norm * gain;  w[j] += |P_1[j] - lambda P_2[j]|
//
// Bound by HBM: every cached row (8 D bytes) is read once for 12 D flops.  A row meets one query only, so the 128-row tiles of tcgen05 would be
// 1/128 full; the arithmetic goes through mma.sync with the cached rows as the wide operand, not for its rate but for the instructions that it
// saves: 16 ldmatrix and 16 mma per 16 tokens at D = 64 where unpacking, fused multiply-adds and sums over lanes took 850
// instructions and bound the kernel (4.2 TB/s at B8 H8 N8192 D128, issue slots 39 % busy with two warps a scheduler).
//
// Split: the tiles of all (sequence, head)s form one line, and every WARP takes an equal, contiguous stretch of it.  Whatever the lengths
// are, all SMs read the same number of bytes, and nobody waits for anybody: a warp loads its own tiles (TMA, a ring of its own), keeps
// its own running maximum, sum and accumulators, and where its stretch leaves a (sequence, head) it writes them down as one piece.  A second
// kernel joins the pieces of a (sequence, head) (exp2(m_i - m) is their weight), applies norm and gain, and updates the weights.
// Everything is summed in a fixed order: results are the same from run to run.
#pragma once
#include "cache.cuh"
#include "fwd.cuh"

namespace da {

struct AttendArgs {
  CacheArgs c;
  const uint4* q1; const uint4* q2;            // strides in 16-byte pieces
  long long q_b, q_h;
  const uint4* nk1; const uint4* nk2; const uint4* nv;     // the new token (or null: the cache as it is)
  long long nk_b, nk_h, nv_b, nv_h;
  const int* counts;                           // [b] or null: only sequences with a positive one get their token
  float scale_log2;                            // log2(e) / sqrt(D): scores are kept in base 2
  const void* lambda_ptr;
  int lambda_dtype, rms_norm;
  float out_scale, eps;
  const float* gain;                           // [2D] or null
  __half* y;                                   // [b][h][2D]
  int box_rows;                                // rows of one TMA box
  int tiles_per_page;                          // 0: tiles run on over the pages; else a tile stays inside its page
  uint32_t tiles_magic;                        // ceil(2^32 / tiles_per_page), 0 for 1
  int workers;                                 // warps of the first kernel
  int join_blocks;                             // CTAs of the second one that join
  // workspace
  int* prefix;                                 // [b + 2] tiles of the sequences before b, per head; at the end the workers that have any
  int* length;                                 // [b] cached tokens, before this call's
  int* position;                               // [b] the new token's position
  float4* stats;                               // [workers + b * h] {m1, l1, m2, l2} of a piece; m: what its exponents are taken from, near its maximum
  float4* acc;                                 // [workers + b * h][D] O1[2D], O2[2D] of a piece
  float* scores;                               // [tiles][2][T] (with weights)
};

namespace attend {
constexpr int MAX_B = 4096;                    // the prefix sums and lengths of all sequences lie in shared memory
template <int D>
struct Geo {
  static constexpr int T = D == 32 ? 32 : 16;  // tokens per tile: 8 KB of K1, K2, V (D = 128: 16 KB)
  static constexpr int WARPS = D == 32 ? 8 : D == 64 ? 7 : 4, THREADS = WARPS * 32;
  // Tiles in flight per warp.  Warps x slots is what an SM has asked for, 112 to 128 KB.  More is slower, because the SMs then get their share of HBM
  // less evenly and the last one counts; fewer warps than this do not keep up.  B64 H16 ragged to 4096 D64: 7 x 2 180 us, 8 x 2 188, 8 x 3
  // 206, 12 x 2 198, 12 x 1 183 (but B1 H16 N16384 33 instead of 30), 6 x 2 207.  D = 32: 7 x 2 32 us, 8 x 2 30; D = 128: 4 x 2 88, 6 x 2 95.
  static constexpr int SLOTS = 2;
  // a tile in shared memory: boxes of T rows of 128 bytes (K at D = 32: 64 bytes), swizzled by the engine: K1, K2, V
  static constexpr int K_ROW = D == 32 ? 64 : 128, K_BOXES = D == 128 ? 2 : 1, V_BOXES = D / 32;
  static constexpr int K_BYTES = T * D * 2, V_BYTES = 2 * K_BYTES, SLOT_BYTES = 2 * K_BYTES + V_BYTES;
  static constexpr int Q_BYTES = 4 * D;        // the two queries of a (sequence, head), beside its first tile
  static constexpr int OFF_Q = WARPS * SLOTS * SLOT_BYTES;
  static constexpr int OFF_BAR = OFF_Q + WARPS * SLOTS * Q_BYTES;
  static constexpr int OFF_SUM = OFF_BAR + WARPS * SLOTS * 8 + 16;
  static constexpr int OFF_PREFIX = OFF_SUM + WARPS * 4;
  static constexpr int SMEM = OFF_PREFIX + 4 + 1024;      // + 8 b bytes of prefix sums and lengths; 1024 to align the ring
  static_assert(SMEM + 8 * MAX_B <= 227 * 1024, "shared memory");
};
}  // namespace attend

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// 8 x 8 transpose of 16-bit elements, two per lane (lane / 4: row, lane % 4: pair of columns)
__device__ __forceinline__ uint32_t movmatrix(uint32_t a) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}
// d[16 x 8] += a[16 x 16] b[16 x 8], fp32 sums
template <bool BF>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A place in the line of tiles: (sequence, head, tile), and the sequence's tiles and cached tokens.
struct TileWalk {
  int b, h, t, n, len;
};

__device__ __forceinline__ int divide(int n, int d, uint32_t magic) {      // as cache_page
  int q = magic ? int(__umulhi(uint32_t(n), magic)) : n;
  if ((long long)q * d > n) --q;
  return q;
}
// tiles of `len` cached tokens; a sequence that gets a token has one tile more, the last, for that alone
template <int T>
__device__ __forceinline__ int attend_tiles(const AttendArgs& a, int len) {
  if (!a.tiles_per_page) return (len + T - 1) / T;
  const int full = cache_page(a.c, len);
  return full * a.tiles_per_page + (len - full * a.c.page_size + T - 1) / T;
}
// the slot of a tile's first row and how many of its rows are live
template <int T>
__device__ __forceinline__ void attend_tile(const AttendArgs& a, int t, int len, int& slot, int& valid, bool& is_new) {
  slot = t * T;
  int end = len;
  if (a.tiles_per_page) {
    const int page = divide(t, a.tiles_per_page, a.tiles_magic);
    slot = page * a.c.page_size + (t - page * a.tiles_per_page) * T;
    end = min(len, (page + 1) * a.c.page_size);
    is_new = t >= attend_tiles<T>(a, len);
  } else {
    is_new = slot >= len;
  }
  valid = min(T, end - slot);
  if (is_new) {
    slot = len;
    valid = 1;
  }
}
// A division of 64-bit numbers costs 0.25 us, and four of them stood in a row before the first load; nearly always 32 bits do.
__device__ __forceinline__ long long quotient(long long n, long long d) {
  return ((n | d) >> 32) == 0 ? (long long)(uint32_t(n) / uint32_t(d)) : n / d;
}
__device__ __forceinline__ long long stretch_begin(long long units, int workers, int w) { return quotient(units * w, workers); }

// tile `u` of the line
__device__ __forceinline__ TileWalk walk_at(const AttendArgs& a, const int* prefix, const int* length, long long u) {
  int lo = 0, hi = a.c.b - 1;                  // the last b with h * prefix[b] <= u (sequences without tiles share a prefix: the last one has some)
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if ((long long)prefix[mid] * a.c.h <= u) lo = mid;
    else hi = mid - 1;
  }
  TileWalk w;
  w.b = lo;
  w.n = prefix[lo + 1] - prefix[lo];
  const long long r = u - (long long)prefix[lo] * a.c.h;
  w.h = int(quotient(r, w.n));
  w.t = int(r - (long long)w.h * w.n);
  w.len = length[lo];
  return w;
}
__device__ __forceinline__ void walk_next(const AttendArgs& a, const int* prefix, const int* length, TileWalk& w) {
  if (++w.t < w.n) return;
  w.t = 0;
  if (++w.h < a.c.h) return;
  w.h = 0;
  do {
    if (++w.b >= a.c.b) return;                // (behind the last tile: never used)
    w.n = prefix[w.b + 1] - prefix[w.b];
  } while (w.n == 0);
  w.len = length[w.b];
}

template <int D, bool BF, bool TRACK>
__global__ void __launch_bounds__(attend::Geo<D>::THREADS, 1)
diffattn_cache_attend_kernel(const __grid_constant__ CUtensorMap tm_k1, const __grid_constant__ CUtensorMap tm_k2,
                             const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ AttendArgs a) {
  using G = attend::Geo<D>;
  constexpr int T = G::T, WARPS = G::WARPS, SLOTS = G::SLOTS, THREADS = G::THREADS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* ring = smem + warp * (SLOTS * G::SLOT_BYTES);
  uint8_t* ring_q = smem + G::OFF_Q + warp * (SLOTS * G::Q_BYTES);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + G::OFF_BAR) + warp * SLOTS;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + G::OFF_BAR + WARPS * SLOTS * 8);
  volatile int* drain_flag = abort_flag + 1;
  int* part_sum = reinterpret_cast<int*>(smem + G::OFF_SUM);
  int* prefix = reinterpret_cast<int*>(smem + G::OFF_PREFIX);
  int* length = prefix + a.c.b + 1;            // (read once: all that follows has to agree on it)

  if (lane == 0) {
    for (int i = 0; i < SLOTS; ++i) mbar_init(&full[i], 1);
    mbar_init_fence();
  }
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    *drain_flag = 0;
    tma_prefetch_desc(&tm_k1); tma_prefetch_desc(&tm_k2); tma_prefetch_desc(&tm_v);
  }
  griddep_wait();
  griddep_launch();

  // ---- tiles of every sequence, summed up: a thread takes `per` consecutive sequences
  const int nb = a.c.b, per = (nb + THREADS - 1) / THREADS;
  const int b0 = min(int(threadIdx.x) * per, nb), b1 = min(b0 + per, nb);
  int sum = 0;
  for (int b = b0; b < b1; ++b) {
    const int len = cache_length(a.c, b);
    sum += attend_tiles<T>(a, len) + (a.nk1 && (!a.counts || a.counts[b] > 0) ? 1 : 0);
    prefix[b + 1] = sum;
    length[b] = len;
    if (blockIdx.x == 0) {                     // for the joining kernel, which finds the lengths moved on
      a.length[b] = len;
      if (a.nk1 && a.c.next_position) a.position[b] = a.c.next_position[b];
    }
  }
  int before = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += x;
  }
  if (lane == 31) part_sum[warp] = before;
  before -= sum;
  __syncthreads();
  for (int w = 0; w < warp; ++w) before += part_sum[w];
  for (int b = b0; b < b1; ++b) prefix[b + 1] += before;
  if (threadIdx.x == 0) prefix[0] = 0;
  __syncthreads();
  // Each worker's piece costs the joining kernel about 1 / 80 of what a tile costs here (a CTA joins them, four rounds of loads for 64), so with
  // very few heads more than sqrt(80 tiles heads) workers lose more there than they gain: B1 H1 N16384 D64 21.5 -> 15.7 us
  const long long units = (long long)prefix[nb] * a.c.h;
  const int most = int(min((long long)a.workers, units)), best = int(sqrtf(80.f * float(units) * float(nb * a.c.h)));
  const int workers = units > 0 ? max(min(most, best), 1) : 0;
  if (blockIdx.x == 0) {
    for (int b = threadIdx.x; b <= nb; b += THREADS) a.prefix[b] = prefix[b];
    if (threadIdx.x == 0) a.prefix[nb + 1] = workers;
  }

  const int worker = warp * int(gridDim.x) + int(blockIdx.x);      // few tiles: one to a CTA before any CTA has two
  if (worker >= workers) return;
  const long long first = stretch_begin(units, workers, worker);
  const int count = int(stretch_begin(units, workers, worker + 1) - first);

  // ---- loads.  Lane i fetches box i of a tile; its page is looked up one request ahead.
  TileWalk ahead = walk_at(a, prefix, length, first);
  auto next = [&](TileWalk& w) { walk_next(a, prefix, length, w); };
  struct Box { int page, in_page; };           // page -1: the engine fills the box with zeros; in_page -1: no such box
  auto look_up = [&](const TileWalk& w) {
    int slot, valid;
    bool is_new;
    attend_tile<T>(a, w.t, w.len, slot, valid, is_new);
    Box x{-1, -1};
    if (!is_new && lane * a.box_rows < valid) {
      slot += lane * a.box_rows;
      const int entry = cache_page(a.c, slot);
      x.in_page = slot - entry * a.c.page_size;
      x.page = cache_page_id(a.c, w.b, entry);
    }
    return x;
  };
  auto request = [&](const TileWalk& w, const Box& x, int s, bool with_q) {
    uint8_t* at = ring + s * G::SLOT_BYTES;
    const int boxes = __popc(__ballot_sync(0xffffffffu, x.in_page >= 0));      // 0: the new token
    if (lane == 0) {
      mbar_expect_tx(&full[s], (boxes ? boxes * a.box_rows * 8 * D : 8 * D) + (with_q ? G::Q_BYTES : 0));
      if (with_q) {
        bulk_load_1d(ring_q + s * G::Q_BYTES, a.q1 + w.b * a.q_b + w.h * a.q_h, 2 * D, &full[s]);
        bulk_load_1d(ring_q + s * G::Q_BYTES + 2 * D, a.q2 + w.b * a.q_b + w.h * a.q_h, 2 * D, &full[s]);
      }
      if (boxes == 0) {
        // row 0 of every box: the swizzle leaves it as it is
        for (int i = 0; i < G::K_BOXES; ++i) {
          bulk_load_1d(at + i * T * G::K_ROW, a.nk1 + w.b * a.nk_b + w.h * a.nk_h + i * 8, G::K_ROW, &full[s]);
          bulk_load_1d(at + G::K_BYTES + i * T * G::K_ROW, a.nk2 + w.b * a.nk_b + w.h * a.nk_h + i * 8, G::K_ROW, &full[s]);
        }
        for (int i = 0; i < G::V_BOXES; ++i) bulk_load_1d(at + 2 * G::K_BYTES + i * T * 128, a.nv + w.b * a.nv_b + w.h * a.nv_h + i * 8, 128, &full[s]);
      }
    }
    __syncwarp();
    if (x.in_page >= 0) {
      uint8_t* k = at + lane * a.box_rows * G::K_ROW;
      uint8_t* v = at + 2 * G::K_BYTES + lane * a.box_rows * 128;
#pragma unroll
      for (int i = 0; i < G::K_BOXES; ++i) {
        tma_load_4d(k + i * T * G::K_ROW, &tm_k1, &full[s], i * 64, x.in_page, w.h, x.page);
        tma_load_4d(k + G::K_BYTES + i * T * G::K_ROW, &tm_k2, &full[s], i * 64, x.in_page, w.h, x.page);
      }
#pragma unroll
      for (int i = 0; i < G::V_BOXES; ++i) tma_load_4d(v + i * T * 128, &tm_v, &full[s], i * 64, x.in_page, w.h, x.page);
    }
  };
  TileWalk cur = ahead;
  Box box{-1, -1};
  {
    TileWalk w[SLOTS];
    Box x[SLOTS];
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
      w[i] = ahead;
      if (i < count) x[i] = look_up(ahead);
      if (i + 1 < count) next(ahead);
    }
#pragma unroll
    for (int i = 0; i < SLOTS; ++i)
      if (i < count) request(w[i], x[i], i, i == 0 || w[i].t == 0);
    if (SLOTS < count) box = look_up(ahead);
  }

  // ---- the stretch.  With the rows r = 8 x matrix and columns c of the fragments as mma.sync lays them out:
  //  scores  S_b[16 tokens x 8] = K_b Q^T, Q^T's columns q1, q1, q2, q2, 0, 0, 0, 0: lane % 4 = 0 has S_1, lane % 4 = 1 has S_2 of tokens lane / 4
  //          and lane / 4 + 8, the other lanes nothing
  //  P       a probability as two 16-bit numbers, its rounding and what that left out, side by side in columns 2 b, 2 b + 1: transposed it is the
  //          operand of
  //  output  O^T[16 values x 8] += V^T P^T, columns O_1 (two shares), O_2 (two shares): the same lanes have the same branch
  // What P loses: bf16 2^-17 of a probability.  fp16 has too few exponents for that in a long cache, where one token may be far above thousands that
  // count together.  So its first number is kept 2^UP higher (the largest one between 2^7 and 2^15, where fp16 ends at 2^16) and its second one,
  // which is 2^-11 of the first, 2^LOW higher again: off by 2^-22 of a probability, or 2^-43 of the largest one, whichever is more.
  // (Without, 2^-25 of the largest: 16384 tokens of that size were lost from O but not from l.)
  constexpr float UP = BF ? 0.f : 7.f, SLACK = 8.f, LOW = BF ? 1.f : 2048.f;
  const int branch = lane & 3;                 // 0, 1; 2 and 3: none
  const uint32_t row_k = smem_u32(ring) + (lane & 15) * G::K_ROW, row_v = smem_u32(ring) + 2 * G::K_BYTES + ((lane & 7) + ((lane >> 4) << 3)) * 128;
  const uint32_t sw_k = D == 32 ? ((lane >> 4) ^ ((lane >> 1) & 3)) << 4 : ((lane >> 4) ^ (lane & 7)) << 4, sw_v = (((lane >> 3) & 1) ^ (lane & 7)) << 4;
  uint32_t q[D / 16][2];
  float o[D / 8][4];
  float m = 0.f, l = 0.f;                      // of this lane's branch; l: of the tokens that this lane had
  int s = 0, phase = 0;
  for (int i = 0; i < count; ++i) {
    if (!mbar_wait_warp(&full[s], phase, abort_flag, 801, i)) {
      // copies still in flight must land before the shared memory goes away
      for (int k = 1; k < SLOTS && i + k < count; ++k) {
        const int s2 = (s + k) % SLOTS;
        mbar_wait_warp(&full[s2], s + k >= SLOTS ? phase ^ 1 : phase, drain_flag, 802, i);
      }
      return;
    }
    int slot, valid;
    bool is_new;
    attend_tile<T>(a, cur.t, cur.len, slot, valid, is_new);
    if (i == 0 || cur.t == 0) {
      // a (sequence, head) begins
      const int n = lane >> 2;
      const uint32_t* src = reinterpret_cast<const uint32_t*>(ring_q + s * G::Q_BYTES + (n < 2 ? 0 : 2 * D)) + branch;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        q[k][0] = n < 4 ? src[k * 8] : 0u;
        q[k][1] = n < 4 ? src[k * 8 + 4] : 0u;
      }
#pragma unroll
      for (int k = 0; k < D / 8; ++k) o[k][0] = o[k][1] = o[k][2] = o[k][3] = 0.f;
      m = -3e38f;                              // (finite: a score of -inf then counts as 0 instead of as not a number)
      l = 0.f;
    }
    if (valid < T) {
      uint8_t* tile = ring + s * G::SLOT_BYTES;
      if (is_new && slot < a.c.slots) {
        // the new token goes into the cache on its way
        const int entry = cache_page(a.c, slot);
        const int page = cache_page_id(a.c, cur.b, entry);
        for (int part = lane; page >= 0 && part < D / 2; part += 32) {
          const int c = part < D / 8 ? part : part < D / 4 ? part - D / 8 : part - D / 4;      // 16-byte piece of its row; eight to a box
          const int off = part < D / 4 ? (part < D / 8 ? 0 : G::K_BYTES) + (c >> 3) * T * G::K_ROW : 2 * G::K_BYTES + (c >> 3) * T * 128;
          *cache_piece<D>(a.c, page, cur.h, slot - entry * a.c.page_size, part) = *reinterpret_cast<const uint4*>(tile + off + (c & 7) * 16);
        }
      }
      // whatever lies in rows of V that are not live: 0 times it has to be 0
      for (int r = valid + (lane >> 3); r < T; r += 4)
#pragma unroll
        for (int x = 0; x < G::V_BOXES; ++x) *reinterpret_cast<uint4*>(tile + 2 * G::K_BYTES + x * T * 128 + r * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
      __syncwarp();
    }
    const uint32_t at_k = row_k + s * G::SLOT_BYTES, at_v = row_v + s * G::SLOT_BYTES;
    float p[T / 16][2];
    float top = -INFINITY;
#pragma unroll
    for (int g = 0; g < T / 16; ++g) {
      float s1[4] = {0.f, 0.f, 0.f, 0.f}, s2[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        const uint32_t off = (k >> 2) * T * G::K_ROW + g * 16 * G::K_ROW + (sw_k ^ ((k & 3) << 5));
        uint32_t x[4];
        ldsm4(x, at_k + off);
        mma16816<BF>(s1, x, q[k][0], q[k][1]);
        ldsm4(x, at_k + G::K_BYTES + off);
        mma16816<BF>(s2, x, q[k][0], q[k][1]);
      }
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        p[g][x] = (branch ? s2[2 * x] : s1[2 * x]) * a.scale_log2;
        if (branch > 1 || g * 16 + x * 8 + (lane >> 2) >= valid) p[g][x] = -INFINITY;
        if (TRACK && branch < 2) a.scores[((first + i) * 2 + branch) * T + g * 16 + x * 8 + (lane >> 2)] = p[g][x];
        top = fmaxf(top, p[g][x]);
      }
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
    // m, 2^UP below a maximum, moves only when that is exceeded by more than 2^SLACK: the probabilities stay inside fp16's range either way
    const bool need = top > m + (UP + SLACK);
    if (__any_sync(0xffffffffu, need)) {
      const float to = need ? top - UP : m, f = ex2(m - to);
      l *= f;
      m = to;
#pragma unroll
      for (int k = 0; k < D / 8; ++k) {
        o[k][0] *= f; o[k][1] *= f; o[k][2] *= f; o[k][3] *= f;
      }
    }
#pragma unroll
    for (int g = 0; g < T / 16; ++g) {
      uint32_t pb[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float e = ex2(p[g][x] - m);
        l += e;
        const float hi = to_float16b<BF>(from_float16b<BF>(e));
        pb[x] = movmatrix(pack2<BF>(hi, (e - hi) * LOW));
      }
#pragma unroll
      for (int k = 0; k < D / 8; ++k) {
        uint32_t x[4];
        ldsm4_trans(x, at_v + (k >> 2) * T * 128 + g * 16 * 128 + (sw_v ^ ((k & 3) << 5)));
        mma16816<BF>(o[k], x, pb[0], pb[1]);
      }
    }
    if (valid < T) fence_proxy_async_smem();   // (rows were written by this warp)
    __syncwarp();                              // the tile is read: its slot takes the next one
    if (i + SLOTS < count) {
      request(ahead, box, s, ahead.t == 0);
      if (i + SLOTS + 1 < count) {
        next(ahead);
        box = look_up(ahead);
      }
    }
    if (cur.t == cur.n - 1 || i == count - 1) {
      // the stretch leaves this (sequence, head)
      l += __shfl_xor_sync(0xffffffffu, l, 4);
      l += __shfl_xor_sync(0xffffffffu, l, 8);
      l += __shfl_xor_sync(0xffffffffu, l, 16);
      const size_t at = size_t(worker) + size_t(cur.b) * a.c.h + cur.h;      // a piece's place: grows with every piece along the line
      if (lane < 2) reinterpret_cast<float2*>(a.stats + at)[lane] = make_float2(m, l);
      if (branch < 2) {
        float* to = reinterpret_cast<float*>(a.acc + at * D) + branch * 2 * D + (lane >> 2);
#pragma unroll
        for (int k = 0; k < D / 8; ++k) {
          to[k * 16] = o[k][0] + o[k][1] * (1.f / LOW);
          to[k * 16 + 8] = o[k][2] + o[k][3] * (1.f / LOW);
        }
      }
    }
    if (i + 1 < count) next(cur);
    if (++s == SLOTS) { s = 0; phase ^= 1; }
  }
}

// ---------------------------------------------------------------------------------------------
// Joins the pieces of every (sequence, head), and adds the tokens' weights.
// ---------------------------------------------------------------------------------------------
struct Joined { float m1, l1, m2, l2; };       // the largest m and the sum of both branches over all pieces

// the pieces of tiles [u, u + n) of the line: workers w0 .. w1
__device__ __forceinline__ void piece_range(long long units, int workers, long long u, int n, int& w0, int& w1) {
  w0 = int(quotient((u + 1) * workers - 1, units));           // the last worker whose stretch begins at or before u
  w1 = int(quotient((u + n) * workers - 1, units));
}
__device__ __forceinline__ void join(float& m, float& l, float m2, float l2) {
  const float top = fmaxf(m, m2);
  l = l * ex2(m - top) + l2 * ex2(m2 - top);
  m = top;
}
__device__ __forceinline__ void join_lanes(Joined& j) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    join(j.m1, j.l1, __shfl_xor_sync(0xffffffffu, j.m1, o), __shfl_xor_sync(0xffffffffu, j.l1, o));
    join(j.m2, j.l2, __shfl_xor_sync(0xffffffffu, j.m2, o), __shfl_xor_sync(0xffffffffu, j.l2, o));
  }
}
__device__ __forceinline__ Joined join_stats(const float4* stats, int first, int last, int step, int lane) {      // a whole warp: pieces first + lane, ...
  Joined j{-3e38f, 0.f, -3e38f, 0.f};
#pragma unroll 2
  for (int w = first + lane; w <= last; w += step) {
    const float4 x = stats[w];
    join(j.m1, j.l1, x.x, x.y);
    join(j.m2, j.l2, x.z, x.w);
  }
  join_lanes(j);
  return j;
}

// What a call leaves behind besides y, for (sequence, head) bh of n tiles; one thread.
template <int T>
__device__ __forceinline__ void join_finish(const AttendArgs& a, int bh, int b, int head, int n) {
  if (a.nk1 == nullptr) return;
  const int len = a.length[b];
  if (n <= attend_tiles<T>(a, len)) return;    // no token
  if (len < a.c.slots) {
    if (a.c.positions) a.c.positions[(size_t)bh * a.c.slots + len] = a.position[b];
    if (head == 0) {
      a.c.lengths[b] = len + 1;
      if (a.c.next_position) a.c.next_position[b] = a.position[b] + 1;
    }
  } else {
    if (head == 0) a.c.lengths[b] = len;
    cache_fault(kCacheFull, b, len);
  }
}

// The weights of a share of one (sequence, head)'s tokens; a CTA of JT threads.
template <int T, int JT>
__device__ __forceinline__ void join_weights(const AttendArgs& a, int bh, int share, int shares) {
  const int heads = a.c.h, b = bh / heads, head = bh - b * heads, lane = threadIdx.x & 31;
  const int p0 = a.prefix[b], n = a.prefix[b + 1] - p0, len = a.length[b];
  const long long units = (long long)a.prefix[a.c.b] * heads;
  if (n == 0) return;
  const int workers = a.prefix[a.c.b + 1];
  const float lam = load_lambda(a.lambda_ptr, a.lambda_dtype);
  const long long u = (long long)p0 * heads + (long long)head * n;
  int w0, w1;
  piece_range(units, workers, u, n, w0, w1);
  const Joined j = join_stats(a.stats + bh, w0, w1, 32, lane);
  const float c1 = 1.f / j.l1, c2 = lam / j.l2;
  float* to = a.c.weights + (size_t)bh * a.c.slots;
  const float* scores = a.scores + u * 2 * T;
  constexpr int ROUND = 4;                     // tokens of a thread whose loads are under way together
  for (int t0 = share * (JT / T) * ROUND; t0 < n; t0 += shares * (JT / T) * ROUND) {
    float s1[ROUND], s2[ROUND], old[ROUND];
    int at[ROUND];                             // -1: no token
#pragma unroll
    for (int k = 0; k < ROUND; ++k) {
      const int tile = t0 + (k * JT + int(threadIdx.x)) / T, row = threadIdx.x % T;
      at[k] = -1;
      if (tile >= n) continue;
      int slot, valid;
      bool is_new;
      attend_tile<T>(a, tile, len, slot, valid, is_new);
      if (row >= valid || slot + row >= a.c.slots) continue;
      at[k] = slot + row;
      s1[k] = scores[(long long)tile * 2 * T + row];
      s2[k] = scores[(long long)tile * 2 * T + T + row];
      old[k] = is_new ? 0.f : to[at[k]];
    }
#pragma unroll
    for (int k = 0; k < ROUND; ++k)
      if (at[k] >= 0) to[at[k]] = old[k] + fabsf(ex2(s1[k] - j.m1) * c1 - ex2(s2[k] - j.m2) * c2);
  }
}

// Two forms.  What counts is the chain of loads, prefix sums, statistics, sums, each about 0.7 us away in L2.  Several pieces a (sequence, head):
// JT threads join them, so that all loads of a round go out together.  Few: a warp does, without a barrier, and a CTA holds eight.
// In both the first `a.join_blocks` CTAs join and those behind them add weights: neither chain waits for the other.
constexpr int JOIN_FEW = 256;

template <int D, int JT, bool BF, bool TRACK>
__global__ void __launch_bounds__(JT) diffattn_cache_join_kernel(const __grid_constant__ AttendArgs a) {
  constexpr int T = attend::Geo<D>::T;
  constexpr int GROUPS = JT / D;        // pieces summed side by side: a thread has four of a piece's 4 D sums
  constexpr int AHEAD = JT == 256 ? 4 : 6;       // pieces whose sums a thread requests before it knows their weights
  __shared__ float4 red[JT];
  __shared__ Joined part[JT / 32];
  __shared__ float ssq[2 * D / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  griddep_wait();
  griddep_launch();
  const int nb = a.c.b, heads = a.c.h;
  if (int(blockIdx.x) >= a.join_blocks) {
    if constexpr (TRACK) {
      const int at = int(blockIdx.x) - a.join_blocks;
      join_weights<T, JT>(a, at % (nb * heads), at / (nb * heads), int(gridDim.x - a.join_blocks) / (nb * heads));
    }
    return;
  }
  const long long units = (long long)a.prefix[nb] * heads;
  const int workers = a.prefix[nb + 1];
  const float lam = load_lambda(a.lambda_ptr, a.lambda_dtype);
  const int bh = blockIdx.x, b = bh / heads, head = bh - b * heads;
  const int n = a.prefix[b + 1] - a.prefix[b];
  const float gain = a.gain && threadIdx.x < 2 * D ? a.gain[threadIdx.x] : 1.f;
  float out = 0.f;
  if (n > 0) {
    int w0, w1;
    piece_range(units, workers, (long long)a.prefix[b] * heads + (long long)head * n, n, w0, w1);
    const float4* stats = a.stats + bh;
    const int col = threadIdx.x % D, group = threadIdx.x / D;
    const bool second = col >= D / 2;
    const float4* acc = a.acc + (size_t)bh * D + col;
    float4 x[AHEAD];
    float mx[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int w = w0 + group + k * GROUPS;
      if (w <= w1) {
        x[k] = acc[(size_t)w * D];
        mx[k] = second ? stats[w].z : stats[w].x;
      }
    }
    Joined j = join_stats(stats, w0 + warp * 32, w1, JT, lane);
    if (lane == 0) part[warp] = j;
    __syncthreads();
    j = lane < JT / 32 ? part[lane] : Joined{-3e38f, 0.f, -3e38f, 0.f};
    join_lanes(j);
    const float top = second ? j.m2 : j.m1;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](const float4& v, float m) {
      const float c = ex2(m - top);
      sum.x += c * v.x; sum.y += c * v.y; sum.z += c * v.z; sum.w += c * v.w;
    };
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (w0 + group + k * GROUPS <= w1) add(x[k], mx[k]);
#pragma unroll 4
    for (int w = w0 + group + AHEAD * GROUPS; w <= w1; w += GROUPS) add(acc[(size_t)w * D], second ? stats[w].z : stats[w].x);
    red[threadIdx.x] = sum;
    __syncthreads();
    if (threadIdx.x < 2 * D) {
      const float* r = reinterpret_cast<const float*>(red);
      float o1 = 0.f, o2 = 0.f;
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {
        o1 += r[g * 4 * D + threadIdx.x];
        o2 += r[g * 4 * D + 2 * D + threadIdx.x];
      }
      out = o1 / j.l1 - lam * (o2 / j.l2);
      float sq = out * out;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
      if (lane == 0) ssq[warp] = sq;
    }
    __syncthreads();
    if (a.rms_norm) {
      float sq = 0.f;
#pragma unroll
      for (int k = 0; k < 2 * D / 32; ++k) sq += ssq[k];
      out *= rsqrtf(sq / float(2 * D) + a.eps) * a.out_scale;
    }
  }
  if (threadIdx.x < 2 * D) a.y[size_t(bh) * 2 * D + threadIdx.x] = from_float16b<BF>(out * gain);
  if (threadIdx.x == 0) join_finish<T>(a, bh, b, head, n);
}

template <int D, bool BF, bool TRACK>
__global__ void __launch_bounds__(JOIN_FEW) diffattn_cache_join_few_kernel(const __grid_constant__ AttendArgs a) {
  constexpr int T = attend::Geo<D>::T;
  constexpr int C = 2 * D / 32;                // value columns of a lane, neighbours: 2, 4 or 8
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  griddep_wait();
  griddep_launch();
  const int nb = a.c.b, heads = a.c.h;
  if (int(blockIdx.x) >= a.join_blocks) {
    if constexpr (TRACK) {
      const int at = int(blockIdx.x) - a.join_blocks;
      join_weights<T, JOIN_FEW>(a, at % (nb * heads), at / (nb * heads), int(gridDim.x - a.join_blocks) / (nb * heads));
    }
    return;
  }
  const int bh = blockIdx.x * (JOIN_FEW / 32) + warp;
  if (bh >= nb * heads) return;
  const long long units = (long long)a.prefix[nb] * heads;
  const int workers = a.prefix[nb + 1];
  const float lam = load_lambda(a.lambda_ptr, a.lambda_dtype);
  const int b = bh / heads, head = bh - b * heads;
  const int n = a.prefix[b + 1] - a.prefix[b];
  float out[C];
#pragma unroll
  for (int k = 0; k < C; ++k) out[k] = 0.f;
  if (n > 0) {
    int w0, w1;
    piece_range(units, workers, (long long)a.prefix[b] * heads + (long long)head * n, n, w0, w1);
    const float4* stats = a.stats + bh;
    const float* acc = reinterpret_cast<const float*>(a.acc + (size_t)bh * D) + lane * C;
    const Joined j = join_stats(stats, w0, w1, 32, lane);
    float o1[C], o2[C];
#pragma unroll
    for (int k = 0; k < C; ++k) o1[k] = o2[k] = 0.f;
#pragma unroll 4
    for (int w = w0; w <= w1; ++w) {
      const float c1 = ex2(stats[w].x - j.m1), c2 = ex2(stats[w].z - j.m2);
      const float* x = acc + (size_t)w * 4 * D;
#pragma unroll
      for (int k = 0; k < C; k += 2) {
        const float2 p = *reinterpret_cast<const float2*>(x + k), q = *reinterpret_cast<const float2*>(x + 2 * D + k);
        o1[k] += c1 * p.x; o1[k + 1] += c1 * p.y;
        o2[k] += c2 * q.x; o2[k + 1] += c2 * q.y;
      }
    }
    float sq = 0.f;
#pragma unroll
    for (int k = 0; k < C; ++k) {
      out[k] = o1[k] / j.l1 - lam * (o2[k] / j.l2);
      sq += out[k] * out[k];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
    const float scale = a.rms_norm ? rsqrtf(sq / float(2 * D) + a.eps) * a.out_scale : 1.f;
#pragma unroll
    for (int k = 0; k < C; ++k) out[k] *= scale;
  }
  uint32_t* y = reinterpret_cast<uint32_t*>(a.y + size_t(bh) * 2 * D + lane * C);
#pragma unroll
  for (int k = 0; k < C; k += 2) {
    const float g0 = a.gain ? a.gain[lane * C + k] : 1.f, g1 = a.gain ? a.gain[lane * C + k + 1] : 1.f;
    y[k / 2] = pack2<BF>(out[k] * g0, out[k + 1] * g1);
  }
  if (lane == 0) join_finish<T>(a, bh, b, head, n);
}

}  // namespace da
