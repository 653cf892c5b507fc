// Differential attention of one new token per (sequence, head) over a paged cache.
//
//   s_b[j] = q_b . k_b[j] / sqrt(D),  P_b = softmax(s_b),  A = P_1 V - lambda P_2 V,  y = A * norm * gain;  w[j] += |P_1[j] - lambda P_2[j]|
//
// Bound by HBM: every cached row (8 D bytes) is read once for 12 D flops.  A row meets one query only, so there is no matrix product with
// more than one row and the tensor cores have nothing to do; fp32 fused multiply-adds in pairs need a third of the issue slots.
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
  float scale_log2;                            // log2(e) / sqrt(D): scores are kept in base 2
  const void* lambda_ptr;
  int lambda_dtype, rms_norm;
  float out_scale, eps;
  const float* gain;                           // [2D] or null
  __half* y;                                   // [b][h][2D]
  int box_rows;                                // rows of one TMA box; several pages make a tile where this is less than a tile
  int tiles_per_page;                          // 1 where several pages make a tile
  int workers;                                 // warps of the first kernel
  // workspace
  int* prefix;                                 // [b + 1] tiles of the sequences before b, per head
  int* length;                                 // [b] cached tokens, before this call's
  int* position;                               // [b] the new token's position
  float4* stats;                               // [workers + b * h] {m1, l1, m2, l2} of a piece
  float4* acc;                                 // [workers + b * h][D] O1[2D], O2[2D] of a piece
  float* scores;                               // [tiles][2][T] (with weights)
};

namespace attend {
constexpr int WARPS = 8, THREADS = WARPS * 32;
constexpr int SLOTS = 3;                       // tiles in flight per warp: 192 KB of requests per SM
constexpr int MAX_B = 4096;                    // the prefix sums of all sequences lie in shared memory
template <int D>
struct Geo {
  static constexpr int T = 1024 / D;           // tokens per tile: 8 KB of K1, K2, V
  static constexpr int K_BYTES = T * D * 2, V_BYTES = 2 * K_BYTES, Q_BYTES = 2 * D * 2;
  static constexpr int SLOT_BYTES = 2 * K_BYTES + V_BYTES + 512;     // the queries of a stretch's first tile lie behind the tile
  static constexpr int OFF_P = WARPS * SLOTS * SLOT_BYTES;           // probabilities of the current tile, per warp
  static constexpr int OFF_BAR = OFF_P + WARPS * 2 * T * 4;
  static constexpr int OFF_PREFIX = OFF_BAR + WARPS * SLOTS * 8 + 16;
  static constexpr int SMEM = OFF_PREFIX + 16 + THREADS / 32 * 4;    // + 4 (b + 1) bytes of prefix sums
  static_assert(SMEM + 4 * (MAX_B + 1) + 128 <= 227 * 1024, "shared memory");
};
}  // namespace attend

// A place in the line of tiles: (sequence, head, tile), and the sequence's tiles and cached tokens.
struct TileWalk {
  int b, h, t, n, len;
};

template <int T>
__device__ __forceinline__ int attend_tiles(const AttendArgs& a, int len) {
  int n;
  if (a.box_rows < T || a.tiles_per_page == 1) {
    // several pages per tile (T is a multiple of page_size), or a page per tile
    n = a.box_rows < T ? (len + T - 1) / T : cache_page(a.c, len + a.c.page_size - 1);
  } else {
    const int full = cache_page(a.c, len);
    n = full * a.tiles_per_page + (len - full * a.c.page_size + T - 1) / T;
  }
  return n + (a.nk1 != nullptr ? 1 : 0);
}
// where a tile's rows begin and how many of them are live; the new token is a tile of its own, the last
template <int T>
__device__ __forceinline__ void attend_tile(const AttendArgs& a, int t, int n, int len, int& slot, int& in_page, int& valid, bool& is_new) {
  is_new = a.nk1 != nullptr && t == n - 1;
  if (is_new) {
    slot = len; in_page = 0; valid = 1;
    return;
  }
  if (a.box_rows < T) {
    slot = t * T; in_page = 0;
    valid = min(T, len - slot);
    return;
  }
  const int page = a.tiles_per_page == 1 ? t : t / a.tiles_per_page;
  in_page = (t - page * a.tiles_per_page) * T;
  slot = page * a.c.page_size + in_page;
  valid = min(min(T, a.c.page_size - in_page), len - slot);
}
__device__ __forceinline__ long long stretch_begin(long long units, int workers, int w) { return units * w / workers; }

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
  w.h = int(r / w.n);
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

__device__ __forceinline__ f32x2 widen(float2 x) { return pk2(x.x, x.y); }

template <int D, bool BF, bool TRACK>
__global__ void __launch_bounds__(attend::THREADS, 1)
diffattn_cache_attend_kernel(const __grid_constant__ CUtensorMap tm_k1, const __grid_constant__ CUtensorMap tm_k2,
                             const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ AttendArgs a) {
  using namespace attend;
  using G = Geo<D>;
  constexpr int T = G::T;
  constexpr int LPK = D / 8, LPV = D / 4;      // lanes (16-byte pieces) per K row, per V row
  constexpr int M1 = LPK / 2, M2 = LPK / 4, M3 = LPK / 8;      // lane bits that select branch and row in the sums over a row's lanes
  constexpr int NV = LPK < 8 ? 2 : 1;          // scores a lane ends up with
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~uintptr_t(127));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* ring = smem + warp * (SLOTS * G::SLOT_BYTES);
  float* prob = reinterpret_cast<float*>(smem + G::OFF_P) + warp * 2 * T;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + G::OFF_BAR) + warp * SLOTS;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + G::OFF_BAR + WARPS * SLOTS * 8);
  volatile int* drain_flag = abort_flag + 1;
  int* part_sum = reinterpret_cast<int*>(smem + G::OFF_PREFIX);
  int* prefix = part_sum + WARPS;

  if (lane == 0) {
    for (int i = 0; i < SLOTS; ++i) mbar_init(&full[i], 1);
    mbar_init_fence();
  }
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    *drain_flag = 0;
    tma_prefetch_desc(&tm_k1); tma_prefetch_desc(&tm_k2); tma_prefetch_desc(&tm_v);
  }
  griddep_launch();

  // ---- tiles of every sequence, summed up: a thread takes `per` consecutive sequences
  const int nb = a.c.b, per = (nb + THREADS - 1) / THREADS;
  const int b0 = min(int(threadIdx.x) * per, nb), b1 = min(b0 + per, nb);
  int sum = 0;
  for (int b = b0; b < b1; ++b) {
    const int len = cache_length(a.c, b);
    sum += attend_tiles<T>(a, len);
    prefix[b + 1] = sum;
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
  if (blockIdx.x == 0)
    for (int b = threadIdx.x; b <= nb; b += THREADS) a.prefix[b] = prefix[b];

  const long long units = (long long)prefix[nb] * a.c.h;
  const int workers = int(min((long long)a.workers, units));
  const int worker = warp * int(gridDim.x) + int(blockIdx.x);      // few tiles: one to a CTA before any CTA has two
  if (worker >= workers) return;
  const long long first = stretch_begin(units, workers, worker);
  const int count = int(stretch_begin(units, workers, worker + 1) - first);

  // ---- loads.  A tile's boxes: one, or one per page where pages are smaller than a tile; lane i has the page of box i.
  TileWalk ahead = walk_at(a, prefix, a.c.lengths, first);
  ahead.len = min(max(ahead.len, 0), a.c.slots);
  auto next = [&](TileWalk& w) {
    walk_next(a, prefix, a.c.lengths, w);
    w.len = min(max(w.len, 0), a.c.slots);
  };
  auto page_ids = [&](const TileWalk& w) {
    int slot, in_page, valid;
    bool is_new;
    attend_tile<T>(a, w.t, w.n, w.len, slot, in_page, valid, is_new);
    int id = 0;
    if (!is_new && lane * a.box_rows < valid) id = cache_page_id(a.c, w.b, cache_page(a.c, slot) + lane);
    return id;                                 // (-1: the engine fills the box with zeros)
  };
  auto request = [&](const TileWalk& w, int id, int s, bool with_q) {
    int slot, in_page, valid;
    bool is_new;
    attend_tile<T>(a, w.t, w.n, w.len, slot, in_page, valid, is_new);
    uint8_t* at = ring + s * G::SLOT_BYTES;
    if (lane == 0) {
      const int boxes = is_new ? 0 : (valid + a.box_rows - 1) / a.box_rows;
      mbar_expect_tx(&full[s], (is_new ? 8 * D : boxes * a.box_rows * 8 * D) + (with_q ? G::Q_BYTES : 0));
      if (with_q) {
        uint8_t* q = at + 2 * G::K_BYTES + G::V_BYTES;
        bulk_load_1d(q, a.q1 + w.b * a.q_b + w.h * a.q_h, G::Q_BYTES / 2, &full[s]);
        bulk_load_1d(q + G::Q_BYTES / 2, a.q2 + w.b * a.q_b + w.h * a.q_h, G::Q_BYTES / 2, &full[s]);
      }
      if (is_new) {
        bulk_load_1d(at, a.nk1 + w.b * a.nk_b + w.h * a.nk_h, 2 * D, &full[s]);
        bulk_load_1d(at + G::K_BYTES, a.nk2 + w.b * a.nk_b + w.h * a.nk_h, 2 * D, &full[s]);
        bulk_load_1d(at + 2 * G::K_BYTES, a.nv + w.b * a.nv_b + w.h * a.nv_h, 4 * D, &full[s]);
      }
    }
    __syncwarp();
    if (!is_new && lane * a.box_rows < valid) {
      const int off = lane * a.box_rows * 2 * D;
      tma_load_4d(at + off, &tm_k1, &full[s], 0, in_page, w.h, id);
      tma_load_4d(at + G::K_BYTES + off, &tm_k2, &full[s], 0, in_page, w.h, id);
      tma_load_4d(at + 2 * G::K_BYTES + 2 * off, &tm_v, &full[s], 0, in_page, w.h, id);
    }
  };
  TileWalk cur = ahead;
  int id;
  {
    TileWalk w[SLOTS];
    int ids[SLOTS];
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
      w[i] = ahead;
      ids[i] = i < count ? page_ids(ahead) : 0;
      if (i + 1 < count) next(ahead);
    }
#pragma unroll
    for (int i = 0; i < SLOTS; ++i)
      if (i < count) request(w[i], ids[i], i, i == 0 || w[i].t == 0);
    id = SLOTS < count ? page_ids(ahead) : 0;
  }

  // ---- the stretch
  f32x2 q[2][4], o[2][4];
  float m = 0.f, l = 0.f;                      // of this lane's branch (bit M1 of the lane); l: of the scores that this lane had
  const bool second = lane & M1;
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
    const uint8_t* tile = ring + s * G::SLOT_BYTES;
    int slot, in_page, valid;
    bool is_new;
    attend_tile<T>(a, cur.t, cur.n, cur.len, slot, in_page, valid, is_new);
    if (i == 0 || cur.t == 0) {
      // a (sequence, head) begins: its queries, scaled so that scores come out in base 2
      const f32x2 sc = pk2(a.scale_log2, a.scale_log2);
#pragma unroll
      for (int br = 0; br < 2; ++br) {
        const uint4 w = *reinterpret_cast<const uint4*>(tile + 2 * G::K_BYTES + G::V_BYTES + br * 2 * D + (lane & (LPK - 1)) * 16);
        q[br][0] = mul2(widen(unpack2<BF>(w.x)), sc);
        q[br][1] = mul2(widen(unpack2<BF>(w.y)), sc);
        q[br][2] = mul2(widen(unpack2<BF>(w.z)), sc);
        q[br][3] = mul2(widen(unpack2<BF>(w.w)), sc);
#pragma unroll
        for (int k = 0; k < 4; ++k) o[br][k] = pk2(0.f, 0.f);
      }
      m = -3e38f;                              // (finite: a score of -inf then counts as 0 instead of as not a number)
      l = 0.f;
    }
    if (is_new && slot < a.c.slots) {
      // the new token goes into the cache on its way
      const int p = cache_page(a.c, slot);
      const int page = cache_page_id(a.c, cur.b, p);
      for (int part = lane; page >= 0 && part < D / 2; part += 32) {
        const int off = part < D / 8 ? part * 16 : part < D / 4 ? G::K_BYTES + (part - D / 8) * 16 : 2 * G::K_BYTES + (part - D / 4) * 16;
        *cache_piece<D>(a.c, page, cur.h, slot - p * a.c.page_size, part) = *reinterpret_cast<const uint4*>(tile + off);
      }
    }
    // scores: a lane's share of four rows of either branch, then sums over the lanes of a row; every exchange halves the values, so that
    // each lane ends with the scores of NV rows of one branch (7 shuffles for 8 rows instead of 24 at D = 64)
    float part[8];
#pragma unroll
    for (int br = 0; br < 2; ++br)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const uint4 w = *reinterpret_cast<const uint4*>(tile + br * G::K_BYTES + (r * 32 + lane) * 16);
        f32x2 x = mul2(widen(unpack2<BF>(w.x)), q[br][0]);
        x = fma2(widen(unpack2<BF>(w.y)), q[br][1], x);
        x = fma2(widen(unpack2<BF>(w.z)), q[br][2], x);
        x = fma2(widen(unpack2<BF>(w.w)), q[br][3], x);
        float lo, hi;
        up2(x, lo, hi);
        part[br * 4 + r] = lo + hi;
      }
    float sc[NV];
    {
      float x[4], y[2];
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] = (second ? part[4 + k] : part[k]) + __shfl_xor_sync(0xffffffffu, second ? part[k] : part[4 + k], M1);
      const bool up = lane & M2;
#pragma unroll
      for (int k = 0; k < 2; ++k) y[k] = (up ? x[2 + k] : x[k]) + __shfl_xor_sync(0xffffffffu, up ? x[k] : x[2 + k], M2);
      if constexpr (NV == 2) {
        sc[0] = y[0]; sc[1] = y[1];
      } else {
        const bool odd = lane & M3;
        sc[0] = (odd ? y[1] : y[0]) + __shfl_xor_sync(0xffffffffu, odd ? y[0] : y[1], M3);
        if constexpr (LPK == 16) sc[0] += __shfl_xor_sync(0xffffffffu, sc[0], 1);
      }
    }
    int row[NV];
    float top = -INFINITY;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int r = ((lane & M2) ? 2 : 0) + (NV == 2 ? v : (lane & M3) ? 1 : 0);
      row[v] = r * (32 / LPK) + lane / LPK;
      if (row[v] >= valid) sc[v] = -INFINITY;
      top = fmaxf(top, sc[v]);
    }
#pragma unroll
    for (int x = 1; x < 32; x <<= 1)
      if (x != M1 && !(LPK == 16 && x == 1)) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    // the running maximum moves only when it is exceeded by more than 2^8: the probabilities stay far from fp32's limits either way
    const bool need = top > m + 8.f;
    if (__any_sync(0xffffffffu, need)) {
      const float to = need ? top : m, f = ex2(m - to);
      const float g = __shfl_xor_sync(0xffffffffu, f, M1);
      const float f1 = second ? g : f, f2 = second ? f : g;
      l *= f;
      m = to;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        o[0][k] = mul2(o[0][k], pk2(f1, f1));
        o[1][k] = mul2(o[1][k], pk2(f2, f2));
      }
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const float p = ex2(sc[v] - m);
      l += p;
      prob[row[v] * 2 + (second ? 1 : 0)] = p;
      if (TRACK && !(LPK == 16 && (lane & 1))) a.scores[((first + i) * 2 + (second ? 1 : 0)) * T + row[v]] = sc[v];
    }
    __syncwarp();
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const int vr = r * (32 / LPV) + lane / LPV;
      uint4 w = *reinterpret_cast<const uint4*>(tile + 2 * G::K_BYTES + (r * 32 + lane) * 16);
      if (valid < T && vr >= valid) w = make_uint4(0, 0, 0, 0);      // whatever lies there: 0 times it has to be 0
      const float2 p = reinterpret_cast<const float2*>(prob)[vr];
      const f32x2 p1 = pk2(p.x, p.x), p2 = pk2(p.y, p.y);
      const f32x2 v0 = widen(unpack2<BF>(w.x)), v1 = widen(unpack2<BF>(w.y)), v2 = widen(unpack2<BF>(w.z)), v3 = widen(unpack2<BF>(w.w));
      o[0][0] = fma2(v0, p1, o[0][0]); o[0][1] = fma2(v1, p1, o[0][1]); o[0][2] = fma2(v2, p1, o[0][2]); o[0][3] = fma2(v3, p1, o[0][3]);
      o[1][0] = fma2(v0, p2, o[1][0]); o[1][1] = fma2(v1, p2, o[1][1]); o[1][2] = fma2(v2, p2, o[1][2]); o[1][3] = fma2(v3, p2, o[1][3]);
    }
    __syncwarp();                              // the tile is read: its slot takes the next one
    if (i + SLOTS < count) {
      request(ahead, id, s, ahead.t == 0);
      if (i + SLOTS + 1 < count) {
        next(ahead);
        id = page_ids(ahead);
      }
    }
    if (cur.t == cur.n - 1 || i == count - 1) {
      // the stretch leaves this (sequence, head)
      float ov[2][8];
#pragma unroll
      for (int br = 0; br < 2; ++br)
#pragma unroll
        for (int k = 0; k < 4; ++k) up2(o[br][k], ov[br][2 * k], ov[br][2 * k + 1]);
#pragma unroll
      for (int x = LPV; x < 32; x <<= 1)
#pragma unroll
        for (int br = 0; br < 2; ++br)
#pragma unroll
          for (int k = 0; k < 8; ++k) ov[br][k] += __shfl_xor_sync(0xffffffffu, ov[br][k], x);
      float ls = l;
#pragma unroll
      for (int x = 1; x < 32; x <<= 1)
        if (x != M1 && !(LPK == 16 && x == 1)) ls += __shfl_xor_sync(0xffffffffu, ls, x);
      const float mo = __shfl_xor_sync(0xffffffffu, m, M1), lo = __shfl_xor_sync(0xffffffffu, ls, M1);
      const size_t at = size_t(worker) + size_t(cur.b) * a.c.h + cur.h;      // a piece's place: grows with every piece along the line
      if (lane == 0) a.stats[at] = make_float4(m, ls, mo, lo);
      if (lane < LPV) {
        float4* to = a.acc + at * D + lane * 2;
#pragma unroll
        for (int br = 0; br < 2; ++br) {
          to[br * (D / 2)] = make_float4(ov[br][0], ov[br][1], ov[br][2], ov[br][3]);
          to[br * (D / 2) + 1] = make_float4(ov[br][4], ov[br][5], ov[br][6], ov[br][7]);
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
struct Joined { float m1, l1, m2, l2; };       // maximum and sum of both branches over all pieces

// the pieces of tiles [u, u + n) of the line: workers w0 .. w1
__device__ __forceinline__ void piece_range(long long units, int workers, long long u, int n, int& w0, int& w1) {
  w0 = int(((u + 1) * workers - 1) / units);           // the last worker whose stretch begins at or before u
  w1 = int(((u + n) * workers - 1) / units);
}
__device__ __forceinline__ void join(float& m, float& l, float m2, float l2) {
  const float top = fmaxf(m, m2);
  l = l * ex2(m - top) + l2 * ex2(m2 - top);
  m = top;
}
__device__ __forceinline__ Joined join_stats(const float4* stats, int w0, int w1, int lane) {      // a whole warp
  Joined j{-3e38f, 0.f, -3e38f, 0.f};
  for (int w = w0 + lane; w <= w1; w += 32) {
    const float4 x = stats[w];
    join(j.m1, j.l1, x.x, x.y);
    join(j.m2, j.l2, x.z, x.w);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    join(j.m1, j.l1, __shfl_xor_sync(0xffffffffu, j.m1, o), __shfl_xor_sync(0xffffffffu, j.l1, o));
    join(j.m2, j.l2, __shfl_xor_sync(0xffffffffu, j.m2, o), __shfl_xor_sync(0xffffffffu, j.l2, o));
  }
  return j;
}

constexpr int JOIN_THREADS = 256;

template <int D, bool BF, bool TRACK>
__global__ void __launch_bounds__(JOIN_THREADS) diffattn_cache_join_kernel(const __grid_constant__ AttendArgs a) {
  constexpr int T = attend::Geo<D>::T;
  constexpr int GROUPS = JOIN_THREADS / D;     // pieces summed side by side: a thread has four of a piece's 4 D sums
  __shared__ float4 red[JOIN_THREADS];
  __shared__ float ssq[2 * D / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  griddep_wait();
  const int nb = a.c.b, heads = a.c.h;
  const long long units = (long long)a.prefix[nb] * heads;
  const int workers = int(min((long long)a.workers, units));
  const float lam = load_lambda(a.lambda_ptr, a.lambda_dtype);
  for (int bh = blockIdx.x; bh < nb * heads; bh += gridDim.x) {
    const int b = bh / heads, head = bh - b * heads;
    const int n = a.prefix[b + 1] - a.prefix[b];
    float out = 0.f;
    if (n > 0) {
      int w0, w1;
      piece_range(units, workers, (long long)a.prefix[b] * heads + (long long)head * n, n, w0, w1);
      const float4* stats = a.stats + bh;
      const Joined j = join_stats(stats, w0, w1, lane);
      const int col = threadIdx.x % D, group = threadIdx.x / D;
      const bool second = col >= D / 2;
      const float top = second ? j.m2 : j.m1;
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int w = w0 + group; w <= w1; w += GROUPS) {
        const float4 x = a.acc[(size_t(bh) + w) * D + col];
        const float c = ex2((second ? stats[w].z : stats[w].x) - top);
        sum.x += c * x.x; sum.y += c * x.y; sum.z += c * x.z; sum.w += c * x.w;
      }
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
    if (threadIdx.x < 2 * D) {
      if (a.gain) out *= a.gain[threadIdx.x];
      a.y[size_t(bh) * 2 * D + threadIdx.x] = from_float16b<BF>(out);
    }
    if (a.nk1 && threadIdx.x == 0) {
      const int len = a.length[b];
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
  }
  if constexpr (TRACK) {
    // the same line of tiles, cut into the warps of this grid
    const int takers = int(min((long long)gridDim.x * (JOIN_THREADS / 32), units));
    const int taker = warp * int(gridDim.x) + int(blockIdx.x);
    if (taker >= takers) return;
    long long u = stretch_begin(units, takers, taker);
    const long long end = stretch_begin(units, takers, taker + 1);
    TileWalk w = walk_at(a, a.prefix, a.length, u);
    while (u < end) {
      const int n = int(min((long long)(w.n - w.t), end - u));      // tiles of this (sequence, head)
      const int bh = w.b * heads + w.h;
      int w0, w1;
      piece_range(units, workers, u - w.t, w.n, w0, w1);
      const Joined j = join_stats(a.stats + bh, w0, w1, lane);
      const float c1 = 1.f / j.l1, c2 = lam / j.l2;
      float* to = a.c.weights + (size_t)bh * a.c.slots;
      for (int e = lane; e < n * T; e += 32) {
        int slot, in_page, valid;
        bool is_new;
        attend_tile<T>(a, w.t + e / T, w.n, w.len, slot, in_page, valid, is_new);
        const int row = e % T;
        if (row >= valid || slot + row >= a.c.slots) continue;
        const float* s = a.scores + (u + e / T) * 2 * T + row;
        const float x = fabsf(ex2(s[0] - j.m1) * c1 - ex2(s[T] - j.m2) * c2);
        to[slot + row] = is_new ? x : to[slot + row] + x;
      }
      u += n;
      w.t += n - 1;
      if (u < end) walk_next(a, a.prefix, a.length, w);
    }
  }
}

}  // namespace da
