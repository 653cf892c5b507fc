// Entry points of the key-value cache (include/diffattn.h): argument checks, workspace layout, launches.  Part of diffattn.cu.
#pragma once

namespace {

// How a tile of T rows is fetched: it runs on over the pages in boxes of r rows, r the common divisor of page size and T, each inside one page; or it
// stays inside its page, whose last tile is then not full.  Eight or more rows to a box cost nothing.  Fewer cost more requests: B8 H16
// N2048 D64 takes 29 us with pages of 8, 32 with 4, 55 with 1.  So tiles stay inside their pages where that wastes less, by these factors (D =
// 32 / 128, pages of 100: 33 / 32 us against 36 / 38).  A box's rows have to fill 128 bytes of shared memory; where they lie in the swizzle's
// pattern goes by their address.
struct TileShape { int rows, box_rows, tiles_per_page; };
int tile_rows(int D) { return D == 32 ? da::attend::Geo<32>::T : D == 64 ? da::attend::Geo<64>::T : da::attend::Geo<128>::T; }
TileShape tile_shape(const DiffAttnCacheParams* p) {
  const int T = tile_rows(p->D), row_bytes = p->D == 32 ? 64 : 128;
  int r = T;
  while (p->page_size % r) r /= 2;             // (T is a power of two)
  if (r >= 8) return {T, r, 0};
  const int per_page = (p->page_size - 1) / T + 1;
  const bool fits = 10ll * per_page * T <= (long long)p->page_size * (r == 4 ? 13 : r == 2 ? 15 : 20);
  if (fits || r * row_bytes < 128) return {T, T, per_page};
  return {T, r, 0};
}
// tiles of a full sequence
long long most_tiles(const DiffAttnCacheParams* p) {
  const TileShape s = tile_shape(p);
  const long long slots = (long long)p->max_pages * p->page_size;
  return (s.tiles_per_page ? (long long)p->max_pages * s.tiles_per_page : (slots + s.rows - 1) / s.rows) + 1;      // + 1: the new token
}

int attend_workers(const DiffAttnCacheParams* p) {
  return sm_count(p->device) * (p->D == 32 ? da::attend::Geo<32>::WARPS : p->D == 64 ? da::attend::Geo<64>::WARPS : da::attend::Geo<128>::WARPS);
}

struct AttendSpace {
  uint64_t prefix, length, position, stats, acc, scores, bytes;
};
AttendSpace attend_space(const DiffAttnCacheParams* p) {
  AttendSpace s;
  const uint64_t pieces = uint64_t(attend_workers(p)) + uint64_t(p->B) * p->H;
  uint64_t at = 0;
  auto take = [&](uint64_t& where, uint64_t bytes) { where = at; at += round256(bytes); };
  take(s.prefix, 4 * (uint64_t(p->B) + 2));
  take(s.length, 4 * uint64_t(p->B));
  take(s.position, 4 * uint64_t(p->B));
  take(s.stats, 16 * pieces);
  take(s.acc, 16 * pieces * p->D);
  take(s.scores, p->weights ? uint64_t(most_tiles(p)) * p->B * p->H * 2 * tile_rows(p->D) * 4 : 0);
  s.bytes = at;
  return s;
}
int evict_most(const DiffAttnCacheParams* p) { return std::min(p->keep, p->max_pages * p->page_size - p->keep); }

// The selecting kernel moves rows itself where they are few a CTA (one launch less), or there are three CTAs and more for every SM, whose moves and
// selections then overlap.  Appending a chunk and evicting as many tokens at D 64 with the second kernel / without, us: 512 moves, 16 CTAs
// 20 / 39, 128 CTAs 34 / 46; 256 moves, 160 CTAs 24 / 28, 256 CTAs 33 / 36, 384 CTAs 46.7 / 47.7; 1024 moves, 256 CTAs 104 / 133, 512 CTAs 194 / 192;
// 128 moves, 64 CTAs 16 / 20, 512 CTAs 34 / 31; 64 moves, 64 CTAs 15.2 / 14.5, 256 CTAs 14.8 / 14.5, 1024 CTAs 38 / 36.
bool evict_at_once(const DiffAttnCacheParams* p) { return evict_most(p) <= 64 || p->B * p->H >= 3 * sm_count(p->device); }
struct EvictSpace {
  uint64_t moves, bytes;
};
EvictSpace evict_space(const DiffAttnCacheParams* p) {
  const uint64_t bh = uint64_t(p->B) * p->H, most = uint64_t(evict_most(p));
  const bool at_once = evict_at_once(p);
  EvictSpace s;
  s.moves = at_once ? 0 : round256(4 * bh);
  s.bytes = s.moves + (at_once && most <= da::SELECT_LIST ? 0 : round256(8 * bh * most));
  return s;
}

bool aligned_to(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
bool good_stride(int64_t s, bool used) { return !used || (s > 0 && s % 8 == 0); }

// sizes alone, for the workspace query too
int check_cache_sizes(const DiffAttnCacheParams* p) {
  if (!p) return fail(DIFFATTN_ERR_NULL_PTR, "params is NULL");
  if (p->struct_size != sizeof(DiffAttnCacheParams))
    return fail(DIFFATTN_ERR_BAD_STRUCT, "struct_size %u != %zu", p->struct_size, sizeof(DiffAttnCacheParams));
  if (p->device < 0 || p->device >= kMaxDevices) return fail(DIFFATTN_ERR_BAD_SHAPE, "device ordinal %d outside [0,%d)", p->device, kMaxDevices);
  if (p->D != 32 && p->D != 64 && p->D != 128) return fail(DIFFATTN_ERR_UNSUPPORTED_D, "head dim %d is not compiled in (supported: 32, 64, 128)", p->D);
  if (p->B < 0 || p->H < 0 || p->B > da::attend::MAX_B || (long long)p->B * p->H > 65535)
    return fail(DIFFATTN_ERR_BAD_SHAPE, "B=%d H=%d: B <= %d and B*H <= 65535", p->B, p->H, da::attend::MAX_B);
  if (p->page_size <= 0 || p->num_pages <= 0 || p->max_pages <= 0)
    return fail(DIFFATTN_ERR_BAD_SHAPE, "page_size=%d num_pages=%d max_pages=%d must be positive", p->page_size, p->num_pages, p->max_pages);
  // In 32 bits the kernels add to a slot: a page, two tiles, a round of the selection's loads or runs.  To a tile: a round of all
  // shares that add weights, 4 x 64 tiles each.
  constexpr int slot_step = std::max(2 * da::SELECT_THREADS * da::SELECT_AHEAD, 31 * da::SELECT_THREADS), tile_step = 1 << 17;
  if ((long long)p->max_pages * p->page_size + std::max(p->page_size, slot_step) > INT32_MAX || most_tiles(p) + tile_step > INT32_MAX ||
      most_tiles(p) * std::max(p->B, 1) > INT32_MAX || most_tiles(p) * std::max(p->B, 1) * std::max(p->H, 1) > (1ll << 39))
    return fail(DIFFATTN_ERR_BAD_SHAPE, "max_pages=%d of %d slots: too long", p->max_pages, p->page_size);
  return DIFFATTN_OK;
}

// what every operation needs; 1: nothing to do
int check_cache(const DiffAttnCacheParams* p) {
  int rc = check_cache_sizes(p);
  if (rc) return rc;
  if (p->io_dtype != DIFFATTN_IO_F16 && p->io_dtype != DIFFATTN_IO_BF16) return fail(DIFFATTN_ERR_BAD_DTYPE, "io_dtype %d unknown", p->io_dtype);
  if (p->B == 0 || p->H == 0) return 1;
  const void* ptrs[] = {p->k1_pages, p->k2_pages, p->v_pages, p->page_table, p->lengths};
  const char* names[] = {"k1_pages", "k2_pages", "v_pages", "page_table", "lengths"};
  for (int i = 0; i < 5; ++i)
    if (!ptrs[i]) return fail(DIFFATTN_ERR_NULL_PTR, "%s is NULL", names[i]);
  for (int i = 0; i < 3; ++i)
    if (!aligned16(ptrs[i])) return fail(DIFFATTN_ERR_MISALIGNED, "%s is not 16-byte aligned", names[i]);
  const void* words[] = {p->page_table, p->lengths, p->next_position, p->positions, p->weights, p->counter};
  for (const void* w : words)
    if (!aligned_to(w, 4)) return fail(DIFFATTN_ERR_MISALIGNED, "page_table, lengths, next_position, positions, weights and counter must be 4-byte aligned");
  if ((p->positions != nullptr) != (p->next_position != nullptr)) return fail(DIFFATTN_ERR_NULL_PTR, "positions and next_position go together");
  const int64_t st[] = {p->kp_stride_page, p->kp_stride_head, p->kp_stride_slot, p->vp_stride_page, p->vp_stride_head, p->vp_stride_slot};
  const bool used[] = {p->num_pages > 1, p->H > 1, p->page_size > 1, p->num_pages > 1, p->H > 1, p->page_size > 1};
  for (int i = 0; i < 6; ++i)
    if (!good_stride(st[i], used[i]))
      return fail(DIFFATTN_ERR_BAD_STRIDE, "page stride %d = %lld must be a positive multiple of 8 elements", i, (long long)st[i]);
  for (int i = 0; i < 6; ++i)
    if (used[i] && (st[i] < (i < 3 ? p->D : 2 * p->D) || st[i] >= (1ll << 38)))
      return fail(DIFFATTN_ERR_BAD_STRIDE, "page stride %d = %lld is smaller than a row, or too large", i, (long long)st[i]);
  if (p->B > 1 && p->table_stride < p->max_pages) return fail(DIFFATTN_ERR_BAD_STRIDE, "table_stride %lld < max_pages", (long long)p->table_stride);
  return DIFFATTN_OK;
}

// k1, k2, v of new tokens
int check_tokens(const DiffAttnCacheParams* p, bool rows) {
  const void* ptrs[] = {p->k1, p->k2, p->v};
  const char* names[] = {"k1", "k2", "v"};
  for (int i = 0; i < 3; ++i) {
    if (!ptrs[i]) return fail(DIFFATTN_ERR_NULL_PTR, "%s is NULL", names[i]);
    if (!aligned16(ptrs[i])) return fail(DIFFATTN_ERR_MISALIGNED, "%s is not 16-byte aligned", names[i]);
  }
  if (!good_stride(p->k_stride_b, p->B > 1) || !good_stride(p->k_stride_h, p->H > 1) || !good_stride(p->k_stride_t, rows && p->T > 1) ||
      !good_stride(p->v_stride_b, p->B > 1) || !good_stride(p->v_stride_h, p->H > 1) || !good_stride(p->v_stride_t, rows && p->T > 1))
    return fail(DIFFATTN_ERR_BAD_STRIDE, "strides of k1, k2, v must be positive multiples of 8 elements");
  return DIFFATTN_OK;
}

int check_cache_workspace(const DiffAttnCacheParams* p, uint64_t need) {
  if (need == 0) return DIFFATTN_OK;
  if (!p->workspace || p->workspace_bytes < need)
    return fail(DIFFATTN_ERR_WORKSPACE, "workspace %llu bytes, need %llu", (unsigned long long)p->workspace_bytes, (unsigned long long)need);
  if (reinterpret_cast<uintptr_t>(p->workspace) & 255) return fail(DIFFATTN_ERR_MISALIGNED, "workspace not 256-byte aligned");
  return DIFFATTN_OK;
}

int cache_on_device(const DiffAttnCacheParams* p) {
  const void* ptrs[] = {p->k1_pages, p->k2_pages, p->v_pages, p->page_table, p->lengths, p->next_position, p->positions, p->weights, p->counter};
  const char* names[] = {"k1_pages", "k2_pages", "v_pages", "page_table", "lengths", "next_position", "positions", "weights", "counter"};
  for (int i = 0; i < 9; ++i)
    if (int rc = check_on_device(ptrs[i], p->device, names[i])) return rc;
  return DIFFATTN_OK;
}

int64_t pieces(int64_t stride, bool used) { return used ? stride / 8 : 0; }      // 16 bytes each; a dimension of one element has no stride

da::CacheArgs cache_args(const DiffAttnCacheParams* p) {
  da::CacheArgs c;
  c.b = p->B; c.h = p->H;
  c.page_size = p->page_size; c.max_pages = p->max_pages; c.num_pages = p->num_pages;
  c.slots = p->max_pages * p->page_size;
  c.page_magic = p->page_size > 1 ? uint32_t(((1ull << 32) + p->page_size - 1) / p->page_size) : 0u;
  c.page_table = p->page_table; c.table_stride = p->table_stride;
  c.lengths = p->lengths; c.counter = p->counter; c.next_position = p->next_position; c.positions = p->positions; c.weights = p->weights;
  c.k1 = static_cast<uint4*>(p->k1_pages); c.k2 = static_cast<uint4*>(p->k2_pages); c.v = static_cast<uint4*>(p->v_pages);
  c.k_page = pieces(p->kp_stride_page, p->num_pages > 1); c.k_head = pieces(p->kp_stride_head, p->H > 1); c.k_slot = pieces(p->kp_stride_slot, p->page_size > 1);
  c.v_page = pieces(p->vp_stride_page, p->num_pages > 1); c.v_head = pieces(p->vp_stride_head, p->H > 1); c.v_slot = pieces(p->vp_stride_slot, p->page_size > 1);
  return c;
}

template <int D, bool BF, bool TRACK>
int attend_launch(const DiffAttnCacheParams* p, da::AttendArgs& a) {
  int rc;
  CUtensorMap k1, k2, v;
  auto map = [&](CUtensorMap* m, const void* base, int width, int64_t page, int64_t head, int64_t slot, const char* what) {
    // (a dimension of one element needs a legal stride all the same)
    if (p->page_size == 1) slot = width;
    return make_map<BF>(m, base, width, p->page_size, p->H, p->num_pages, slot, head, page, a.box_rows, what, std::min(width, 64));
  };
  if ((rc = map(&k1, p->k1_pages, D, p->kp_stride_page, p->kp_stride_head, p->kp_stride_slot, "k1_pages"))) return rc;
  if ((rc = map(&k2, p->k2_pages, D, p->kp_stride_page, p->kp_stride_head, p->kp_stride_slot, "k2_pages"))) return rc;
  if ((rc = map(&v, p->v_pages, 2 * D, p->vp_stride_page, p->vp_stride_head, p->vp_stride_slot, "v_pages"))) return rc;
  auto kernel = da::diffattn_cache_attend_kernel<D, BF, TRACK>;
  constexpr int most = da::attend::Geo<D>::SMEM + 8 * da::attend::MAX_B;
  const int smem = da::attend::Geo<D>::SMEM + 8 * p->B;
  if ((rc = set_smem(kernel, most, p->device))) return rc;
  const cudaStream_t stream = static_cast<cudaStream_t>(p->stream);
  const int sms = sm_count(p->device);
  if ((rc = launch(kernel, dim3(sms), da::attend::Geo<D>::THREADS, smem, stream, true, k1, k2, v, a))) return rc;
  // How many pieces a (sequence, head) has goes by how many of them share the workers, and by its tiles.  Whole calls at D 64 without weights, us, joined
  // by 1024 threads / 256 / a warp: 65 pieces (B1 H16 N8192) 19.5 / 22.0 / 38; 40 (H26 N4096) 17.8 / 18.4 / 29; 22 (B2 H24) 24.6 / 24.0 / 31; 16 (B4
  // H16) 30.0 / 29.0 / 34; 4 (B16 H16 N1024) 34.2 / 29.4 / 30.8; 3 (340 heads) 43.5 / 36.8 / 36.9; 2 (384 heads) 47.3 / 40.5 / 40.1; 1 (B64 H16) 110 / 90 / 88.
  // (By the batch's capacity, not by the sequences in use, which the host does not know: few long ones in a large batch are joined slowly.)
  const int bh = p->B * p->H;
  const long long pieces = std::min((long long)a.workers / bh, most_tiles(p));
  auto weights = [&](int blocks) { return TRACK ? bh * ((blocks + bh - 1) / bh) : 0; };
  a.join_blocks = bh;
  if (pieces > 40) return launch(da::diffattn_cache_join_kernel<D, 1024, BF, TRACK>, dim3(bh + weights(sms)), 1024, 0, stream, true, a);
  if (pieces > 2) return launch(da::diffattn_cache_join_kernel<D, 256, BF, TRACK>, dim3(bh + weights(2 * sms)), 256, 0, stream, true, a);
  a.join_blocks = (bh + da::JOIN_FEW / 32 - 1) / (da::JOIN_FEW / 32);
  return launch(da::diffattn_cache_join_few_kernel<D, BF, TRACK>, dim3(a.join_blocks + weights(2 * sms)), da::JOIN_FEW, 0, stream, true, a);
}
template <int D>
int attend_launch(const DiffAttnCacheParams* p, da::AttendArgs& a) {
  const bool bf = p->io_dtype == DIFFATTN_IO_BF16;
  if (p->weights) return bf ? attend_launch<D, true, true>(p, a) : attend_launch<D, false, true>(p, a);
  return bf ? attend_launch<D, true, false>(p, a) : attend_launch<D, false, false>(p, a);
}

template <int D>
int evict_launch(const DiffAttnCacheParams* p, const da::EvictArgs& a) {
  int rc;
  const cudaStream_t stream = static_cast<cudaStream_t>(p->stream);
  const int bh = p->B * p->H;
  if ((rc = set_smem(da::diffattn_cache_select_kernel<D>, da::SELECT_MOST_KEYS * 4, p->device))) return rc;
  if ((rc = launch(da::diffattn_cache_select_kernel<D>, dim3(bh), da::SELECT_THREADS, a.cached_keys ? a.c.slots * 4 : 0, stream, true, a))) return rc;
  if (a.moves_at_once) return DIFFATTN_OK;
  // as many CTAs as the SMs hold, spread over the (sequence, head)s, but no more than there can be moves for
  const int rows = da::MovePlaces<D, da::MOVE_THREADS>::BLOCK;
  const int wide = std::max(1, std::min((a.most + rows - 1) / rows, (sm_count(p->device) * 8 + bh - 1) / bh));
  return launch(da::diffattn_cache_move_kernel<D>, dim3(wide, bh), da::MOVE_THREADS, 0, stream, true, a);
}

}  // namespace

extern "C" {

uint64_t diffattn_cache_workspace_bytes(const DiffAttnCacheParams* p, int32_t operation) {
  if (check_cache_sizes(p) || p->B == 0 || p->H == 0) return 0;
  if (operation == DIFFATTN_CACHE_ATTEND) return attend_space(p).bytes;
  if (operation == DIFFATTN_CACHE_EVICT) {
    if (p->keep < 1 || p->keep > p->max_pages * p->page_size) return 0;
    return evict_space(p).bytes;
  }
  return 0;
}

int diffattn_cache_append(const DiffAttnCacheParams* p) {
  int rc = check_cache(p);
  if (rc) return rc < 0 ? rc : DIFFATTN_OK;
  if (p->T < 0 || p->T > INT32_MAX - 1024) return fail(DIFFATTN_ERR_BAD_SHAPE, "T=%d", p->T);
  if (p->T == 0) return DIFFATTN_OK;
  if ((rc = check_tokens(p, true))) return rc;
  if (!p->counter) return fail(DIFFATTN_ERR_NULL_PTR, "counter is NULL");
  if (!aligned_to(p->counts, 4)) return fail(DIFFATTN_ERR_MISALIGNED, "counts is not 4-byte aligned");
  DeviceGuard guard;
  if ((rc = guard.enter(p->device))) return rc;
  if ((rc = cache_on_device(p))) return rc;
  const void* ptrs[] = {p->k1, p->k2, p->v, p->counts};
  const char* names[] = {"k1", "k2", "v", "counts"};
  for (int i = 0; i < 4; ++i)
    if ((rc = check_on_device(ptrs[i], p->device, names[i]))) return rc;
  da::CacheAppendArgs a;
  a.c = cache_args(p);
  a.t = p->T; a.counts = p->counts;
  a.k1 = static_cast<const uint4*>(p->k1); a.k2 = static_cast<const uint4*>(p->k2); a.v = static_cast<const uint4*>(p->v);
  a.k_b = pieces(p->k_stride_b, p->B > 1); a.k_h = pieces(p->k_stride_h, p->H > 1); a.k_t = pieces(p->k_stride_t, p->T > 1);
  a.v_b = pieces(p->v_stride_b, p->B > 1); a.v_h = pieces(p->v_stride_h, p->H > 1); a.v_t = pieces(p->v_stride_t, p->T > 1);
  const cudaStream_t stream = static_cast<cudaStream_t>(p->stream);
  const int rows = da::APPEND_THREADS / (p->D / 2) * da::APPEND_UNROLL;
  const dim3 grid((p->T + rows - 1) / rows, p->B * p->H);
  auto kernel = p->D == 32 ? da::diffattn_cache_append_kernel<32> : p->D == 64 ? da::diffattn_cache_append_kernel<64> : da::diffattn_cache_append_kernel<128>;
  a.take_tickets = (long long)grid.x * grid.y <= 4 * sm_count(p->device) ? 1 : 0;
  if ((rc = launch(kernel, grid, da::APPEND_THREADS, 0, stream, true, a)) || a.take_tickets) return rc;
  return launch(da::diffattn_cache_advance_kernel, dim3((p->B + da::APPEND_THREADS - 1) / da::APPEND_THREADS), da::APPEND_THREADS, 0, stream, true, a);
}

int diffattn_cache_reset(int32_t device, void* stream, int32_t B, int32_t* lengths, int32_t* next_position) {
  if (B < 0) return fail(DIFFATTN_ERR_BAD_SHAPE, "B=%d", B);
  if (B == 0) return DIFFATTN_OK;
  if (!lengths) return fail(DIFFATTN_ERR_NULL_PTR, "lengths is NULL");
  if (!aligned_to(lengths, 4) || !aligned_to(next_position, 4)) return fail(DIFFATTN_ERR_MISALIGNED, "lengths and next_position must be 4-byte aligned");
  DeviceGuard guard;
  int rc = guard.enter(device);
  if (rc) return rc;
  if ((rc = check_on_device(lengths, device, "lengths")) || (rc = check_on_device(next_position, device, "next_position"))) return rc;
  return launch(da::diffattn_cache_reset_kernel, dim3((B + da::APPEND_THREADS - 1) / da::APPEND_THREADS), da::APPEND_THREADS, 0,
                static_cast<cudaStream_t>(stream), true, lengths, next_position, B);
}

int diffattn_cache_attend(const DiffAttnCacheParams* p) {
  int rc = check_cache(p);
  if (rc) return rc < 0 ? rc : DIFFATTN_OK;
  const void* ptrs[] = {p->q1, p->q2, p->lambda_scale, p->y};
  const char* names[] = {"q1", "q2", "lambda_scale", "y"};
  for (int i = 0; i < 4; ++i)
    if (!ptrs[i]) return fail(DIFFATTN_ERR_NULL_PTR, "%s is NULL", names[i]);
  if (!aligned16(p->q1) || !aligned16(p->q2) || !aligned16(p->y)) return fail(DIFFATTN_ERR_MISALIGNED, "q1/q2/y not 16-byte aligned");
  if (!good_stride(p->q_stride_b, p->B > 1) || !good_stride(p->q_stride_h, p->H > 1))
    return fail(DIFFATTN_ERR_BAD_STRIDE, "strides of q1, q2 must be positive multiples of 8 elements");
  if (p->lambda_dtype != DIFFATTN_LAMBDA_F16 && p->lambda_dtype != DIFFATTN_LAMBDA_F32 && p->lambda_dtype != DIFFATTN_LAMBDA_BF16)
    return fail(DIFFATTN_ERR_BAD_DTYPE, "lambda_dtype %d unknown", p->lambda_dtype);
  if (!aligned_to(p->lambda_scale, p->lambda_dtype == DIFFATTN_LAMBDA_F32 ? 4 : 2) || !aligned_to(p->gain, 4))
    return fail(DIFFATTN_ERR_MISALIGNED, "lambda_scale or gain is not aligned to its type");
  const bool token = p->k1 || p->k2 || p->v;
  if (token && (rc = check_tokens(p, false))) return rc;
  if (!aligned_to(p->counts, 4)) return fail(DIFFATTN_ERR_MISALIGNED, "counts is not 4-byte aligned");
  DeviceGuard guard;
  if ((rc = guard.enter(p->device))) return rc;
  const AttendSpace space = attend_space(p);
  if ((rc = check_cache_workspace(p, space.bytes))) return rc;
  if ((rc = cache_on_device(p))) return rc;
  const void* dp[] = {p->q1, p->q2, p->lambda_scale, p->y, p->k1, p->k2, p->v, p->counts, p->gain, p->workspace};
  const char* dn[] = {"q1", "q2", "lambda_scale", "y", "k1", "k2", "v", "counts", "gain", "workspace"};
  for (int i = 0; i < 10; ++i)
    if ((rc = check_on_device(dp[i], p->device, dn[i]))) return rc;
  da::AttendArgs a;
  a.c = cache_args(p);
  a.q1 = static_cast<const uint4*>(p->q1); a.q2 = static_cast<const uint4*>(p->q2);
  a.q_b = pieces(p->q_stride_b, p->B > 1); a.q_h = pieces(p->q_stride_h, p->H > 1);
  a.nk1 = static_cast<const uint4*>(p->k1); a.nk2 = static_cast<const uint4*>(p->k2); a.nv = static_cast<const uint4*>(p->v);
  a.counts = p->counts;
  a.nk_b = pieces(p->k_stride_b, p->B > 1); a.nk_h = pieces(p->k_stride_h, p->H > 1);
  a.nv_b = pieces(p->v_stride_b, p->B > 1); a.nv_h = pieces(p->v_stride_h, p->H > 1);
  a.scale_log2 = p->sm_scale * 1.4426950408889634f;
  a.lambda_ptr = p->lambda_scale; a.lambda_dtype = p->lambda_dtype; a.rms_norm = p->rms_norm;
  a.out_scale = 1.f - p->lambda_init; a.eps = p->eps;
  a.gain = p->gain; a.y = static_cast<__half*>(p->y);
  const TileShape shape = tile_shape(p);
  a.box_rows = shape.box_rows; a.tiles_per_page = shape.tiles_per_page;
  a.tiles_magic = shape.tiles_per_page > 1 ? uint32_t(((1ull << 32) + shape.tiles_per_page - 1) / shape.tiles_per_page) : 0u;
  a.workers = attend_workers(p);
  uint8_t* ws = static_cast<uint8_t*>(p->workspace);
  a.prefix = reinterpret_cast<int*>(ws + space.prefix);
  a.length = reinterpret_cast<int*>(ws + space.length);
  a.position = reinterpret_cast<int*>(ws + space.position);
  a.stats = reinterpret_cast<float4*>(ws + space.stats);
  a.acc = reinterpret_cast<float4*>(ws + space.acc);
  a.scores = reinterpret_cast<float*>(ws + space.scores);
  return p->D == 32 ? attend_launch<32>(p, a) : p->D == 64 ? attend_launch<64>(p, a) : attend_launch<128>(p, a);
}

int diffattn_cache_evict(const DiffAttnCacheParams* p) {
  int rc = check_cache(p);
  if (rc < 0) return rc;
  if (p->keep < 1 || p->keep > p->max_pages * p->page_size || p->recent < 0 || p->recent > p->keep)
    return fail(DIFFATTN_ERR_BAD_SHAPE, "keep=%d must lie in [1, %d], recent=%d in [0, keep]", p->keep, p->max_pages * p->page_size, p->recent);
  if (rc == 1) return DIFFATTN_OK;
  if (!p->positions || !p->counter) return fail(DIFFATTN_ERR_NULL_PTR, "evict needs positions, next_position and counter");
  DeviceGuard guard;
  if ((rc = guard.enter(p->device))) return rc;
  const EvictSpace space = evict_space(p);
  if ((rc = check_cache_workspace(p, space.bytes))) return rc;
  if ((rc = cache_on_device(p))) return rc;
  if (space.bytes && (rc = check_on_device(p->workspace, p->device, "workspace"))) return rc;
  da::EvictArgs a;
  a.c = cache_args(p);
  a.keep = p->keep; a.recent = p->recent; a.most = evict_most(p);
  a.count = static_cast<int*>(p->workspace);
  a.moves = reinterpret_cast<int2*>(static_cast<uint8_t*>(p->workspace) + space.moves);
  a.cached_keys = a.c.slots <= da::SELECT_MOST_KEYS ? 1 : 0;
  a.moves_at_once = evict_at_once(p) ? 1 : 0;
  return p->D == 32 ? evict_launch<32>(p, a) : p->D == 64 ? evict_launch<64>(p, a) : evict_launch<128>(p, a);
}

}  // extern "C"
