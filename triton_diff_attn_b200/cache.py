"""Key-value cache of differential attention for generation: `DiffAttnCache`.

The reference trains only; what its layer needs to answer with, one token at a time, is here: storing the tokens' K1, K2 and V in pages,
attention of one new token over them, and eviction of the tokens that gather the least attention.  Host side only, as layers.py:
argument checks, output allocation through torch and one call into the C ABI per method (`diffattn_cache_append`, `_attend`,
`_evict`).  No method synchronises the host with the device or reads a length there, so all of them can be captured in a CUDA graph.
"""
from __future__ import annotations

import ctypes as C
import math
import operator

import torch
from torch.autograd import forward_ad

from . import _lib
from .layers import _IO_DTYPES, _LAMBDA_DTYPES, EPS


def _addressable(t) -> bool:
    """Rows the kernels can read as they lie: unit stride in the last dimension, the other strides positive multiples of 8 elements
    (a dimension of one element has none), base pointer 16-byte aligned."""
    return (t.data_ptr() % 16 == 0 and t.stride(-1) == 1
            and all(n <= 1 or (s > 0 and s % 8 == 0) for n, s in zip(t.shape[:-1], t.stride()[:-1])))


def _rows(t):
    """`t` and its strides where its rows can be read as they lie, else a copy."""
    sb, sh, st, sd = strides = t.stride()
    if sd == 1 and sb > 0 and sh > 0 and st > 0 and not (sb | sh | st) % 8 and not t.data_ptr() % 16:
        return t, strides          # (the common case: what the general rule would say)
    if not _addressable(t):
        t = t.clone(memory_format=torch.contiguous_format)
    return t, t.stride()


def _pair(a, b):
    """Two tensors of one shape with the same strides, and these; copied where they differ or cannot be addressed."""
    a, sa = _rows(a)
    b, sb = _rows(b)
    if sa != sb:
        a, b = a.clone(memory_format=torch.contiguous_format), b.clone(memory_format=torch.contiguous_format)
        sa = a.stride()
    return a, b, sa


def _refuse_tangents(**tensors):
    """Inside a level of forward-mode differentiation (the caller looks for one first): what comes out here would have lost a tangent."""
    for name, t in tensors.items():
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{name} has a forward-mode tangent, and the cache has no derivatives")


class DiffAttnCache:
    """A paged cache of K1, K2 and V of `batch` sequences.

    `DiffAttnCache(batch, heads, head_dim, max_tokens)` allocates pages for `max_tokens` tokens of every sequence.  `from_tensors` takes a
    pool and a page table of the caller's own, for pages that are handed out as sequences grow, or that sequences share.

    k1_pages, k2_pages  [num_pages, heads, page_size, D], v_pages [num_pages, heads, page_size, 2D]: fp16 or bf16, any strides that are
                        multiples of 8 elements (so also the [num_pages, page_size, heads, D] storage viewed like this).
    page_table          int32 [batch, max_pages]: the page of each sequence's slots [i * page_size, (i + 1) * page_size).
    lengths             int32 [batch]: tokens in the cache, in slots 0 .. length - 1; 0 is a sequence that is not in use.
    positions           int32 [batch, heads, slots]: the position of the token in each slot (an eviction keeps other tokens in each head).
    next_position       int32 [batch]: tokens the sequence has had.
    weights             float32 [batch, heads, slots] or None: the attention weight each token has gathered (`attend`).

    All of these are the caller's to read and to write (in place) between calls (a new page, a sequence that starts anew: `lengths[b] = 0`,
    `next_position[b] = 0`).  They stay on the device and are not checked on the host: a length outside [0, slots], a page outside the pool or
    a token that finds its sequence full touches no memory it should not, leaves that call's results undefined and makes
    `device_status()` raise.  Slots that a call writes must belong to one sequence.  Calls on one cache that write it (all but
    `attend` without a token and without weights) have to be ordered, as any writes to one tensor; that goes for replays of captured calls too."""

    def __init__(self, batch: int, heads: int, head_dim: int, max_tokens: int, *, page_size: int = 64, track_weights: bool = False,
                 dtype=torch.float16, device=None):
        if min(batch, heads) < 0 or max_tokens < 1 or page_size < 1:
            raise ValueError(f"batch={batch}, heads={heads} must not be negative, max_tokens={max_tokens} and page_size={page_size} be positive")
        device = torch.device("cuda" if device is None else device)
        max_pages = -(-max_tokens // page_size)
        num_pages = max(1, batch * max_pages)
        k1, k2 = (torch.empty(num_pages, heads, page_size, head_dim, dtype=dtype, device=device) for _ in range(2))
        v = torch.empty(num_pages, heads, page_size, 2 * head_dim, dtype=dtype, device=device)
        table = torch.arange(batch * max_pages, dtype=torch.int32, device=device).view(batch, max_pages)
        zeros = lambda *shape, dt=torch.int32: torch.zeros(shape, dtype=dt, device=device)
        slots = max_pages * page_size
        self._take(k1, k2, v, table, zeros(batch), zeros(batch, heads, slots), zeros(batch),
                   zeros(batch, heads, slots, dt=torch.float32) if track_weights else None)

    @classmethod
    def from_tensors(cls, k1_pages, k2_pages, v_pages, page_table, lengths, *, positions=None, next_position=None, weights=None):
        """A cache over tensors that the caller made.  They are used in place, never copied.  Without positions and next_position (both
        or neither) `evict` is refused."""
        cache = cls.__new__(cls)
        cache._take(k1_pages, k2_pages, v_pages, page_table, lengths, positions, next_position, weights)
        return cache

    def _take(self, k1_pages, k2_pages, v_pages, page_table, lengths, positions, next_position, weights):
        pools = (("k1_pages", k1_pages), ("k2_pages", k2_pages), ("v_pages", v_pages))
        for name, t in pools + (("page_table", page_table), ("lengths", lengths)):
            if not torch.is_tensor(t):
                raise TypeError(f"{name} must be a tensor")
            if not t.is_cuda:
                raise RuntimeError(f"{name} must be a CUDA tensor: the cache has no CPU path")
        if not _lib.lib.has_cache:
            raise RuntimeError("this build of libdiffattn has no cache entry points")
        for name, t in pools:
            if t.dtype not in _IO_DTYPES or t.dtype != k1_pages.dtype:
                raise ValueError(f"{name} is {t.dtype}: the pages must be float16 or bfloat16, all three alike")
            if t.dim() != 4:
                raise ValueError(f"{name} must be [num_pages, heads, page_size, D]")
            if not _addressable(t):
                raise ValueError(f"{name}: last dimension contiguous, strides positive multiples of 8 elements, base 16-byte aligned "
                                 f"(got strides {t.stride()}); pages are used in place and not copied")
        pages, heads, page_size, d = k1_pages.shape
        if not _lib.lib.diffattn_supports(d, 0):
            raise ValueError(f"head dim {d} is not compiled in (supported: 32, 64, 128)")
        if k2_pages.shape != k1_pages.shape or k2_pages.stride() != k1_pages.stride():
            raise ValueError("k2_pages must have the shape and strides of k1_pages")
        if tuple(v_pages.shape) != (pages, heads, page_size, 2 * d):
            raise ValueError(f"v_pages shape {tuple(v_pages.shape)} != {(pages, heads, page_size, 2 * d)}")
        if page_table.dim() != 2 or page_table.dtype != torch.int32 or page_table.shape[1] < 1 or (page_table.shape[1] > 1 and page_table.stride(1) != 1):
            raise ValueError("page_table must be int32 [batch, max_pages] with contiguous rows")
        batch, max_pages = page_table.shape
        if batch > 1 and page_table.stride(0) < max_pages:
            raise ValueError("the rows of page_table must not overlap")
        slots = max_pages * page_size
        if max(slots, pages, heads, batch) >= 2 ** 31:      # (the library's fields; it has closer limits of its own)
            raise ValueError(f"{batch} sequences of {max_pages} pages of {page_size} slots, {pages} pages, {heads} heads: too long for 32 bits")
        if (positions is None) != (next_position is None):
            raise ValueError("positions and next_position go together")
        spans = []
        for name, t, shape, dtype in (("lengths", lengths, (batch,), torch.int32), ("next_position", next_position, (batch,), torch.int32),
                                      ("positions", positions, (batch, heads, slots), torch.int32),
                                      ("weights", weights, (batch, heads, slots), torch.float32)):
            if t is None:
                continue
            if not torch.is_tensor(t):
                raise TypeError(f"{name} must be a tensor")
            if t.dtype != dtype or tuple(t.shape) != shape or not t.is_contiguous():
                raise ValueError(f"{name} must be {dtype} {shape}, contiguous")
            if t.is_cuda and t.numel():
                spans.append((t.data_ptr(), t.data_ptr() + 4 * t.numel(), name))
        spans.sort()
        for (_, end, a), (start, _, b) in zip(spans, spans[1:]):
            if start < end:
                raise ValueError(f"{a} and {b} share memory")
        device = k1_pages.device
        for name, t in pools + (("page_table", page_table), ("lengths", lengths), ("positions", positions), ("next_position", next_position),
                                ("weights", weights)):
            if t is not None and t.device != device:
                raise RuntimeError(f"{name} is on {t.device}, k1_pages on {device}")
            if t is not None and t.requires_grad:
                raise ValueError(f"{name} requires a gradient: the cache has no backward pass")
            if forward_ad._current_level >= 0:
                _refuse_tangents(**{name: t})
        self._k1_pages, self._k2_pages, self._v_pages, self._page_table = k1_pages, k2_pages, v_pages, page_table
        self._lengths, self._positions, self._next_position, self._weights = lengths, positions, next_position, weights
        # What append and evict count their CTAs with: 0 between calls, every one of them leaves it so.  Made in a capture it would be 0
        # in that graph's replays only, so a cache made there takes a new one for every call.
        with torch.cuda.device(device):
            self._counter = None if torch.cuda.is_current_stream_capturing() else lengths.new_zeros(1)
        if self._counter is not None:
            torch.cuda.current_stream(device).synchronize()      # (the first call may come on another stream)
        self._shape = (batch, heads, d)
        self._device, self._index, self._dtype = device, k1_pages.get_device(), k1_pages.dtype
        p = _lib.DiffAttnCacheParams()
        p.struct_size = C.sizeof(p)
        p.device = k1_pages.get_device()
        p.B, p.H, p.D = batch, heads, d
        p.io_dtype = _lib.IO_BF16 if k1_pages.dtype == torch.bfloat16 else _lib.IO_F16
        p.page_size, p.num_pages, p.max_pages = page_size, pages, max_pages
        p.kp_stride_page, p.kp_stride_head, p.kp_stride_slot, _ = k1_pages.stride()
        p.vp_stride_page, p.vp_stride_head, p.vp_stride_slot, _ = v_pages.stride()
        p.table_stride = page_table.stride(0)
        p.sm_scale, p.eps = 1.0 / math.sqrt(d), EPS
        # the tensors stay where they are for the cache's life (and their memory with it, whatever becomes of the tensor objects)
        p.k1_pages, p.k2_pages, p.v_pages, p.page_table, p.lengths = (t.data_ptr() for t in (k1_pages, k2_pages, v_pages, page_table, lengths))
        if self._counter is not None:
            p.counter = self._counter.data_ptr()
        if positions is not None:
            p.positions, p.next_position = positions.data_ptr(), next_position.data_ptr()
        if weights is not None:
            p.weights = weights.data_ptr()
        self._memory = [t.untyped_storage() for t in (k1_pages, k2_pages, v_pages, page_table, lengths, positions, next_position, weights) if t is not None]
        self._y = k1_pages.new_empty((batch, heads, 1, 2 * d))      # (a pattern: empty_like is the cheapest way to a new one)
        self._sizes = p
        _lib.check(_lib.lib.diffattn_cache_append(p), "diffattn_cache_append")      # (T = 0: the checks of sizes and strides alone)
        self._attend_bytes = int(_lib.lib.diffattn_cache_workspace_bytes(self._params(), _lib.CACHE_ATTEND))

    k1_pages = property(lambda self: self._k1_pages)
    k2_pages = property(lambda self: self._k2_pages)
    v_pages = property(lambda self: self._v_pages)
    page_table = property(lambda self: self._page_table)
    lengths = property(lambda self: self._lengths)
    positions = property(lambda self: self._positions)
    next_position = property(lambda self: self._next_position)
    weights = property(lambda self: self._weights)
    slots = property(lambda self: self._sizes.max_pages * self._sizes.page_size, doc="tokens that one sequence can hold")

    def _params(self):
        p = _lib.DiffAttnCacheParams.from_buffer_copy(self._sizes)      # a copy per call: calls of several threads do not share it
        p.stream = torch._C._cuda_getCurrentRawStream(self._index)
        return p

    def _check(self, name, t, rows, width):
        batch, heads, _ = self._shape
        if (isinstance(t, torch.Tensor) and t.dtype is self._dtype and t.get_device() == self._index and t.shape == (batch, heads, rows, width)
                and not t.requires_grad):
            return
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a tensor")
        if t.device != self._device:
            raise RuntimeError(f"{name} is on {t.device}, the cache on {self._device}")
        if t.dtype != self._dtype:
            raise ValueError(f"{name} is {t.dtype}, the cache {self._dtype}")
        if tuple(t.shape) != (batch, heads, rows, width):
            raise ValueError(f"{name} shape {tuple(t.shape)} != {(batch, heads, rows, width)}")
        if t.requires_grad and torch.is_grad_enabled():
            raise RuntimeError(f"{name} requires a gradient, and the cache has no backward pass: call it under torch.no_grad()")

    def _tokens(self, p, k1, k2, v, rows):
        d = self._shape[2]
        self._check("k1", k1, rows, d)
        self._check("k2", k2, rows, d)
        self._check("v", v, rows, 2 * d)
        if forward_ad._current_level >= 0:
            _refuse_tangents(k1=k1, k2=k2, v=v)
        k1, k2, sk = _pair(k1, k2)
        v, sv = _rows(v)
        p.k1, p.k2, p.v = k1.data_ptr(), k2.data_ptr(), v.data_ptr()
        p.k_stride_b, p.k_stride_h, p.k_stride_t, _ = sk
        p.v_stride_b, p.v_stride_h, p.v_stride_t, _ = sv
        return k1, k2, v

    def _counts(self, p, counts, most):
        if not isinstance(counts, torch.Tensor):
            raise TypeError("counts must be a tensor")
        if counts.get_device() != self._index:
            raise RuntimeError(f"counts is on {counts.device}, the cache on {self._device}")
        if counts.dtype not in (torch.int32, torch.int64) or tuple(counts.shape) != (self._shape[0],):
            raise ValueError(f"counts must be int32 or int64 of shape {(self._shape[0],)}")
        if counts.dtype is not torch.int32:
            counts = counts.clamp(0, most).to(torch.int32)      # (not the lowest 32 bits of whatever it is)
        counts = counts.contiguous()
        p.counts = counts.data_ptr()
        return counts

    def _count_with(self, p):
        """The counter of a call that writes, where the cache has none of its own; to be kept until the call is enqueued."""
        if self._counter is not None:
            return None
        counter = self._lengths.new_zeros(1)
        p.counter = counter.data_ptr()
        return counter

    def _workspace(self, p, nbytes):
        ws = self._lengths.new_empty(max(nbytes, 256) // 4)
        p.workspace, p.workspace_bytes = ws.data_ptr(), nbytes
        return ws

    def reset(self) -> None:
        """Every sequence starts anew: nothing is cached."""
        _lib.check(_lib.lib.diffattn_cache_reset(self._index, torch._C._cuda_getCurrentRawStream(self._index), self._shape[0], self._sizes.lengths,
                                                 self._sizes.next_position), "diffattn_cache_reset")

    def append(self, k1, k2, v, counts=None) -> None:
        """Stores the tokens k1, k2 [B, H, T, D], v [B, H, T, 2D] behind each sequence's last one.  `counts` (an integer tensor [B]): sequence b
        gets the first counts[b] of them, all where there are not so many (a padded batch; what lies behind is not read).
        Their weights start at 0, and only `attend` adds to them."""
        if not isinstance(k1, torch.Tensor) or k1.dim() != 4:
            raise (ValueError if isinstance(k1, torch.Tensor) else TypeError)("k1 must be a tensor [B, H, T, D]")
        p = self._params()
        p.T = k1.shape[2]
        keep = self._tokens(p, k1, k2, v, p.T)  # noqa: F841  (copies stay until the call is enqueued)
        if counts is not None:
            counts = self._counts(p, counts, p.T)
        counter = self._count_with(p)  # noqa: F841
        _lib.check(_lib.lib.diffattn_cache_append(p), "diffattn_cache_append")

    def attend(self, q1, q2, lambda_scale, lambda_init: float = 0.8, rms_norm: bool = False, gain=None, k1=None, k2=None, v=None,
               counts=None):
        """Differential attention of one query per sequence and head, q1, q2 [B, H, 1, D], over the sequence's tokens; returns [B, H, 1, 2D].
        lambda_scale, lambda_init, rms_norm and gain as in `MultiheadDiffAttnKernel`, scale 1/sqrt(D).  A sequence without tokens gives 0.

        With k1, k2 [B, H, 1, D] and v [B, H, 1, 2D] (all or none) that token is stored first, in the same launches, and takes part: the
        step of a generation.  Without them nothing is stored: a query over an encoder's states, say, that `append` put there.
        `counts` (an integer tensor [B]): only sequences with a positive one get their token; the others' state stays as it is, so the unused rows
        of a batch (length 0, no pages) take part in nothing.

        A cache with `weights` adds |P1 - lambda P2| to each token's."""
        d = self._shape[2]
        self._check("q1", q1, 1, d)
        self._check("q2", q2, 1, d)
        lam = lambda_scale
        if not (isinstance(lam, torch.Tensor) and lam.get_device() == self._index and lam.numel() == 1 and lam.dtype in _LAMBDA_DTYPES):
            self._refuse_lambda(lam)
        if gain is not None:
            if not isinstance(gain, torch.Tensor) or gain.get_device() != self._index or gain.shape != (2 * d,) or not gain.is_floating_point():
                raise ValueError("gain must be a floating-point tensor of shape [2*D] on the cache's device")
        if (lam.requires_grad or (gain is not None and gain.requires_grad)) and torch.is_grad_enabled():
            raise RuntimeError("lambda_scale or gain requires a gradient, and the cache has no backward pass: call it under torch.no_grad()")
        if forward_ad._current_level >= 0:
            _refuse_tangents(q1=q1, q2=q2, lambda_scale=lam, gain=gain)
        p = self._params()
        if k1 is not None or k2 is not None or v is not None:
            keep = self._tokens(p, k1, k2, v, 1)  # noqa: F841  (copies stay until the call is enqueued)
            if counts is not None:
                counts = self._counts(p, counts, 1)
        elif counts is not None:
            raise ValueError("counts goes with a token: k1, k2 and v are missing")
        q1, q2, sq = _pair(q1, q2)
        p.q1, p.q2, p.q_stride_b, p.q_stride_h = q1.data_ptr(), q2.data_ptr(), sq[0], sq[1]
        p.lambda_scale, p.lambda_dtype = lam.data_ptr(), _LAMBDA_DTYPES[lam.dtype]
        p.rms_norm, p.lambda_init = 1 if rms_norm else 0, float(lambda_init)
        if gain is not None:
            if gain.dtype is not torch.float32 or gain.stride(0) != 1:
                gain = gain.detach().to(torch.float32).contiguous()
            p.gain = gain.data_ptr()
        y = torch.empty_like(self._y)
        p.y = y.data_ptr()
        ws = self._workspace(p, self._attend_bytes)  # noqa: F841
        _lib.check(_lib.lib.diffattn_cache_attend(p), "diffattn_cache_attend")
        return y

    def _refuse_lambda(self, lam):
        if not isinstance(lam, torch.Tensor):
            raise TypeError("lambda_scale must be a 1-element CUDA tensor")
        if lam.numel() != 1 or lam.dtype not in _LAMBDA_DTYPES:
            raise ValueError("lambda_scale must hold one float16, bfloat16 or float32 element")
        raise RuntimeError(f"lambda_scale is on {lam.device}, the cache on {self._device}")

    def evict(self, keep: int, recent: int = 0) -> None:
        """Cuts every sequence longer than `keep` back to `keep` tokens, per head: the tokens of its last `recent` positions stay, then those with
        the largest `weights` (ties: the lowest slot); without weights those of the largest positions.  `evict(n, recent=n)` is a window of the
        last n tokens.  Weights are what `attend` has added since a token was stored: right behind a prompt's `append` they are all 0, and but for `recent`
        the oldest tokens stay; a few steps later they rank tokens by those steps.  Survivors move into the slots that come free, so tokens change
        their slots (`positions` says which is where).  Pages behind the new lengths are free again."""
        keep, recent = operator.index(keep), operator.index(recent)      # (a field of 32 bits would take the lowest ones of any number)
        if not (1 <= keep <= self.slots and 0 <= recent <= keep):
            raise ValueError(f"keep={keep} must lie in [1, {self.slots}], recent={recent} in [0, keep]")
        p = self._params()
        p.keep, p.recent = keep, recent
        nbytes = int(_lib.lib.diffattn_cache_workspace_bytes(p, _lib.CACHE_EVICT))
        ws = self._workspace(p, nbytes) if nbytes else None  # noqa: F841
        counter = self._count_with(p)  # noqa: F841
        _lib.check(_lib.lib.diffattn_cache_evict(p), "diffattn_cache_evict")
