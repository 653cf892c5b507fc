"""What `DiffAttnCache` makes of its arguments before anything is launched (no GPU: a library that only writes down what it is given)."""
import ctypes
from types import SimpleNamespace

import pytest
import torch

from triton_diff_attn_b200 import _lib, cache as cache_module


class _Library:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(p, *rest):
            if name != "diffattn_cache_workspace_bytes":
                self.calls.append((name, _lib.DiffAttnCacheParams.from_buffer_copy(p)))
            return 0
        return call


@pytest.fixture
def bare(monkeypatch):
    """A cache of 2 sequences, 3 heads, D = 64 and 64 slots without memory, and its library."""
    library = _Library()
    monkeypatch.setattr(cache_module, "_lib", SimpleNamespace(**{**vars(_lib), "lib": library}))
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0, raising=False)
    c = cache_module.DiffAttnCache.__new__(cache_module.DiffAttnCache)
    p = _lib.DiffAttnCacheParams()
    p.struct_size = ctypes.sizeof(p)
    p.B, p.H, p.D, p.page_size, p.num_pages, p.max_pages = 2, 3, 64, 16, 9, 4
    c._sizes, c._shape, c._device, c._index, c._dtype = p, (2, 3, 64), torch.device("cpu"), -1, torch.float16
    c._lengths, c._y, c._attend_bytes = torch.zeros(2, dtype=torch.int32), torch.empty(2, 3, 1, 128, dtype=torch.float16), 0
    c._counter = torch.zeros(1, dtype=torch.int32)
    return c, library.calls


@pytest.mark.parametrize("keep,recent,error", [
    (2 ** 32 + 5, 0, ValueError), (-2 ** 32 + 5, 0, ValueError), (5, 2 ** 32, ValueError), (5, -2 ** 32 + 1, ValueError), (65, 0, ValueError), (0, 0, ValueError),
    (5, 6, ValueError), (5, -1, ValueError), (40.9, 0, TypeError), (40, 1.5, TypeError), ("40", 0, TypeError), (None, 0, TypeError),
])
def test_evict_refuses_sizes(bare, keep, recent, error):
    c, calls = bare
    with pytest.raises(error):
        c.evict(keep, recent)
    assert not calls


def test_evict_takes_whole_numbers(bare):
    np = pytest.importorskip("numpy")
    c, calls = bare
    for keep, recent in ((40, 7), (np.int64(40), np.int32(7)), (torch.tensor(40), torch.tensor(7)), (64, 64), (1, 0)):
        c.evict(keep, recent)
        name, p = calls.pop()
        assert (name, p.keep, p.recent) == ("diffattn_cache_evict", int(keep), int(recent)) and not calls


def _tensors():
    r = lambda *shape: torch.ones(shape, dtype=torch.float16)
    return dict(q1=r(2, 3, 1, 64), q2=r(2, 3, 1, 64), lambda_scale=torch.full((1,), 0.5), gain=torch.ones(128), k1=r(2, 3, 1, 64), k2=r(2, 3, 1, 64), v=r(2, 3, 1, 128))


@pytest.mark.parametrize("name", list(_tensors()))
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_tangents_are_refused(bare, name, grad):
    """y would come back without one.  (no_grad does not switch forward mode off.)"""
    import torch.autograd.forward_ad as fw
    c, calls = bare
    with fw.dual_level(), torch.set_grad_enabled(grad):
        t = _tensors()
        c.attend(**t)                                     # a level alone is no tangent
        c.append(t["k1"], t["k2"], t["v"])
        assert [n for n, _ in calls] == ["diffattn_cache_attend", "diffattn_cache_append"]
        t[name] = fw.make_dual(t[name], torch.ones_like(t[name]))
        with pytest.raises(NotImplementedError, match=name):
            c.attend(**t)
        if name in ("k1", "k2", "v"):
            with pytest.raises(NotImplementedError, match=name):
                c.append(t["k1"], t["k2"], t["v"])
        assert len(calls) == 2
    with fw.dual_level(), torch.inference_mode():         # (this does)
        c.attend(**t)
    assert len(calls) == 3


def test_decode_refuses_tangents(bare):
    import torch.autograd.forward_ad as fw
    from triton_diff_attn_b200 import DiffAttnCore
    c, calls = bare
    core, t = DiffAttnCore(64, causal=True), _tensors()
    rows = [t[n] for n in ("q1", "q2", "k1", "k2", "v")]
    core.decode(*rows, c)
    with fw.dual_level():
        for i in range(5):
            with pytest.raises(NotImplementedError):
                core.decode(*(fw.make_dual(x, x) if i == j else x for j, x in enumerate(rows)), c)
        for n in ("lambda_q1", "gain"):
            p = dict(core.named_parameters())[n]
            dual = {n: fw.make_dual(p.detach(), torch.ones_like(p))}
            with pytest.raises(NotImplementedError):
                torch.func.functional_call(_Decode(core), {"core." + k: x for k, x in dual.items()}, (rows, c))
    assert len(calls) == 1


class _Decode(torch.nn.Module):
    def __init__(self, core):
        super().__init__()
        self.core = core

    def forward(self, rows, cache):
        return self.core.decode(*rows, cache)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_counts_beyond_32_bits(bare, monkeypatch, dtype):
    """More than there are rows means all of them, less than none means none, whatever the number."""
    c, _ = bare
    seen = []
    read = lambda p, *_: seen.append(list((ctypes.c_int32 * 2).from_address(p.counts))) or 0
    monkeypatch.setattr(cache_module._lib.lib, "diffattn_cache_append", read, raising=False)
    monkeypatch.setattr(cache_module._lib.lib, "diffattn_cache_attend", read, raising=False)
    t = _tensors()
    rows = [torch.ones(2, 3, 5, w, dtype=torch.float16) for w in (64, 64, 128)]
    far = [2 ** 32, 2 ** 32 + 3, 2 ** 31, -2 ** 32 + 2, -2 ** 63, 2 ** 63 - 1] if dtype == torch.int64 else [2 ** 31 - 1, -2 ** 31]
    for n in far + [0, 1, 3, 5, 6, -1]:
        counts = torch.tensor([n, 2], dtype=dtype)
        c.append(*rows, counts)
        a, b = seen.pop()
        assert (min(max(a, 0), 5), b) == (min(max(n, 0), 5), 2)      # (the kernels clamp what they get)
        c.attend(**t, counts=counts)
        a, b = seen.pop()
        assert (a > 0, b > 0) == (n > 0, True)
        assert counts.tolist() == [n, 2]
