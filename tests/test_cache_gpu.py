"""GPU tests of the key-value cache (`DiffAttnCache`): every operator against its definition in 64 bits (cache_reference.py), at the
lengths, pages and contents where it can go wrong."""
import math

import pytest
import torch

import cache_reference as ref
from oracle import diffattn_oracle as oracle

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pkg():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import triton_diff_attn_b200
    return triton_diff_attn_b200


DEV = torch.device("cuda", 0)


def make(pkg, lengths, h, d, page, *, dt=torch.float16, slot_major=False, track=False, extra=0, seed=0, scale=1.0, room=0, first_position=0):
    """A cache with sequences of these lengths: pages anywhere in the pool, not a number in every slot that holds no token, and table entries
    behind the used ones that are no pages."""
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    b = len(lengths)
    max_pages = max(1, -(-(max(lengths) + room) // page))
    num = b * max_pages + 2 + extra

    def pool(w):
        shape = (num, page, h, w) if slot_major else (num, h, page, w)
        t = torch.full(shape, math.nan, dtype=dt, device=DEV)
        return t.transpose(1, 2) if slot_major else t

    k1, k2, v = pool(d), pool(d), pool(2 * d)
    table = torch.randperm(num, generator=g, device=DEV)[:b * max_pages].to(torch.int32).view(b, max_pages)
    for i, n in enumerate(lengths):
        at = torch.arange(n, device=DEV)
        pages = table[i].long()[at // page]
        for t, w in ((k1, d), (k2, d), (v, 2 * d)):
            t[pages, :, at % page] = (torch.randn((n, h, w), generator=g, device=DEV) * scale).to(dt)
        used = -(-(n + room) // page)
        bad = torch.tensor([-1, -7, num, 2 ** 31 - 1], dtype=torch.int32, device=DEV)
        if used < max_pages:
            table[i, used:] = bad[torch.arange(max_pages - used, device=DEV) % 4]
    slots = max_pages * page
    lens = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    pos = torch.full((b, h, slots), -9, dtype=torch.int32, device=DEV)
    weights = torch.full((b, h, slots), math.nan, device=DEV) if track else None
    for i, n in enumerate(lengths):
        pos[i, :, :n] = torch.arange(n, device=DEV, dtype=torch.int32) + first_position
        if track:
            weights[i, :, :n] = torch.rand((h, n), generator=g, device=DEV)
    return pkg.DiffAttnCache.from_tensors(k1, k2, v, table, lens, positions=pos, next_position=lens + first_position, weights=weights)


def queries(b, h, d, dt, seed=1, t=1):
    g = torch.Generator(device=DEV)
    g.manual_seed(1000 + seed)
    r = lambda w: torch.randn((b, h, t, w), generator=g, device=DEV).to(dt)
    return r(d), r(d), r(d), r(d), r(2 * d)


def snapshot(c):
    # a tensor's bits: what has to stay as it was may hold values that are not numbers
    whole = lambda t: t if t is None or t.dtype == torch.int32 else t.view(torch.int32 if t.dtype == torch.float32 else torch.int16)
    return [None if t is None else whole(t).clone() for t in (c.k1_pages, c.k2_pages, c.v_pages, c.lengths, c.next_position, c.positions, c.weights)]


def check_attend(c, before, y, q1, q2, lam, lengths, token=None, rms=True, gain=None, lambda_init=0.8):
    """y and the weights of every (sequence, head) against the definition; `before`: lengths before the call."""
    b, h, _, d2 = y.shape
    d, page, io = d2 // 2, c.k1_pages.shape[2], c.k1_pages.dtype
    old_w = before["weights"]
    for i in range(b):
        n = lengths[i]
        for j in range(h):
            k1, k2, v = (ref.rows(t, c.page_table[i], page, j, n) for t in (c.k1_pages, c.k2_pages, c.v_pages))
            if token is not None:
                k1, k2, v = (torch.cat([x, t[i, j].double()]) for x, t in zip((k1, k2, v), token))
            want, w, dy, dw = ref.attend(q1[i, j, 0].double(), q2[i, j, 0].double(), k1, k2, v, lam, lambda_init, rms, gain, io)
            off = (y[i, j, 0].double() - want).abs()
            assert bool((off <= dy).all()), (i, j, n, float((off / dy).max()))
            if old_w is not None:
                m = len(w)
                base = old_w[i, j, :m].double().clone()
                if token is not None:
                    base[n] = 0.0
                got = c.weights[i, j, :m].double()
                tol = dw + 2 * ref.U32 * (base + w)
                assert bool(((got - base - w).abs() <= tol).all()), (i, j, n, float(((got - base - w).abs() / tol).max()))


LENGTHS = {   # by head dim: around a tile's 1024 / D tokens
    32: [0, 1, 31, 32, 33, 64, 200, 7],
    64: [1, 0, 15, 16, 17, 48, 130, 3],
    128: [7, 8, 9, 0, 1, 40, 77, 2],
}


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("page", [1, 2, 4, 7, 8, 16, 24, 33, 64, 100])
@pytest.mark.parametrize("form", ["plain", "track", "token", "token_track"])
def test_attend_pages_and_lengths(pkg, d, page, form):
    dt = torch.bfloat16 if (page + d // 32) % 2 else torch.float16
    track, token = "track" in form, "token" in form
    lengths = LENGTHS[d]
    c = make(pkg, lengths, 3, d, page, dt=dt, track=track, slot_major=page in (7, 16, 64), seed=page * 7 + d, room=1 if token else 0)
    q1, q2, nk1, nk2, nv = queries(len(lengths), 3, d, dt, seed=page)
    gain = torch.linspace(0.5, 1.5, 2 * d, device=DEV)
    lam = torch.tensor([0.6], device=DEV)
    before, old = snapshot(c), {"weights": None if c.weights is None else c.weights.clone()}
    y = c.attend(q1, q2, lam, 0.8, True, gain=gain, **(dict(k1=nk1, k2=nk2, v=nv) if token else {}))
    pkg.device_status(0)
    check_attend(c, old, y, q1, q2, float(lam), lengths, (nk1, nk2, nv) if token else None, True, gain)
    # what the call stored, and nothing else
    for i, n in enumerate(lengths if token else []):
        at = int(c.page_table[i, n // page])
        for t, new in zip((c.k1_pages, c.k2_pages, c.v_pages), (nk1, nk2, nv)):
            assert torch.equal(t[at, :, n % page], new[i, :, 0])
            t[at, :, n % page] = math.nan
        assert bool((c.positions[i, :, n] == n).all())
        c.positions[i, :, n] = -9
    if token:
        assert c.lengths.tolist() == [n + 1 for n in lengths] and c.next_position.tolist() == [n + 1 for n in lengths]
        c.lengths.sub_(1); c.next_position.sub_(1)
    if track:
        for i, n in enumerate(lengths):
            m = n + (1 if token else 0)
            c.weights[i, :, :m] = old["weights"][i, :, :m]
    for a, w in zip(snapshot(c), before):
        assert a is None or torch.equal(a, w)


@pytest.mark.parametrize("d,dt,b,h,n,page,scale", [
    (64, torch.float16, 1, 2, 5000, 64, 1.0),       # one long sequence: a hundred and more pieces to join
    (64, torch.bfloat16, 2, 1, 3001, 16, 1.0),
    (128, torch.float16, 1, 1, 2777, 128, 1.0),
    (32, torch.bfloat16, 1, 3, 4097, 33, 1.0),
    (64, torch.float16, 1, 2, 900, 64, 4.0),        # scores up to a hundred: the running maximum moves
    (64, torch.float16, 70, 20, 40, 16, 1.0),       # more (sequence, head)s than warps: several to a stretch
    (32, torch.float16, 300, 5, 3, 8, 1.0),         # more sequences than threads, a tile each
])
def test_attend_splits(pkg, d, dt, b, h, n, page, scale):
    lengths = [max(0, n - 3 * i) for i in range(b)] if b < 50 else [(7 * i) % (n + 1) for i in range(b)]
    c = make(pkg, lengths, h, d, page, dt=dt, track=True, scale=scale, seed=n)
    q1, q2, *_ = queries(b, h, d, dt, seed=n)
    lam = torch.tensor([-0.4], dtype=torch.bfloat16, device=DEV)
    old = {"weights": c.weights.clone()}
    y = c.attend(q1, q2, lam)
    pkg.device_status(0)
    keep = sorted({0, 1, b // 2, b - 1} & set(range(b)))
    sub = type("C", (), dict(k1_pages=c.k1_pages, k2_pages=c.k2_pages, v_pages=c.v_pages, page_table=c.page_table[keep], weights=c.weights[keep]))
    check_attend(sub, {"weights": old["weights"][keep]}, y[keep], q1[keep], q2[keep], float(lam), [lengths[i] for i in keep], rms=False)
    y2 = c.attend(q1, q2, lam)
    assert torch.equal(y, y2)                        # the order of every sum is fixed


def test_attend_extreme_scores(pkg):
    """One token takes all the weight, scores far below and far above it, values of the largest size that the type holds beside it."""
    c = make(pkg, [130], 1, 64, 16, seed=3)
    q1, q2, *_ = queries(1, 1, 64, torch.float16, seed=3)
    rows = torch.arange(130, device=DEV)
    pages = c.page_table[0].long()[rows // 16]
    c.k1_pages[pages, 0, rows % 16] = -30.0 * q1[0, 0, 0].sign()
    c.k2_pages[pages, 0, rows % 16] = -30.0 * q2[0, 0, 0].sign()
    c.v_pages[pages, 0, rows % 16] = 60000.0
    at = int(c.page_table[0, 100 // 16])
    c.k1_pages[at, 0, 100 % 16] = 30.0 * q1[0, 0, 0].sign()
    c.k2_pages[at, 0, 100 % 16] = 30.0 * q2[0, 0, 0].sign()
    c.v_pages[at, 0, 100 % 16] = 1.0
    y = c.attend(q1, q2, torch.tensor([0.5], device=DEV))
    assert torch.allclose(y.float(), torch.full_like(y.float(), 0.5), rtol=0, atol=1e-6)


@pytest.mark.parametrize("lam_dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lambda_init,rms", [(0.2, True), (0.2, False)])
def test_attend_norm_and_lambda(pkg, lam_dtype, lambda_init, rms):
    c = make(pkg, [50, 9], 2, 64, 16, seed=5)
    q1, q2, *_ = queries(2, 2, 64, torch.float16, seed=5)
    lam = torch.tensor([0.7], dtype=lam_dtype, device=DEV)
    y = c.attend(q1, q2, lam, lambda_init, rms)
    check_attend(c, {"weights": None}, y, q1, q2, float(lam), [50, 9], rms=rms, lambda_init=lambda_init)


def test_attend_strided_queries_and_shared_pages(pkg):
    """q as a slice of a packed projection, k1/k2/v of a step likewise (one of them at an odd address); two sequences on the same pages."""
    c = make(pkg, [40, 40], 4, 64, 16, seed=6, room=8)
    c.page_table[1, :2] = c.page_table[0, :2]                # a common prefix of two full pages
    packed = torch.randn(2, 1, 4, 6 * 64 + 3, device=DEV).half()
    cut = lambda lo, w: packed[..., lo:lo + w].transpose(1, 2)
    q1, q2, k1, k2, v = cut(0, 64), cut(64, 64), cut(128, 64), cut(192, 64), cut(259, 128)
    old = {"weights": None}
    lam = torch.tensor([0.5], device=DEV)
    y = c.attend(q1, q2, lam, k1=k1, k2=k2, v=v)
    check_attend(c, old, y, q1, q2, 0.5, [40, 40], (k1, k2, v), rms=False)
    pkg.device_status(0)


@pytest.mark.parametrize("d,page", [(64, 16), (32, 7), (128, 100)])
@pytest.mark.parametrize("track", [False, True])
def test_attend_some_get_a_token(pkg, d, page, track):
    """A batch with rows that are not in use: no pages, no length, nothing of them written; others only look."""
    lengths, counts = [0, 20, 0, 33, 48, 0, 7], [1, 1, 0, 0, 1, 0, 0]
    c = make(pkg, lengths, 2, d, page, track=track, seed=page, room=1)
    for i in (2, 5):
        c.page_table[i] = -1
    q1, q2, k1, k2, v = queries(7, 2, d, torch.float16, seed=d)
    lam = torch.tensor([0.5], device=DEV)
    before, old = snapshot(c), {"weights": None if c.weights is None else c.weights.clone()}
    y = c.attend(q1, q2, lam, k1=k1, k2=k2, v=v, counts=torch.tensor(counts, device=DEV))
    pkg.device_status(0)
    for got in (0, 1):
        at = [i for i in range(7) if counts[i] == got]
        sub = type("C", (), dict(k1_pages=c.k1_pages, k2_pages=c.k2_pages, v_pages=c.v_pages, page_table=c.page_table[at],
                                 weights=None if c.weights is None else c.weights[at]))
        check_attend(sub, {"weights": None if c.weights is None else old["weights"][at]}, y[at], q1[at], q2[at], 0.5, [lengths[i] for i in at],
                     tuple(x[at] for x in (k1, k2, v)) if got else None, rms=False)
    assert c.lengths.tolist() == [n + m for n, m in zip(lengths, counts)] == c.next_position.tolist()
    for i, (n, m) in enumerate(zip(lengths, counts)):
        if m:
            for t, x in zip((c.k1_pages, c.k2_pages, c.v_pages), (k1, k2, v)):
                p = int(c.page_table[i, n // page])
                assert torch.equal(t[p, :, n % page], x[i, :, 0])
                t[p, :, n % page] = math.nan
            assert bool((c.positions[i, :, n] == n).all())
            c.positions[i, :, n] = -9
        if track:
            c.weights[i, :, :n + m] = old["weights"][i, :, :n + m]
    c.lengths.copy_(torch.tensor(lengths, dtype=torch.int32)); c.next_position.copy_(c.lengths)
    for a, w in zip(snapshot(c), before):
        assert a is None or torch.equal(a, w)
    with pytest.raises(ValueError):
        c.attend(q1, q2, lam, counts=torch.tensor(counts, device=DEV))


def test_attend_far_pages(pkg):
    """Rows more than 2^32 bytes behind the pool's base."""
    page, d, h = 256, 128, 1
    num = (2 ** 32 // (page * d * 2)) + 3
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    k1, k2 = (torch.empty(num, h, page, d, dtype=torch.float16, device=DEV) for _ in range(2))
    v = torch.empty(num, h, page, 2 * d, dtype=torch.float16, device=DEV)
    table = torch.tensor([[num - 1, 0, num - 2]], dtype=torch.int32, device=DEV)
    lens = torch.zeros(1, dtype=torch.int32, device=DEV)
    slots = 3 * page
    c = pkg.DiffAttnCache.from_tensors(k1, k2, v, table, lens, positions=torch.zeros(1, h, slots, dtype=torch.int32, device=DEV),
                                       next_position=torch.zeros_like(lens), weights=torch.zeros(1, h, slots, device=DEV))
    n = 2 * page + 10
    _, _, nk1, nk2, nv = queries(1, h, d, torch.float16, seed=8, t=n)
    c.append(nk1, nk2, nv)
    q1, q2, t1, t2, tv = queries(1, h, d, torch.float16, seed=9)
    y = c.attend(q1, q2, torch.tensor([0.5], device=DEV), k1=t1, k2=t2, v=tv)
    check_attend(c, {"weights": None}, y, q1, q2, 0.5, [n], (t1, t2, tv), rms=False)
    c.weights[0, 0, :n + 1] = torch.arange(n + 1, device=DEV).float()
    want = [t[num - 2, 0, 10].clone() for t in (k1, k2, v)]      # the newest token, the one with the largest weight, moves into slot 0
    c.evict(n)
    assert all(torch.equal(t[num - 1, 0, 0], w) for t, w in zip((k1, k2, v), want))
    pkg.device_status(0)


@pytest.mark.parametrize("d,dt,page,slot_major", [(64, torch.float16, 16, False), (32, torch.bfloat16, 7, True), (128, torch.float16, 1, False), (64, torch.bfloat16, 100, True)])
@pytest.mark.parametrize("counts", [None, [5, 0, 33, 100]])
def test_append(pkg, d, dt, page, slot_major, counts):
    lengths, t = [0, 3, 17, 64], 33
    c = make(pkg, lengths, 2, d, page, dt=dt, slot_major=slot_major, track=True, room=t, seed=d + page, first_position=5)
    g = torch.Generator(device=DEV); g.manual_seed(4)
    k1, k2, v = (torch.randn((4, t, 2, w), generator=g, device=DEV).to(dt).transpose(1, 2) for w in (d, d, 2 * d))
    before = snapshot(c)
    gets = [t] * 4 if counts is None else [min(n, t) for n in counts]
    c.append(k1, k2, v, None if counts is None else torch.tensor(counts, device=DEV))
    pkg.device_status(0)
    assert c.lengths.tolist() == [n + m for n, m in zip(lengths, gets)]
    assert c.next_position.tolist() == [5 + n + m for n, m in zip(lengths, gets)]
    after = snapshot(c)
    # rebuild what has to be there from what was
    dt_bits = torch.int16
    for i, (n, m) in enumerate(zip(lengths, gets)):
        at = torch.arange(n, n + m, device=DEV)
        pages = c.page_table[i].long()[at // page]
        for which, new in enumerate((k1, k2, v)):
            before[which][pages, :, at % page] = new[i, :, :m].contiguous().view(dt_bits).transpose(0, 1)
        before[5][i, :, n:n + m] = (5 + at).to(torch.int32)
        before[6][i, :, n:n + m] = 0
    before[3], before[4] = c.lengths, c.next_position
    for a, w in zip(after, before):
        assert torch.equal(a, w)


def test_append_large(pkg):
    """As many rows as have the lengths moved on by a kernel of their own."""
    b, h, t, d = 4, 16, 700, 64
    c = make(pkg, [0, 30, 700, 9], h, d, 16, track=True, room=t, seed=3)
    g = torch.Generator(device=DEV); g.manual_seed(5)
    k1, k2, v = (torch.randn((b, h, t, w), generator=g, device=DEV).half() for w in (d, d, 2 * d))
    for counts in (None, [700, 0, 333, 1]):
        gets = counts or [t] * b
        c.lengths.copy_(torch.tensor([0, 30, 700, 9], dtype=torch.int32)); c.next_position.copy_(c.lengths)
        for p in (c.k1_pages, c.k2_pages, c.v_pages):
            p.fill_(math.nan)
        c.append(k1, k2, v, None if counts is None else torch.tensor(counts, device=DEV))
        pkg.device_status(0)
        for i, (n, m) in enumerate(zip([0, 30, 700, 9], gets)):
            at = torch.arange(n, n + m, device=DEV)
            pages = c.page_table[i].long()[at // 16]
            for p, x in ((c.k1_pages, k1), (c.k2_pages, k2), (c.v_pages, v)):
                assert torch.equal(p[pages, :, at % 16], x[i, :, :m].transpose(0, 1))
            assert bool((c.positions[i, :, n:n + m] == at).all()) and not bool(c.weights[i, :, n:n + m].any())
        assert c.lengths.tolist() == [n + m for n, m in zip([0, 30, 700, 9], gets)] == c.next_position.tolist()
        assert sum(int(torch.isfinite(p[..., 0]).sum()) for p in (c.k1_pages, c.k2_pages, c.v_pages)) == 3 * h * sum(gets)


EVICT = [
    # lengths, keep, recent, weights
    ([40, 33, 32, 0, 5], 32, 0, "random"),
    ([100, 64, 31], 30, 10, "random"),
    ([100, 64, 31], 30, 30, "random"),       # a window
    ([100, 64, 31], 1, 0, "random"),
    ([700, 513, 1100], 512, 7, "ties"),      # several rounds of the selection, most weights alike
    ([200, 90], 64, 0, "odd"),               # zeros of both signs, infinities, not a number, negative ones
    ([200, 90], 64, 3, "none"),              # no weights: the newest stay
    ([60, 90], 89, 0, "zeros"),
]


@pytest.mark.parametrize("lengths,keep,recent,kind", EVICT)
@pytest.mark.parametrize("d,page", [(64, 16), (32, 7), (128, 64)])
def test_evict(pkg, lengths, keep, recent, kind, d, page):
    h = 2
    c = make(pkg, lengths, h, d, page, track=kind != "none", slot_major=page == 7, room=max(0, keep - max(lengths)), seed=keep + d, first_position=3)
    g = torch.Generator(device=DEV); g.manual_seed(keep)
    if kind == "ties":
        c.weights.copy_(torch.randint(0, 3, c.weights.shape, generator=g, device=DEV).float())
    elif kind == "zeros":
        c.weights.zero_()
    elif kind == "odd":
        pick = torch.tensor([0.0, -0.0, math.inf, -math.inf, math.nan, -math.nan, -1.0, 1e-40, 2.0, -3e38, 3e38], device=DEV)
        c.weights.copy_(pick[torch.randint(0, len(pick), c.weights.shape, generator=g, device=DEV)])
    for i, n in enumerate(lengths):                       # as after an earlier eviction: other tokens in each head, in no order
        for j in range(h):
            c.positions[i, j, :n] = torch.randperm(n, generator=g, device=DEV).to(torch.int32) + 3
    before = snapshot(c)
    w_cpu, p_cpu = None if c.weights is None else c.weights.cpu(), c.positions.cpu()
    c.evict(keep, recent)
    pkg.device_status(0)
    assert c.lengths.tolist() == [min(n, keep) for n in lengths]
    for i, n in enumerate(lengths):
        for j in range(h):
            for to, frm in ref.evict(None if w_cpu is None else w_cpu[i, j], p_cpu[i, j], n, n + 3, keep, recent):
                a, b = int(c.page_table[i, to // page]), int(c.page_table[i, frm // page])
                for t in before[:3]:
                    t[a, j, to % page] = t[b, j, frm % page]
                for t in before[5:]:
                    if t is not None:
                        t[i, j, to] = t[i, j, frm]
    before[3] = c.lengths
    for a, w in zip(snapshot(c), before):
        assert a is None or torch.equal(a, w)


@pytest.mark.parametrize("slots", [49000, 50000])
def test_evict_long(pkg, slots):
    """Around the number of keys that shared memory holds."""
    n, keep = slots, slots - 1500
    c = make(pkg, [n], 1, 32, 1000, track=True, seed=2)
    c.weights[0, 0] = torch.randperm(n, device=DEV).float()
    w = c.weights[0, 0].clone()
    c.evict(keep)
    pkg.device_status(0)
    assert int(c.lengths[0]) == keep
    assert torch.equal(c.weights[0, 0, :keep].sort().values, w.sort().values[-keep:])
    stay = w[:keep] >= 1500
    assert torch.equal(c.weights[0, 0, :keep][stay], w[:keep][stay])
    assert torch.equal(c.weights[0, 0, :keep][~stay], w[keep:][w[keep:] >= 1500])


def test_bad_contents_are_reported_and_touch_nothing(pkg):
    """Lengths outside the cache, pages outside the pool, full sequences: memory stays as it was, device_status() raises."""
    q1, q2, k1, k2, v = queries(2, 2, 64, torch.float16)
    lam = torch.tensor([0.5], device=DEV)
    for what in ("page", "length", "full"):
        for call in ("attend", "token", "append", "evict"):
            c = make(pkg, [40, 20], 2, 64, 16, track=True, seed=1)
            if what == "page":
                c.page_table[0, 0 if call in ("attend", "evict") else 2] = 2 ** 30
                if call == "evict":
                    c.weights[0, :, 1:].fill_(1.0); c.weights[0, :, 0].zero_()      # slot 0, on the bad page, is the hole
            elif what == "length":
                c.lengths[0] = -3 if call in ("attend", "append") else 49
            elif call in ("token", "append"):
                c.lengths[0] = 48
            else:
                continue
            before = snapshot(c)
            if call == "attend":
                c.attend(q1, q2, lam)
            elif call == "token":
                c.attend(q1, q2, lam, k1=k1, k2=k2, v=v)
            elif call == "append":
                c.append(k1, k2, v)
            else:
                c.evict(39)
            with pytest.raises(ValueError, match="BAD_CACHE"):
                pkg.device_status(0)
            pkg.device_status(0)                          # the report is given once
            after = snapshot(c)
            rest = torch.ones(c.k1_pages.shape[0], dtype=torch.bool, device=DEV)
            for i in range(2):                            # pages that belong to a sequence may have changed, no others
                for p in c.page_table[i].tolist():
                    if 0 <= p < len(rest):
                        rest[p] = False
            for a, w in zip(after[:3], before[:3]):
                assert torch.equal(a[rest], w[rest])
            assert 0 <= int(c.lengths[0]) <= c.slots or call in ("attend", "evict")


def test_capture_streams_and_threads(pkg):
    """A step captured once and replayed gives what eager calls give; so do calls on another stream."""
    def fresh():
        return make(pkg, [37, 60, 0], 2, 64, 16, track=True, seed=11, room=20)
    qs = [queries(3, 2, 64, torch.float16, seed=s) for s in range(6)]
    lam = torch.tensor([0.5], device=DEV)

    def step(c, q):
        y = c.attend(q[0], q[1], lam, 0.8, True, k1=q[2], k2=q[3], v=q[4])
        c.evict(50, recent=4)
        return y

    a = fresh()
    want = [step(a, q) for q in qs]
    b = fresh()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [step(b, q) for q in qs]
    torch.cuda.current_stream().wait_stream(side)
    c = fresh()
    static = [t.clone() for t in qs[0]]
    saved = [None if t is None else t.clone() for t in (c.k1_pages, c.k2_pages, c.v_pages, c.lengths, c.next_position, c.positions, c.weights)]
    step(c, static)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step(c, static)
    for t, s in zip((c.k1_pages, c.k2_pages, c.v_pages, c.lengths, c.next_position, c.positions, c.weights), saved):
        t.copy_(s)
    for i, q in enumerate(qs):
        for t, x in zip(static, q):
            t.copy_(x)
        graph.replay()
        assert torch.equal(y, want[i]) and torch.equal(got[i], want[i])
    for x, w, z in zip(snapshot(c), snapshot(a), snapshot(b)):
        assert torch.equal(x, w) and torch.equal(z, w)
    pkg.device_status(0)


@pytest.mark.parametrize("captured", [False, True])
def test_right_behind_its_inputs(pkg, captured):
    """Kernels and copies that write queries, lengths, page table and rows right in front of a call: it reads what they wrote."""
    h, d, page, n = 4, 64, 16, 300
    c = make(pkg, [n, n], h, d, page, track=True, seed=14, room=40)
    lam = torch.tensor([0.5], device=DEV)
    q1, q2, k1, k2, v = queries(2, h, d, torch.float16, seed=14)
    other = c.page_table.flip(0).contiguous()            # the two sequences change places: pages, rows and weights go along
    lens = [torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([n, 100], [37, n])]
    big = torch.randn(64 << 20, device=DEV)
    zero = torch.zeros_like(c.weights)

    def calls():
        out = []
        for i in range(6):
            big.mul_(1.0)                                # something long ahead, so that the call is enqueued while it runs
            q1.mul_(-1.0)
            c.page_table.copy_(other if i % 2 else other.flip(0))
            c.lengths.copy_(lens[i % 2])
            c.weights.copy_(zero)
            c.v_pages.mul_(-1.0)
            y = c.attend(q1, q2, lam, k1=k1, k2=k2, v=v)
            c.append(k1, k2, v)
            c.evict(30)
            out += [y, c.weights.clone(), c.lengths.clone()]
        return out

    state = [t.clone() for t in (c.k1_pages, c.k2_pages, c.v_pages, c.page_table, c.lengths, c.next_position, c.positions, c.weights, q1)]

    def restore():
        for t, x in zip((c.k1_pages, c.k2_pages, c.v_pages, c.page_table, c.lengths, c.next_position, c.positions, c.weights, q1), state):
            t.copy_(x)
        torch.cuda.synchronize()

    class Slow:                                          # the same calls with a wait behind every one of them
        def __getattr__(self, name):
            def call(*a, **kw):
                torch.cuda.synchronize()
                r = getattr(c0, name)(*a, **kw)
                torch.cuda.synchronize()
                return r
            return call if name in ("attend", "append", "evict") else getattr(c0, name)

    c0, c = c, Slow()
    restore()
    want = calls()
    c = c0
    restore()
    if captured:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = calls()
        restore()
        g.replay()
    else:
        got = calls()
    torch.cuda.synchronize()
    same = lambda a, b: torch.equal(a.view(torch.int16) if a.dtype == torch.float16 else a.view(torch.int32), b.view(torch.int16) if b.dtype == torch.float16 else b.view(torch.int32))
    assert all(same(a, b) for a, b in zip(got, want))
    pkg.device_status(0)


def test_two_graphs_at_once(pkg):
    """Queries that write nothing may overlap: two captured calls on one cache, replayed on two streams, have workspaces of their own."""
    c = make(pkg, [900, 0, 333, 1500], 4, 64, 16, seed=12)
    lam = torch.tensor([0.5], device=DEV)
    qs = [queries(4, 4, 64, torch.float16, seed=s) for s in (1, 2)]
    want = [c.attend(q[0], q[1], lam) for q in qs]
    graphs, ys = [], []
    for q in qs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ys.append(c.attend(q[0], q[1], lam))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in qs]
    for _ in range(20):
        for st, g in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(y, w) for y, w in zip(ys, want))


def test_attend_many_sequences(pkg):
    """The largest batch, most of it not in use."""
    lengths = [0] * 4096
    for i in (0, 1, 31, 32, 255, 256, 2048, 4094, 4095):
        lengths[i] = 1 + i % 50
    c = make(pkg, lengths, 1, 32, 64, seed=13)
    q1, q2, *_ = queries(4096, 1, 32, torch.float16, seed=13)
    y = c.attend(q1, q2, torch.tensor([0.5], device=DEV))
    used = [i for i, n in enumerate(lengths) if n]
    sub = type("C", (), dict(k1_pages=c.k1_pages, k2_pages=c.k2_pages, v_pages=c.v_pages, page_table=c.page_table[used], weights=None))
    check_attend(sub, {"weights": None}, y[used], q1[used], q2[used], 0.5, [lengths[i] for i in used], rms=False)
    rest = torch.ones(4096, dtype=torch.bool, device=DEV)
    rest[used] = False
    assert not bool(y[rest].any())
    with pytest.raises(ValueError):
        pkg.DiffAttnCache(4097, 1, 32, 8, device=DEV).attend(*(torch.zeros(4097, 1, 1, 32, dtype=torch.float16, device=DEV),) * 2, torch.tensor([0.5], device=DEV))
    pkg.device_status(0)


@pytest.mark.parametrize("d,dt", [(64, torch.float16), (128, torch.bfloat16), (32, torch.float16)])
def test_prompt_then_generation(pkg, d, dt):
    """A layer core's prompt through its causal forward, its tokens into the cache, then token by token: every step is the last row of the causal
    forward over everything so far, with a cache that was cut down it is the attention over what stayed."""
    b, h, n, steps = 2, 4, 70, 5
    torch.manual_seed(3)
    core = pkg.DiffAttnCore(d, causal=True, device=DEV).eval()
    with torch.no_grad():
        core.gain.uniform_(0.5, 1.5)
    q1, q2, k1, k2, v = queries(b, h, d, dt, seed=17, t=n + steps)
    cache = pkg.DiffAttnCache(b, h, d, n + steps, page_size=16, track_weights=True, dtype=dt, device=DEV)
    cut = lambda t, lo, hi: t[:, :, lo:hi]
    with torch.no_grad():
        core(*(cut(t, 0, n) for t in (q1, q2, k1, k2, v)))
        whole = core(q1, q2, k1, k2, v)
        lam = float(pkg.lambda_from_reparam(core.lambda_q1, core.lambda_k1, core.lambda_q2, core.lambda_k2, 0.8))
    cache.append(*(cut(t, 0, n) for t in (k1, k2, v)))
    gathered = torch.zeros(b, h, n + steps, dtype=torch.float64, device=DEV)
    for s in range(n, n + steps):
        y = core.decode(*(cut(t, s, s + 1) for t in (q1, q2, k1, k2, v)), cache)
        assert not y.requires_grad
        for i in range(b):
            for j in range(h):
                want, w, dy, _ = ref.attend(*(t[i, j, s].double() for t in (q1, q2)), *(t[i, j, :s + 1].double() for t in (k1, k2, v)), lam, 0.8, True,
                                            core.gain.detach(), dt)
                assert bool(((y[i, j, 0].double() - want).abs() <= dy + 2 * ref.U32 * want.abs()).all())
                gathered[i, j, :s + 1] += w
        m = oracle.error_metrics(y.float().cpu(), whole[:, :, s:s + 1].float().cpu())
        assert m["rel_l2"] <= (1e-3 if dt == torch.float16 else 8e-3) * 2, m       # the forward's own bound, and the rounding of y
    assert torch.allclose(cache.weights[..., :n + steps].double(), gathered, rtol=1e-4, atol=1e-6)
    cache.evict(40, recent=8)
    keep = cache.positions[..., :40].long()
    assert bool((torch.sort(keep, -1).values[..., -8:] == torch.arange(n + steps - 8, n + steps, device=DEV)).all())
    q = queries(b, h, d, dt, seed=18)
    with torch.no_grad():
        y = cache.attend(q[0], q[1], torch.tensor([lam], device=DEV), 0.8, True, gain=core.gain)
    for i in range(b):
        for j in range(h):
            at = keep[i, j]
            want, _, dy, _ = ref.attend(q[0][i, j, 0].double(), q[1][i, j, 0].double(), *(t[i, j, at].double() for t in (k1, k2, v)), lam, 0.8, True,
                                        core.gain.detach(), dt)
            assert bool(((y[i, j, 0].double() - want).abs() <= dy + 2 * ref.U32 * want.abs()).all())
    pkg.device_status(0)


def test_refusals(pkg):
    c = make(pkg, [10, 20], 2, 64, 16, track=True, room=4)
    q1, q2, k1, k2, v = queries(2, 2, 64, torch.float16)
    lam = torch.tensor([0.5], device=DEV)
    for bad, err in ((dict(q1=q1.bfloat16()), ValueError), (dict(q1=q1[:1]), ValueError), (dict(q2=q2.cpu()), RuntimeError), (dict(q1=None), TypeError),
                     (dict(lambda_scale=0.5), TypeError), (dict(lambda_scale=torch.zeros(2, device=DEV)), ValueError), (dict(gain=torch.ones(64, device=DEV)), ValueError),
                     (dict(k1=k1), TypeError), (dict(k1=k1, k2=k2, v=v[..., :64]), ValueError), (dict(q1=q1.clone().requires_grad_()), RuntimeError),
                     (dict(lambda_scale=lam.clone().requires_grad_()), RuntimeError)):
        before = snapshot(c)
        with pytest.raises(err):
            c.attend(**{**dict(q1=q1, q2=q2, lambda_scale=lam), **bad})
        assert all(torch.equal(a, w) for a, w in zip(snapshot(c), before))
    for keep, recent in ((0, 0), (c.slots + 1, 0), (5, 6), (5, -1)):
        with pytest.raises(ValueError):
            c.evict(keep, recent)
    with pytest.raises(ValueError):
        c.append(k1, k2, v, torch.ones(3, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError):
        c.append(k1, k2, v, torch.ones(2, device=DEV))
    with pytest.raises(ValueError):
        c.append(k1, k2, v[:, :, :0])
    take = pkg.DiffAttnCache.from_tensors
    good = (c.k1_pages, c.k2_pages, c.v_pages, c.page_table, c.lengths)
    for i, t, err in ((0, c.k1_pages[:1].expand(4, -1, -1, -1), ValueError), (1, c.k2_pages[:-1], ValueError), (2, c.v_pages[..., :64], ValueError),
                      (0, c.k1_pages.float(), ValueError), (3, c.page_table.long(), ValueError), (4, c.lengths.long(), ValueError), (3, c.page_table.cpu(), RuntimeError)):
        with pytest.raises(err):
            take(*(t if i == k else x for k, x in enumerate(good)))
    flat = torch.zeros(64 * 200, dtype=torch.float16, device=DEV)
    lapped = flat.as_strided((2, 2, 16, 64), (2048, 32, 64, 1))       # heads half a row apart
    with pytest.raises(ValueError):
        take(lapped, lapped, torch.zeros(2, 2, 16, 128, dtype=torch.float16, device=DEV), c.page_table, c.lengths)
    with pytest.raises(ValueError):
        take(c.k1_pages[:0], c.k2_pages[:0], c.v_pages[:0], c.page_table, c.lengths)
    with pytest.raises(ValueError):
        pkg.DiffAttnCache(5000, 1, 32, 16, device=DEV)
    column = take(*good[:3], c.page_table[:, :1], c.lengths)           # (a column of a wider table: rows of one entry)
    assert column.slots == 16
    with pytest.raises(ValueError):
        take(*good, positions=c.positions)
    with pytest.raises(ValueError):
        take(*good, weights=c.weights[:, :, :-1])
    with pytest.raises(ValueError):
        take(*good).evict(5)                              # without positions nothing can be evicted
    with pytest.raises(ValueError):
        pkg.DiffAttnCache(1, 1, 48, 10)
    pkg.device_status(0)


def test_empty_calls(pkg):
    c = pkg.DiffAttnCache(0, 4, 64, 100, device=DEV)
    q1, q2, k1, k2, v = queries(0, 4, 64, torch.float16)
    assert c.attend(q1, q2, torch.tensor([0.5], device=DEV), k1=k1, k2=k2, v=v).shape == (0, 4, 1, 128)
    c.append(k1, k2, v)
    c.evict(5)
    c = pkg.DiffAttnCache(2, 2, 64, 100, device=DEV)
    q1, q2, k1, k2, v = queries(2, 2, 64, torch.float16, t=0)
    c.append(k1, k2, v)
    q1, q2, k1, k2, v = queries(2, 2, 64, torch.float16)
    assert int(c.lengths.sum()) == 0 and not bool(c.attend(q1, q2, torch.tensor([0.5], device=DEV)).any())
    pkg.device_status(0)
