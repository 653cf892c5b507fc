"""Probabilities far below the largest one: what a long cache's many small ones sum up to has to reach the output, whatever takes the largest."""
import math

import pytest
import torch

import cache_reference as ref

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


@pytest.fixture(scope="module")
def pkg():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import triton_diff_attn_b200
    return triton_diff_attn_b200


def bound(p1, p2, v, lam, big, n, io):
    """How far A = P1 V - lam P2 V may be off before the norm.  With u = 2^-24 and sums that may cut off (2 u per addition): a score is one exact
    product, scaled once, so a probability is off by a factor exp(+-2 u * 12 * S) as in `cache_reference.attend` (S: the largest score); a lane's sums are
    chains of at most n / 4 + 64 additions in the product and n / 8 + 64 in the row sum, each of which loses at most 2 u of what it has
    so far.  What the 16-bit pair of a probability loses: its two roundings, (eps / 2)^2 of it, in fp16 at least half of the smallest step, 2^-25, of
    a second number that is kept 2^11 times larger than it is, beside a largest probability kept as 2^7 or more: 2^-43 of the largest one."""
    info = torch.finfo(io)
    rel = 4.0 * ref.U32 * (12 * big + 64 + n / 4)
    da = (rel + 2 * (info.eps / 2) ** 2) * ((p1 + abs(lam) * p2) @ v.abs())
    if io == torch.float16:
        da = da + 2.0 ** -43 * (float(p1.max()) + abs(lam) * float(p2.max())) * v.abs().sum(0)
    return da


@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("d,n,dt,below", [
    (64, 16384, torch.float16, (12.75, 12.75)), (32, 5000, torch.float16, (13.0, 13.0)), (128, 3001, torch.float16, (12.0, 16.0)),
    (64, 16384, torch.float16, (17.4, 17.6)),      # each below 2^-25 of the largest
    (32, 16384, torch.float16, (20.0, 21.0)),      # each below 2^-28
    (64, 16384, torch.bfloat16, (17.4, 17.6)),
])
def test_many_small_probabilities(pkg, d, n, dt, below, rms):
    """The first token takes the weight and has V = 0; the others lie `below` (natural logarithms) it and are all that the output holds.  So many sequences
    (on the same pages) that a warp walks through all tokens of one."""
    b, page = 1300, 64
    g = torch.Generator(device=DEV); g.manual_seed(n + d)
    rand = lambda *s: torch.rand(s, generator=g, device=DEV)
    pages, root = -(-n // page), math.sqrt(d)
    k = torch.zeros(2, pages, 1, page, d, device=DEV)
    k[..., 0] = -(below[0] + (below[1] - below[0]) * rand(2, pages, 1, page)) * root
    v = (0.5 + rand(pages, 1, page, 2 * d)).to(dt)
    k[:, 0, :, 0] = 0
    v[0, :, 0] = 0
    k1, k2 = k.to(dt)
    q = torch.zeros(b, 1, 1, d, dtype=dt, device=DEV)
    q[..., 0] = 1
    table = torch.arange(pages, dtype=torch.int32, device=DEV).expand(b, -1).contiguous()
    c = pkg.DiffAttnCache.from_tensors(k1, k2, v, table, torch.full((b,), n, dtype=torch.int32, device=DEV))
    lam = 0.25
    y = c.attend(q, q, torch.tensor([lam], device=DEV), 0.8, rms)
    pkg.device_status(0)
    info = torch.finfo(dt)
    r1, r2, rv = (ref.rows(t, table[0], page, 0, n) for t in (k1, k2, v))
    s1, s2 = r1[:, 0] / root, r2[:, 0] / root
    p1, p2 = torch.softmax(s1, 0), torch.softmax(s2, 0)
    a = p1 @ rv - lam * (p2 @ rv)
    da = bound(p1, p2, rv, lam, float(torch.maximum(s1.abs().max(), s2.abs().max())), n, dt)
    if rms:
        s = 1.0 / math.sqrt(float((a * a).mean()) + 1e-5)
        da = 0.2 * s * (da + a.abs() * s * float((da * da).mean()) ** 0.5 + 8 * ref.U32 * a.abs())
        a = a * s * 0.2
    dy = da + (a.abs() + da) * info.eps / 2 + info.tiny * info.eps
    off = (y[:, 0, 0].double() - a).abs()
    assert bool((off <= dy).all()), (float((off / dy).max()), float((off / a.abs()).max()))
