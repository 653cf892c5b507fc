"""Eviction in a batch of so many (sequence, head)s that the selecting kernel carries its moves out, few and many, and of a few less."""
import pytest
import torch

import cache_reference as ref
from test_cache_gpu import DEV, make, snapshot

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pkg():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import triton_diff_attn_b200
    return triton_diff_attn_b200


@pytest.mark.parametrize("heads_per_sm", [1, 2.9, 3.1])
@pytest.mark.parametrize("d,page,longest,keep,recent", [(32, 16, 400, 200, 7), (64, 64, 1150, 530, 0), (128, 7, 300, 100, 100)])
def test_evict_from_many(pkg, heads_per_sm, d, page, longest, keep, recent):
    h = 5
    b = round(heads_per_sm * torch.cuda.get_device_properties(0).multi_processor_count / h)
    lengths = [longest - (37 * i) % (longest + 1) for i in range(b)]
    c = make(pkg, lengths, h, d, page, track=True, seed=d, first_position=2)
    before = snapshot(c)
    c.evict(keep, recent)
    pkg.device_status(0)
    assert c.lengths.tolist() == [min(n, keep) for n in lengths]
    after, w, p = snapshot(c), before[6].view(torch.float32).cpu(), before[5].cpu()
    at = torch.arange(c.slots, device=DEV)
    pages = c.page_table.long().clamp(0, c.k1_pages.shape[0] - 1)
    for i in sorted({0, 1, b // 3, b // 2, b - 2, b - 1}):
        n = lengths[i]
        for j in (0, h - 1):
            source = torch.arange(c.slots)
            for to, frm in ref.evict(w[i, j], p[i, j], n, n + 2, keep, recent):
                source[to] = frm
            source = source.to(DEV)
            live = at < n                                  # (behind it the table names no pages)
            for x, y in zip(after[:3], before[:3]):
                rows = lambda t, s: t[pages[i][s // page], j, s % page]
                assert torch.equal(rows(x, at[live]), rows(y, source[live]))
            for x, y in zip(after[5:], before[5:]):
                assert torch.equal(x[i, j], y[i, j][source])
    # everywhere: as many rows, and the weights that stay are the largest
    old, new = before[6].view(torch.float32), after[6].view(torch.float32)
    for i, n in enumerate(lengths):
        if n > keep and recent == 0:
            assert torch.equal(new[i, :, :keep].sort(-1).values, old[i, :, :n].sort(-1).values[:, n - keep:])
        elif n <= keep:
            assert all(torch.equal(x[i], y[i]) for x, y in zip(after[5:], before[5:]))
