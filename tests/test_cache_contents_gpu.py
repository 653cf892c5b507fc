"""The key-value cache's tensors and contents that a user can hand over, and what must not come of them."""
import math

import pytest
import torch

from test_cache_gpu import DEV, check_attend, make, queries, snapshot

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pkg():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import triton_diff_attn_b200
    return triton_diff_attn_b200


def test_a_cache_made_in_a_capture(pkg):
    """Calls on it outside the graph, before its first replay and after, move the lengths on as those in the graph do."""
    c0 = make(pkg, [5, 20], 2, 64, 16, track=True, room=28, seed=1)
    state = (c0.k1_pages, c0.k2_pages, c0.v_pages, c0.page_table, c0.lengths)
    more = dict(positions=c0.positions, next_position=c0.next_position, weights=c0.weights)
    q1, q2, k1, k2, v = queries(2, 2, 64, torch.float16, seed=1)
    c0.append(k1, k2, v)
    torch.cuda.synchronize()
    pool = torch.cuda.graph_pool_handle()
    soil = torch.cuda.CUDAGraph()
    with torch.cuda.graph(soil, pool=pool):              # what lies in the graphs' memory is not 0
        dirt = [torch.full((64,), 7, dtype=torch.int32, device=DEV) for _ in range(64)]
    soil.replay()
    torch.cuda.synchronize()
    del dirt
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, pool=pool):
        c = pkg.DiffAttnCache.from_tensors(*state, **more)
        c.append(k1, k2, v)
        c.evict(18)
    assert c.lengths.tolist() == [6, 21]
    for eager in (True, False, True, False):
        c.lengths.copy_(torch.tensor([6, 18], dtype=torch.int32))
        if eager:
            c.append(k1, k2, v)
            assert c.lengths.tolist() == [7, 19]
            c.evict(18)
        else:
            graph.replay()
        assert c.lengths.tolist() == [7, 18]
    pkg.device_status(0)


def test_state_that_shares_memory_is_refused(pkg):
    """`append` would count twice what is both a length and a next position."""
    c = make(pkg, [5, 20], 2, 64, 16, track=True, room=4)
    pools = (c.k1_pages, c.k2_pages, c.v_pages, c.page_table)
    take = pkg.DiffAttnCache.from_tensors
    both = torch.zeros(3, dtype=torch.int32, device=DEV)
    for lengths, following, positions, weights in (
            (c.lengths, c.lengths, c.positions, None), (both[:2], both[1:], c.positions, None),
            (c.lengths, c.positions.view(-1)[:2], c.positions, None), (c.lengths, c.next_position, c.positions, c.positions.view(torch.float32))):
        with pytest.raises(ValueError, match="share memory"):
            take(*pools, lengths, positions=positions, next_position=following, weights=weights)
    state = torch.zeros(4, dtype=torch.int32, device=DEV)      # neighbours do not
    take(*pools, state[:2], positions=c.positions, next_position=state[2:], weights=c.weights).reset()
    empty = torch.zeros(0, dtype=torch.int32, device=DEV)
    take(*pools[:3], c.page_table[:0], empty, positions=c.positions[:0], next_position=empty)
    pkg.device_status(0)


def test_a_page_table_wider_than_32_bits_is_refused(pkg):
    """It would be taken for one of as many columns as its lowest 32 bits say."""
    pools = tuple(torch.zeros(2, 1, 16, w, dtype=torch.float16, device=DEV) for w in (64, 64, 128))
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    for columns in (2 ** 32 + 4, 2 ** 31, 2 ** 27):      # (the last: too many slots)
        with pytest.raises(ValueError, match="too long"):
            pkg.DiffAttnCache.from_tensors(*pools, none.new_empty(0, columns), none)
    assert pkg.DiffAttnCache.from_tensors(*pools, none.new_empty(0, 4), none).slots == 64


@pytest.mark.parametrize("bad", [0, 1])
@pytest.mark.parametrize("what,call", [("page", "attend"), ("page", "token"), ("page", "append"), ("page", "evict"), ("length", "attend"), ("length", "token"),
                                       ("length", "append"), ("length", "evict"), ("negative", "attend"), ("negative", "token"), ("negative", "evict"),
                                       ("full", "token"), ("full", "append")])
def test_a_bad_sequence_leaves_the_others_alone(pkg, what, call, bad):
    """One sequence's length or page is bad, or it is full: the other one gets what a call without that gives it, and of the bad one only
    slots that the call may write for it change."""
    good, h, page, keep, t = 1 - bad, 2, 16, 39, 2
    lengths = [0, 0]
    lengths[bad], lengths[good] = 48 if what == "full" else 40, 45
    q1, q2, k1, k2, v = queries(2, h, 64, torch.float16, seed=2)
    rows = queries(2, h, 64, torch.float16, seed=3, t=t)[2:]
    lam = torch.tensor([0.5], device=DEV)

    def run(fault):
        c = make(pkg, [48, 48], h, 64, page, track=True, seed=5)      # (the same pages and rows, whatever the lengths)
        c.lengths.copy_(torch.tensor(lengths, dtype=torch.int32)); c.next_position.copy_(c.lengths)
        for i in range(2):
            c.weights[i, :, lengths[i]:].fill_(7.0)
        names = c.page_table.clone()
        if fault and what == "page":
            c.page_table[bad, 0 if call in ("attend", "evict") else 2] = 2 ** 30
        elif fault and what in ("length", "negative"):
            c.lengths[bad] = 49 if what == "length" else -3
        c.weights[bad, :, 1:48] = 1.0
        c.weights[bad, :, 0] = 0.0                        # the first slot is a hole
        before = snapshot(c)
        old = {"weights": c.weights.clone()}
        y = None
        if call == "attend":
            y = c.attend(q1, q2, lam)
        elif call == "token":
            y = c.attend(q1, q2, lam, k1=k1, k2=k2, v=v)
        elif call == "append":
            c.append(*rows)
        else:
            c.evict(keep)
        if fault:
            with pytest.raises(ValueError, match="BAD_CACHE"):
                pkg.device_status(0)
        pkg.device_status(0)
        return c, names, before, snapshot(c), y, old

    c, names, before, after, y, old = run(True)
    lengths[bad] = 40
    want = run(False)[3]
    mine, other = names[bad].tolist(), names[good].tolist()
    for a, b, w in zip(after[:3], before[:3], want[:3]):
        for p in range(a.shape[0]):
            if p in other:
                assert torch.equal(a[p], w[p])
            elif p not in mine:
                assert torch.equal(a[p], b[p])
    for i in (3, 4, 5):                                   # lengths, next_position, positions
        assert torch.equal(after[i][good], want[i][good])
    if y is None:
        assert torch.equal(after[6][good], want[6][good])
    else:                                                 # (its tiles are split among other warps than in a call without the fault)
        sub = type("C", (), dict(k1_pages=c.k1_pages, k2_pages=c.k2_pages, v_pages=c.v_pages, page_table=names[good:good + 1], weights=c.weights[good:good + 1]))
        check_attend(sub, {"weights": old["weights"][good:good + 1]}, y[good:good + 1], q1[good:good + 1], q2[good:good + 1], 0.5, [45],
                     tuple(x[good:good + 1] for x in (k1, k2, v)) if call == "token" else None, rms=False)
        behind = 46 if call == "token" else 45
        assert torch.equal(after[6][good, :, behind:], before[6][good, :, behind:])
    # the bad one: [first, end) are the slots that its call may write rows in, by the length it counts with
    n = {"page": 40, "full": 48, "length": 48, "negative": 0}[what]
    first, end = {"attend": (0, 0), "token": (n, n + 1), "append": (n, n + t), "evict": (0, keep if n > keep else 0)}[call]
    for entry, p in enumerate(mine):
        named = int(c.page_table[bad, entry]) == p
        for s in range(page):
            slot = entry * page + s
            if not (named and first <= slot < end):
                assert all(torch.equal(a[p, :, s], b[p, :, s]) for a, b in zip(after[:3], before[:3])), slot
    for s in range(48):
        if not first <= s < end:
            assert torch.equal(after[5][bad, :, s], before[5][bad, :, s])
            if call in ("append", "evict") or s >= n:     # (attention adds to the weights of all live slots)
                assert torch.equal(after[6][bad, :, s], before[6][bad, :, s])
