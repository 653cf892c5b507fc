"""The key-value cache's tensors and contents that a user can hand over, and what must not come of them."""
import math

import pytest
import torch

from test_cache_gpu import DEV, make, queries, snapshot

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
