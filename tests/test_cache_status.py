"""Reports of the cache's kernels and of waits that gave up do not hide each other (read off the source: no call makes a wait give up)."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "triton_diff_attn_b200", "csrc")


def _source(name):
    return re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())


def test_cache_reports_have_a_word_of_their_own():
    for name in ("cache.cuh", "cache_attend.cuh", "cache_evict.cuh"):
        assert not re.search(r"\bg_status\b", _source(name)), name
    fault = _source("cache.cuh").split("void cache_fault(", 1)[1].split("\n}", 1)[0]
    assert "atomicCAS(&g_cache_status[0], 0" in fault


def test_a_wait_that_gave_up_is_reported_first_and_clears_nothing_else():
    body = _source("diffattn.cu").split("int diffattn_status(", 1)[1].split("\n}", 1)[0]
    wait = body.index("DIFFATTN_ERR_TIMEOUT")
    assert "g_cache_status" not in body[:wait] and "DIFFATTN_ERR_BAD_CACHE" not in body[:wait]
    assert not re.search(r"\bg_status\b", body[wait:])
