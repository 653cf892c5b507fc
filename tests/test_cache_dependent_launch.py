"""The cache's kernels start before the grid ahead of them has ended: in each of them every thread has to wait for that grid before it touches
global memory.  Read off the source: a missing wait gives right results nearly always."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "triton_diff_attn_b200", "csrc")


def _source(name):
    return re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())


def _kernels():
    found = []
    for name in ("cache.cuh", "cache_attend.cuh", "cache_evict.cuh"):
        text = _source(name)
        for m in re.finditer(r"__global__", text):
            rest = text[m.start():]
            kernel = re.search(r"\b(diffattn_cache_\w+)\(", rest).group(1)
            body = rest[rest.index("{\n"):]
            found.append((kernel, body[:body.index("\n}\n")]))
    return found


KERNELS = _kernels()
# what reads or writes global memory: the arguments' pointers, the functions that use them, copies by the engine
TOUCHES = (r"\b(?:a|c|a\.c)\.(?:page_table|lengths|next_position|counter|positions|weights|k1|k2|v|q1|q2|nk1|nk2|nv|counts|lambda_ptr|gain|y|prefix|length|position|stats"
           r"|acc|scores|count|moves)\b|\b(?:lengths|next_position)\[|cache_|append_|attend_|join|walk_|load_lambda|place_row|move_rows|evict_key|bulk_load|tma_load|mbar_wait|mbar_expect|atomic")


def test_all_of_them_are_here():
    assert sorted(k for k, _ in KERNELS) == ["diffattn_cache_advance_kernel", "diffattn_cache_append_kernel", "diffattn_cache_attend_kernel",
                                             "diffattn_cache_join_few_kernel", "diffattn_cache_join_kernel", "diffattn_cache_move_kernel",
                                             "diffattn_cache_reset_kernel", "diffattn_cache_select_kernel"]
    launched = set(re.findall(r"da::(diffattn_cache_\w+)", _source("cache_host.cuh")))
    assert launched == {k for k, _ in KERNELS}


@pytest.mark.parametrize("kernel,body", KERNELS, ids=[k for k, _ in KERNELS])
def test_every_thread_waits_first(kernel, body):
    ahead, _, behind = body.partition("\n  griddep_wait();\n")      # (two spaces: in no branch, in no role)
    assert behind and "griddep_wait" not in ahead + behind
    assert not re.search(r"\breturn\b", ahead)
    assert not re.search(TOUCHES, ahead), re.search(TOUCHES, ahead).group(0)
    assert re.search(TOUCHES, behind)
    # the grid behind may start only once this one has passed its own wait, so that what it waits for includes what this one waited for
    assert "griddep_launch" not in ahead and behind.startswith("  griddep_launch();\n")


def test_the_check_sees_a_missing_wait():
    kernel, body = KERNELS[0]
    assert re.search(TOUCHES, body.replace("  griddep_wait();\n", "", 1).partition("\n  griddep_wait();\n")[0])
