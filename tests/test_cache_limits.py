"""The longest cache that the library admits: every step that its kernels add to a slot's or a tile's number in 32 bits has to fit."""
import ctypes
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "triton_diff_attn_b200", "csrc")
MAX = 2 ** 31 - 1
CALLS = ("append", "attend", "evict")


@pytest.fixture(scope="module")
def L():
    from triton_diff_attn_b200 import _lib
    return _lib


def _params(L, d, page, max_pages, h=1):
    p = L.DiffAttnCacheParams()
    p.struct_size = ctypes.sizeof(p)
    p.B, p.H, p.D, p.page_size, p.num_pages, p.max_pages, p.T = 1, h, d, page, 1, max_pages, 1
    p.kp_stride_slot, p.kp_stride_head, p.vp_stride_slot, p.vp_stride_head = d * h, d, 2 * d * h, 2 * d
    p.k_stride_h = p.q_stride_h = d
    p.v_stride_h = 2 * d
    p.table_stride, p.lambda_dtype, p.keep, p.workspace_bytes = max_pages, 1, 8, 1 << 60
    p.device = 63            # no such device: a call that passes the checks of sizes ends there, with another code
    for f in ("k1_pages", "k2_pages", "v_pages", "page_table", "lengths", "next_position", "positions", "k1", "k2", "v", "q1", "q2", "lambda_scale", "y", "workspace", "counter"):
        setattr(p, f, 0x10000)
    return p


def _constant(name, text):
    return int(re.search(r"\b%s = (\d+)" % name, text).group(1))


def _steps():
    """The largest numbers that the kernels add to a slot (eviction: loads ahead, runs of 31) and to a tile (joining: a round of every share of a
    (sequence, head), with one of them on a GPU of up to 256 SMs)."""
    evict = open(os.path.join(CSRC, "cache_evict.cuh")).read()
    threads, ahead = _constant("SELECT_THREADS", evict), _constant("SELECT_AHEAD", evict)
    assert "i0 += SELECT_THREADS * SELECT_AHEAD" in evict and "c0 += 31 * SELECT_THREADS" in evict
    attend = open(os.path.join(CSRC, "cache_attend.cuh")).read()
    rounds = _constant("ROUND", attend)
    assert "t0 += shares * (JT / T) * ROUND" in attend
    return max(2 * threads * ahead, 31 * threads), 256 * 2 * (1024 // 16) * rounds


@pytest.mark.parametrize("page", [1, 7, 16, 4096])
def test_slots_near_the_end_of_32_bits(L, page):
    slot_step, _ = _steps()
    for call in CALLS:
        p = _params(L, 64, page, (MAX - slot_step) // page + 1)
        assert getattr(L.lib, "diffattn_cache_" + call)(p) == -3, call
        assert "too long" in L.last_error()
    assert L.lib.diffattn_cache_workspace_bytes(p, L.CACHE_ATTEND) == 0


def test_tiles_near_the_end_of_32_bits(L):
    """Head dim 32 with pages of one slot: a tile per slot."""
    _, tile_step = _steps()
    p = _params(L, 32, 1, MAX - tile_step)
    for call in CALLS:
        assert getattr(L.lib, "diffattn_cache_" + call)(p) == -3, call
        assert "too long" in L.last_error()


@pytest.mark.parametrize("d,page,max_pages", [(64, 16, 2 ** 26), (64, 1, 2 ** 30), (32, 1, 2 ** 30), (128, 2 ** 29, 2)])
def test_half_of_them_is_admitted(L, d, page, max_pages):
    p = _params(L, d, page, max_pages)
    for call in CALLS:
        assert getattr(L.lib, "diffattn_cache_" + call)(p) == -9, call      # (the device)
