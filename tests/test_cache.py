"""CPU tests of the key-value cache: the ABI's struct and its refusals, and the walk of its attention kernel over tiles, pages and pieces on a
model of it in plain Python (the same arithmetic, for every kind of page and length)."""
import ctypes
import os
import random
import re
import shutil
import subprocess

import pytest
import torch

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def L():
    from triton_diff_attn_b200 import _lib
    return _lib


def _good(L, d=64):
    p = L.DiffAttnCacheParams()
    p.struct_size = ctypes.sizeof(p)
    p.B, p.H, p.D, p.page_size, p.num_pages, p.max_pages, p.T = 2, 3, d, 16, 9, 4, 5
    p.kp_stride_slot, p.kp_stride_head, p.kp_stride_page = d, 16 * d, 48 * d
    p.vp_stride_slot, p.vp_stride_head, p.vp_stride_page = 2 * d, 32 * d, 96 * d
    p.k_stride_t, p.k_stride_h, p.k_stride_b = d, 5 * d, 15 * d
    p.v_stride_t, p.v_stride_h, p.v_stride_b = 2 * d, 10 * d, 30 * d
    p.q_stride_h, p.q_stride_b, p.table_stride = d, 3 * d, 4
    for f in ("k1_pages", "k2_pages", "v_pages", "page_table", "lengths", "next_position", "positions", "k1", "k2", "v", "q1", "q2", "lambda_scale", "y", "workspace", "counter"):
        setattr(p, f, 0x10000)          # never dereferenced: every check below fails before a launch
    p.lambda_dtype, p.keep, p.recent, p.workspace_bytes = 1, 8, 2, 1 << 40
    return p


ALL = ("append", "attend", "evict")
BAD = [
    (ALL, "struct_size", 8, -2), (ALL, "D", 48, -4), (ALL, "B", -1, -3), (ALL, "B", 5000, -3), (ALL, "H", 40000, -3), (ALL, "page_size", 0, -3),
    (ALL, "num_pages", 0, -3), (ALL, "max_pages", 0, -3), (ALL, "max_pages", 2 ** 28, -3), (ALL, "io_dtype", 2, -7), (ALL, "k1_pages", 0, -1),
    (ALL, "page_table", 0, -1), (ALL, "lengths", 0, -1), (ALL, "v_pages", 0x10008, -6), (ALL, "kp_stride_head", 60, -5), (ALL, "kp_stride_page", 0, -5),
    (ALL, "vp_stride_slot", 64, -5), (ALL, "table_stride", 3, -5), (ALL, "positions", 0, -1), (ALL, "device", 64, -3), (ALL, "device", -1, -3),
    (("append",), "T", -1, -3), (("append", "attend"), "k2", 0, -1), (("append", "attend"), "v", 0x10008, -6), (("append", "attend"), "v_stride_h", 12, -5),
    (("append", "evict"), "counter", 0, -1), (ALL, "counter", 0x10002, -6), (("append",), "T", 2 ** 31 - 1, -3), (("append", "attend"), "counts", 0x10002, -6), (ALL, "lengths", 0x10002, -6), (ALL, "page_table", 0x10001, -6),
    (ALL, "weights", 0x10002, -6), (("attend",), "y", 0x10002, -6), (("attend",), "gain", 0x10002, -6), (("attend",), "lambda_scale", 0x10002, -6),
    (("append",), "k_stride_t", 0, -5), (("attend",), "q1", 0, -1), (("attend",), "q2", 0x10004, -6), (("attend",), "q_stride_h", 4, -5),
    (("attend",), "lambda_dtype", 9, -7), (("attend",), "y", 0, -1), (("attend",), "lambda_scale", 0, -1),
    (("evict",), "keep", 0, -3), (("evict",), "keep", 65, -3), (("evict",), "recent", 9, -3), (("evict",), "recent", -1, -3),
]


@pytest.mark.parametrize("calls,field,value,code", BAD)
def test_refusals(L, calls, field, value, code):
    for call in calls:
        p = _good(L)
        setattr(p, field, value)
        assert getattr(L.lib, "diffattn_cache_" + call)(p) == code, (call, L.last_error())
        assert L.last_error()
    assert L.lib.diffattn_cache_attend(None) == -1


def test_empty_and_workspace_sizes(L):
    for call in ALL:
        p = _good(L)
        p.B = 0
        assert getattr(L.lib, "diffattn_cache_" + call)(p) == 0
    p = _good(L)
    size = lambda op: L.lib.diffattn_cache_workspace_bytes(p, op)
    assert size(L.CACHE_APPEND) == 0 and size(7) == 0
    assert size(L.CACHE_EVICT) == 0                       # few moves: the selecting kernel keeps them
    plain = size(L.CACHE_ATTEND)
    p.weights = 0x10000
    assert size(L.CACHE_ATTEND) - plain == 5 * 6 * 2 * 16 * 4      # four tiles of 16 tokens and the new token's, two scores each
    p.max_pages, p.keep = 64, 500                         # 500 of 1024 slots: a list of moves, counts of them
    assert size(L.CACHE_EVICT) == 256 + -(-8 * 6 * 500 // 256) * 256
    p.keep = 0
    assert size(L.CACHE_EVICT) == 0
    assert L.lib.diffattn_cache_reset(0, None, 0, None, None) == 0
    assert L.lib.diffattn_cache_reset(0, None, -1, 0x10000, None) == -3 and L.lib.diffattn_cache_reset(0, None, 2, None, None) == -1
    assert L.lib.diffattn_cache_reset(0, None, 2, 0x10002, None) == -6 and L.lib.diffattn_cache_reset(64, None, 2, 0x10000, None) == -3


def test_struct_matches_the_header(L, tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    names = [n for n, _ in L.DiffAttnCacheParams._fields_]
    src = tmp_path / "o.c"
    src.write_text('#include "diffattn.h"\n#include <stdio.h>\nint main(void){' +
                   "".join(f'printf("%zu ",offsetof(DiffAttnCacheParams,{n}));' for n in names) + 'printf("%zu",sizeof(DiffAttnCacheParams));return 0;}')
    subprocess.run([cc, "-I", os.path.join(REPO, "include"), "-o", str(tmp_path / "o"), str(src)], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "o")], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [getattr(L.DiffAttnCacheParams, n).offset for n in names] + [ctypes.sizeof(L.DiffAttnCacheParams)]


def test_no_cpu_path():
    import triton_diff_attn_b200 as pkg
    t = torch.zeros(2, 1, 16, 64, dtype=torch.float16)
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        pkg.DiffAttnCache.from_tensors(t, t, torch.zeros(2, 1, 16, 128, dtype=torch.float16), i.view(1, 1), i)
    with pytest.raises(TypeError):
        pkg.DiffAttnCache.from_tensors(None, t, t, i.view(1, 1), i)
    with pytest.raises(ValueError):
        pkg.DiffAttnCache(1, 1, 64, 0)


# ---- the walk over tiles, as csrc/cache_attend.cuh and cache_host.cuh have it -------------------------------------------------------------
def tile_shape(d, page):
    t = 32 if d == 32 else 16
    r = t
    while page % r:
        r //= 2
    per_page = -(-page // t)
    if r >= 8:
        return t, r, 0
    if 10 * per_page * t <= page * {4: 13, 2: 15, 1: 20}[r] or r * (64 if d == 32 else 128) < 128:
        return t, t, per_page
    return t, r, 0


def tiles_of(n, page, shape):
    t, _, per_page = shape
    if not per_page:
        return -(-n // t)
    full = n // page
    return full * per_page + -(-(n - full * page) // t)


def tile_at(i, n, page, shape):
    t, _, per_page = shape
    slot, end = i * t, n
    if per_page:
        p = i // per_page
        slot, end = p * page + (i - p * per_page) * t, min(n, (p + 1) * page)
        new = i >= tiles_of(n, page, shape)
    else:
        new = slot >= n
    return (n, 1, True) if new else (slot, min(t, end - slot), False)


@pytest.mark.parametrize("d", [32, 64, 128])
def test_tiles_cover_every_token_once(d):
    for page in list(range(1, 40)) + [48, 64, 100, 128, 1000]:
        shape = tile_shape(d, page)
        t, box, per_page = shape
        assert t % box == 0 and box * (64 if d == 32 else 128) % 128 == 0 and (per_page or page % box == 0)
        for n in list(range(0, 3 * t + 2)) + [page - 1, page, page + 1, 4 * page, 4 * page + 1]:
            for token in (0, 1):
                m, seen = tiles_of(n, page, shape) + token, []
                for i in range(m):
                    slot, valid, new = tile_at(i, n, page, shape)
                    assert 1 <= valid <= t
                    assert new == (token == 1 and i == m - 1)
                    if new:
                        assert slot == n
                        continue
                    boxes = [lane for lane in range(32) if lane * box < valid]
                    assert len(boxes) * box <= t
                    for row in range(valid):
                        start = slot + row // box * box          # the box's first slot
                        entry, in_page = divmod(start, page)
                        assert row // box in boxes and entry * page + in_page + row % box == slot + row
                        assert in_page + row % box < page and entry <= (n - 1) // page
                        seen.append(slot + row)
                assert seen == list(range(n))
        # the bound that the workspace is sized by
        slots = 4 * page
        most = (4 * per_page if per_page else -(-slots // t)) + 1
        assert max(tiles_of(n, page, shape) + 1 for n in range(slots + 1)) <= most


def test_pieces_of_the_line():
    """Every tile belongs to one worker, a piece's place is its own and inside the workspace, the joining kernel finds exactly the pieces."""
    rng = random.Random(4)
    for _ in range(300):
        b, h, all_workers = rng.randint(1, 9), rng.randint(1, 5), rng.choice([8, 24, 1184])
        tiles = [rng.choice([0, 0, 1, 2, rng.randint(0, 40), rng.randint(0, 900)]) for _ in range(b)]
        prefix = [0]
        for n in tiles:
            prefix.append(prefix[-1] + n)
        units = prefix[-1] * h
        workers = min(all_workers, units)
        if units == 0:
            continue
        line = [(i * h + j) for i in range(b) for j in range(h) for _ in range(tiles[i])]
        place, pieces = {}, {}
        for w in range(workers):
            lo, hi = units * w // workers, units * (w + 1) // workers
            assert hi > lo
            for u in range(lo, hi):
                # walk_at: the last sequence whose tiles begin at or before u
                seq = max(i for i in range(b) if prefix[i] * h <= u)
                r = u - prefix[seq] * h
                assert seq * h + r // tiles[seq] == line[u]
                pieces.setdefault(line[u], set()).add(w)
        for bh, ws in pieces.items():
            for w in ws:
                at = w + bh
                assert at not in place and at < all_workers + b * h
                place[at] = (w, bh)
            seq, head = divmod(bh, h)
            u = prefix[seq] * h + head * tiles[seq]
            w0, w1 = ((u + 1) * workers - 1) // units, ((u + tiles[seq]) * workers - 1) // units
            assert ws == set(range(w0, w1 + 1))


def test_page_of_a_slot_without_division():
    rng = random.Random(1)
    for page in [2, 3, 5, 7, 16, 24, 100, 999, 4096, 2 ** 20 + 7, 2 ** 30]:
        magic = (2 ** 32 + page - 1) // page
        assert magic < 2 ** 32
        for slot in [0, 1, page - 1, page, 2 ** 31 - 1 - page, *(rng.randrange(2 ** 31 - page) for _ in range(200))]:
            p = (slot * magic) >> 32
            if p * page > slot:
                p -= 1
            assert p == slot // page


def test_header_names_the_error():
    hdr = open(os.path.join(REPO, "include", "diffattn.h")).read()
    from triton_diff_attn_b200 import _lib
    assert "DIFFATTN_ERR_BAD_CACHE = -12" in hdr and _lib.ERR_NAMES[-12] == "BAD_CACHE" and -12 in _lib.VALUE_ERRORS
    assert re.search(r"typedef struct DiffAttnCacheParams", hdr)
