"""The operators of the key-value cache (`DiffAttnCache`) as work to be measured: attention of one new token over a paged cache,
storing new tokens in it, eviction from it, and a generation step of all of them.

A case is a dict of plain values.  `kind`:
  attend  one query per (sequence, head) over the live tokens; `track`: the tokens' accumulated attention weights are updated too
  append  a prompt's tokens go into an empty cache
  evict   a chunk of `t` tokens is appended to a full cache of `n`, which is then cut back to `n`: the chunk stays and the tokens with
          the least accumulated weight go
  step    one token of generation with a window of `n` tokens: store and attend, then the oldest token goes
b, h, d: sequences, heads, head dim (the value width is 2 d).  n: tokens per sequence (the longest one's with `ragged`).  page: slots per page.
slot_major: pages are stored [page, slot, head, d] instead of [page, head, slot, d].  bf16: bfloat16 instead of float16.  gain: the output
norm has a learned gain.  Pages of a sequence lie anywhere in the pool, in any order.

With `own` false the operators are elementary tensor operations in 32 bits; with `own` true they are the framework's calls.
"""
import math

import torch

own = False

EPS = 1e-5
LAMBDA_INIT = 0.8
MOST_TOKENS = {"attend": 64 * 16 * 4096 * 64, "append": 8 * 16 * 4096 * 64, "evict": 8 * 16 * 4608 * 64, "step": 32 * 16 * 2048 * 64}   # b h n d


def _case(kind, b, h, n, d, *, t=1, page=64, ragged=False, slot_major=False, bf16=False, track=False, gain=True, rms=True, lam=0.5, name=None):
    c = dict(kind=kind, b=b, h=h, n=n, d=d, t=t, page=page, ragged=ragged, slot_major=slot_major, bf16=bf16, track=track, gain=gain, rms=rms, lam=lam)
    if name is not None:
        c["name"] = name
    return c


def listed():
    return [
        # the first tokens of an answer to a short prompt: launches and latency are all there is
        _case("attend", 1, 16, 77, 64, page=16, bf16=True, name="attend_b1h16n77d64"),
        # one user with a long document
        _case("attend", 1, 16, 16384, 64, name="attend_b1h16n16384d64"),
        # a full serving batch, sequences of every length, one of them not in use: the largest case
        _case("attend", 64, 16, 4096, 64, ragged=True, bf16=True, name="attend_b64h16n4096d64_ragged"),
        # wide heads, pages as a layer's projections leave them ([page, slot, head, d])
        _case("attend", 8, 8, 8192, 128, page=128, slot_major=True, bf16=True, lam=0.7, name="attend_b8h8n8192d128"),
        # the narrow head dim without the norm, a page size that is no power of two
        _case("attend", 16, 16, 2047, 32, page=24, gain=False, rms=False, name="attend_b16h16n2047d32"),
        # generation that keeps score for an eviction
        _case("attend", 8, 16, 4096, 64, track=True, bf16=True, name="attend_b8h16n4096d64_track"),
        # prompts of one length
        _case("append", 4, 16, 2048, 64, bf16=True, name="append_b4h16n2048d64"),
        # a padded batch of short prompts, few heads
        _case("append", 3, 5, 777, 32, page=16, ragged=True, slot_major=True, track=True, name="append_b3h5n777d32"),
        # a prompt that streams through a bounded cache in chunks
        _case("evict", 8, 16, 4096, 64, t=512, track=True, bf16=True, name="evict_b8h16n4096t512d64"),
        # the same for a small cache, token by token
        _case("evict", 2, 4, 128, 64, t=1, page=16, track=True, name="evict_b2h4n128t1d64"),
        # a generation step of one user
        _case("step", 1, 16, 512, 64, bf16=True, name="step_b1h16n512d64"),
        # a generation step of a batch that keeps score
        _case("step", 32, 16, 2048, 64, track=True, bf16=True, name="step_b32h16n2048d64_track"),
    ]


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "append", "evict", "step"])
    while True:
        d = rng.choice([32, 64, 64, 128])
        b = round(math.exp(rng.uniform(0.0, math.log(64.4))))
        h = rng.choice([1, 2, 4, 5, 8, 12, 16, 16, 32])
        n = round(math.exp(rng.uniform(math.log(16), math.log(20000))))
        t = 1 if kind == "step" else min(n, round(math.exp(rng.uniform(0.0, math.log(600)))))
        if b * h * (n + (t if kind in ("evict", "step") else 0)) * d <= MOST_TOKENS[kind] and b * h * n * d >= 1 << 14:
            break
    page = rng.choice([8, 16, 16, 32, 64, 64, 128, 256, rng.randint(9, 100)])
    track = rng.random() < 0.4 or kind == "evict"
    return _case(kind, b, h, n, d, t=t, page=page, ragged=kind in ("attend", "append") and rng.random() < 0.5, slot_major=rng.random() < 0.4,
                 bf16=rng.random() < 0.5, track=track, gain=rng.random() < 0.6, rms=rng.random() < 0.8, lam=rng.choice([0.3, 0.5, 0.7, -0.4]))


def _lengths(c):
    """Tokens per sequence: all `n`, or with `ragged` from n / 8 to n, some sequences of the batch being empty."""
    if not c["ragged"]:
        return [c["n"]] * c["b"]
    return [0 if i % 8 == 5 else max(1, c["n"] * (8 - 3 * i % 8) // 8) for i in range(c["b"])]


def prepare(case, seed):
    c = case
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    dt = torch.bfloat16 if c["bf16"] else torch.float16
    b, h, n, d, t, page = c["b"], c["h"], c["n"], c["d"], c["t"], c["page"]
    max_pages = -(-(n + (t if c["kind"] in ("evict", "step") else 0)) // page)
    num = b * max_pages + 3                                  # the pool has pages that no sequence owns

    def normal(*shape):
        return torch.randn(shape, generator=g, device=dev, dtype=dt)

    def pool(w):
        return normal(num, page, h, w).transpose(1, 2) if c["slot_major"] else normal(num, h, page, w)

    s = dict(case=c, k1_pages=pool(d), k2_pages=pool(d), v_pages=pool(2 * d))
    s["page_table"] = torch.randperm(num, generator=g, device=dev)[:b * max_pages].to(torch.int32).view(b, max_pages)
    s["lam"] = torch.tensor([c["lam"]], device=dev)
    s["gain"] = 1.0 + 0.1 * torch.randn(2 * d, generator=g, device=dev) if c["gain"] else None
    lens = torch.tensor(_lengths(c), dtype=torch.int32, device=dev)
    cap = max_pages * page
    s["lengths"] = torch.zeros_like(lens) if c["kind"] == "append" else lens
    s["next_position"] = s["lengths"].clone()
    s["positions"] = torch.arange(cap, dtype=torch.int32, device=dev).expand(b, h, cap).contiguous()
    # accumulated weights of a softmax's shape: many small ones, a few large ones
    s["weights"] = torch.randn((b, h, cap), generator=g, device=dev).mul_(2.0).exp_().mul_(1.0 / n) if c["track"] else None
    s["q1"], s["q2"] = normal(b, h, 1, d), normal(b, h, 1, d)
    m = n if c["kind"] == "append" else t
    # head-interleaved, as a projection followed by a head split leaves them
    s["k1"], s["k2"], s["v"] = (normal(b, m, h, w).transpose(1, 2) for w in (d, d, 2 * d))
    s["counts"] = lens if c["kind"] == "append" and c["ragged"] else None
    if own:
        from triton_diff_attn_b200 import DiffAttnCache
        s["cache"] = DiffAttnCache.from_tensors(s["k1_pages"], s["k2_pages"], s["v_pages"], s["page_table"], s["lengths"], positions=s["positions"],
                                                next_position=s["next_position"], weights=s["weights"])
    return s


def _run_own(s):
    c, cache = s["case"], s["cache"]
    if c["kind"] == "attend":
        y = cache.attend(s["q1"], s["q2"], s["lam"], LAMBDA_INIT, c["rms"], gain=s["gain"])
        return [y, cache.weights]
    if c["kind"] == "append":
        cache.reset()
        cache.append(s["k1"], s["k2"], s["v"], s["counts"])
        return [cache.k1_pages, cache.k2_pages, cache.v_pages, cache.positions, cache.lengths, cache.weights]
    if c["kind"] == "evict":
        cache.append(s["k1"], s["k2"], s["v"])
        cache.evict(c["n"], recent=c["t"])
        return [cache.k1_pages, cache.k2_pages, cache.v_pages, cache.positions, cache.lengths, cache.weights]
    y = cache.attend(s["q1"], s["q2"], s["lam"], LAMBDA_INIT, c["rms"], gain=s["gain"], k1=s["k1"], k2=s["k2"], v=s["v"])
    cache.evict(c["n"], recent=c["n"])
    return [y, cache.positions, cache.lengths, cache.weights]


# ---- the plain form -------------------------------------------------------------------------------------------------------------
def _append(s, k1, k2, v, counts):
    t, page = k1.shape[2], s["case"]["page"]
    steps = torch.arange(t, device=k1.device)
    slot = s["lengths"][:, None] + steps                                                     # [b, t]
    pos = s["next_position"][:, None] + steps
    if counts is None:
        pages = s["page_table"].gather(1, slot // page).long()
        for pool, x in ((s["k1_pages"], k1), (s["k2_pages"], k2), (s["v_pages"], v)):
            pool[pages, :, slot % page] = x.transpose(1, 2)
        s["positions"].scatter_(2, slot[:, None].expand(-1, k1.shape[1], -1).long(), pos[:, None].expand(-1, k1.shape[1], -1).to(torch.int32))
        if s["weights"] is not None:
            s["weights"].scatter_(2, slot[:, None].expand(-1, k1.shape[1], -1).long(), 0.0)
        s["lengths"] += t
        s["next_position"] += t
    else:
        bi, ti = torch.nonzero(steps < counts[:, None], as_tuple=True)
        slot = slot[bi, ti]
        pages = s["page_table"][bi, slot // page].long()
        for pool, x in ((s["k1_pages"], k1), (s["k2_pages"], k2), (s["v_pages"], v)):
            pool[pages, :, slot % page] = x[bi, :, ti]
        s["positions"][bi, :, slot] = pos[bi, ti][:, None].expand(-1, k1.shape[1]).to(torch.int32)
        if s["weights"] is not None:
            s["weights"][bi, :, slot] = 0.0
        s["lengths"] += counts
        s["next_position"] += counts


def _rows(pool, table):
    """All slots of every sequence, [b, h, slots, width], in 32 bits."""
    x = pool[table.long()].transpose(1, 2).float()                                           # [b, h, pages, page, width]
    return x.reshape(x.shape[0], x.shape[1], -1, x.shape[-1])


def _probabilities(q, k, live):
    s = (k @ q.float().transpose(-1, -2)).squeeze(-1) / math.sqrt(q.shape[-1])               # [b, h, slots]
    s = s.masked_fill(~live, -math.inf)
    top = s.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)                 # a sequence without tokens has no maximum
    e = torch.exp(s - top)
    return e / e.sum(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).tiny)


def _attend(s):
    c = s["case"]
    table, slots = s["page_table"], s["page_table"].shape[1] * c["page"]
    live = (torch.arange(slots, device=table.device) < s["lengths"][:, None])[:, None]       # [b, 1, slots]
    p1 = _probabilities(s["q1"], _rows(s["k1_pages"], table), live)
    p2 = _probabilities(s["q2"], _rows(s["k2_pages"], table), live)
    p = p1 - s["lam"] * p2
    if s["weights"] is not None:
        s["weights"] += p.abs()
    a = p[:, :, None] @ _rows(s["v_pages"], table).masked_fill_(~live[..., None], 0.0)       # [b, h, 1, 2 d]
    if c["rms"]:
        a = a * torch.rsqrt(a.square().mean(-1, keepdim=True) + EPS) * (1.0 - LAMBDA_INIT)
    if s["gain"] is not None:
        a = a * s["gain"]
    return a.to(s["q1"].dtype)


def _evict(s, keep, recent):
    page, slots = s["case"]["page"], s["positions"].shape[-1]
    at = torch.arange(slots, device=s["positions"].device)
    live = (at < s["lengths"][:, None])[:, None]
    newest = s["positions"] >= (s["next_position"] - recent)[:, None, None]
    key = (s["weights"] if s["weights"] is not None else s["positions"].float()).masked_fill(newest, math.inf).masked_fill(~live, -math.inf)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    kept = torch.zeros_like(live.expand_as(key)).scatter(2, order[..., :keep], True) & live
    bi, hi, src = torch.nonzero(kept & (at >= keep), as_tuple=True)
    _, _, dst = torch.nonzero(~kept & live & (at < keep) & (s["lengths"] > keep)[:, None, None], as_tuple=True)
    table = s["page_table"].long()
    for pool in (s["k1_pages"], s["k2_pages"], s["v_pages"]):
        pool[table[bi, dst // page], hi, dst % page] = pool[table[bi, src // page], hi, src % page]
    for x in (s["positions"], s["weights"]):
        if x is not None:
            x[bi, hi, dst] = x[bi, hi, src]
    s["lengths"].clamp_(max=keep)


def run(state):
    if own:
        return _run_own(state)
    s, c = state, state["case"]
    if c["kind"] == "attend":
        return [_attend(s), s["weights"]]
    if c["kind"] == "append":
        s["lengths"].zero_()
        s["next_position"].zero_()
        _append(s, s["k1"], s["k2"], s["v"], s["counts"])
        return [s["k1_pages"], s["k2_pages"], s["v_pages"], s["positions"], s["lengths"], s["weights"]]
    if c["kind"] == "evict":
        _append(s, s["k1"], s["k2"], s["v"], None)
        _evict(s, c["n"], c["t"])
        return [s["k1_pages"], s["k2_pages"], s["v_pages"], s["positions"], s["lengths"], s["weights"]]
    _append(s, s["k1"], s["k2"], s["v"], None)
    y = _attend(s)
    _evict(s, c["n"], c["n"])
    return [y, s["positions"], s["lengths"], s["weights"]]


def work(case):
    c = case
    tokens, width = sum(_lengths(c)) * c["h"], c["d"]
    row = 8 * width                                           # K1, K2 and V of one token and head, in bytes
    if c["kind"] == "append":
        return {"bytes": tokens * (2 * row + 4 + (4 if c["track"] else 0)), "flops": 0}
    new = c["b"] * c["h"] * c["t"]
    if c["kind"] == "evict":
        # the chunk is read and written, the weight and the position of every token read, and the chunk's rows move once more
        return {"bytes": new * (2 * row + 8) + (tokens + new) * 8 + new * 2 * (row + 8), "flops": 0}
    ends = c["b"] * c["h"] * 8 * width                        # the queries and y
    bytes_ = tokens * row + ends + (tokens * 8 if c["track"] else 0)
    if c["kind"] == "step":
        bytes_ += new * (2 * row + 8) + tokens * 4 + new * 2 * row
    return {"bytes": bytes_, "flops": tokens * 12 * width}


def exact(case, seed):
    """y and the accumulated weights from the definition, sequence by sequence in 64 bits.  Moved and stored rows have no computed value."""
    c = case
    if c["kind"] in ("append", "evict"):
        return None
    s = prepare(case, seed)
    d, page = c["d"], c["page"]
    y, weights = [], s["weights"].double() if c["track"] else None
    for i, length in enumerate(_lengths(c)):
        ids = s["page_table"][i, :-(-length // page)].long()

        def tokens(pool, new):
            x = torch.movedim(pool[ids], 1, 0).double().flatten(1, 2)[:, :length]            # [h, tokens, width]
            return torch.cat([x, new[i].double()], 1) if c["kind"] == "step" else x

        k1, k2, v = tokens(s["k1_pages"], s["k1"]), tokens(s["k2_pages"], s["k2"]), tokens(s["v_pages"], s["v"])
        if v.shape[1] == 0:
            y.append(torch.zeros(c["h"], 1, 2 * d, dtype=torch.float64, device=v.device))
            continue
        p1, p2 = (torch.softmax(torch.einsum("hd,htd->ht", q[i, :, 0].double(), k) * d ** -0.5, -1) for q, k in ((s["q1"], k1), (s["q2"], k2)))
        w = p1 - float(s["lam"]) * p2
        a = torch.einsum("ht,htw->hw", w, v)
        if c["rms"]:
            a = (1.0 - LAMBDA_INIT) * a / torch.sqrt((a * a).sum(-1, keepdim=True) / (2 * d) + EPS)
        if c["gain"]:
            a = a * s["gain"].double()
        y.append(a[:, None])
        if weights is not None and c["kind"] == "attend":
            weights[i, :, :length] += w.abs()
        elif weights is not None:
            # the window's oldest token (slot 0) goes, the new one (the last) takes its place; what lies behind it stays
            weights[i, :, 1:length] += w[:, 1:length].abs()
            weights[i, :, 0] = w[:, length].abs()
            weights[i, :, length] = w[:, length].abs()
    y = torch.stack(y)
    return [y, weights] if c["kind"] == "attend" else [y, None, None, weights]
