"""The key-value cache's operators from their definitions, in 64 bits on whatever device the tensors are on, and the error that the kernels'
arithmetic may have.  Shared by the cache tests."""
import math

import torch

U32 = 2.0 ** -24


def rows(pool, table_row, page_size, head, n):
    """The first n cached rows of one sequence and head, 64 bits."""
    at = torch.arange(n, device=pool.device)
    return pool[table_row.long()[at // page_size], head, at % page_size].double()


def attend(q1, q2, k1, k2, v, lam, lambda_init=0.8, rms=False, gain=None, io=torch.float16, eps=1e-5):
    """One head: q [D], k [n, D], v [n, 2D] in 64 bits.  Returns y, |P1 - lam P2|, and how far y and the weights may be off.

    Error of the kernels, in fp32 (unit roundoff u): a score is a sum of D products (relative error of each at most (D + 8) u with the scaling
    of q and the sum over lanes), so a probability is off by a factor exp(+-(D + 8) u S) with S = max_j sum |q_i k_ji| / sqrt(D), the
    exponential itself by a few u and by u times its argument (subtraction of the maximum, at most 2 S), sums over n terms in chains of at
    most n / 4 + 64 additions by that many u.  Numerator and denominator: twice.  The result's rounding to 16 bits: eps / 2."""
    n, d = k1.shape
    if n == 0:
        z = torch.zeros(v.shape[1], dtype=torch.float64, device=v.device)
        return z, z[:0], z, z[:0]
    s1, s2 = (k1 @ q1) / math.sqrt(d), (k2 @ q2) / math.sqrt(d)
    p1, p2 = torch.softmax(s1, 0), torch.softmax(s2, 0)
    big = max(float((k1.abs() @ q1.abs()).max()), float((k2.abs() @ q2.abs()).max())) / math.sqrt(d)
    rel = 2.0 * U32 * ((d + 12) * big + 64 + n / 4)
    a = p1 @ v - lam * (p2 @ v)
    da = rel * ((p1 + abs(lam) * p2) @ v.abs())
    if rms:
        r = 1.0 / math.sqrt(float((a * a).mean()) + eps)
        da = (1.0 - lambda_init) * r * (da + a.abs() * r * float((da * da).mean()) ** 0.5 + 8 * U32 * a.abs())
        a = a * r * (1.0 - lambda_init)
    if gain is not None:
        a, da = a * gain.double(), da * gain.double().abs() + 2 * U32 * (a * gain.double()).abs()
    info = torch.finfo(io)
    dy = da + (a.abs() + da) * info.eps / 2 + info.tiny * info.eps
    w = (p1 - lam * p2).abs()
    return a, w, dy, rel * (p1 + abs(lam) * p2)


def evict(weights, positions, length, next_position, keep, recent):
    """One head: which slot each slot's token comes from afterwards (list of (to, from)), by the definition."""
    if length <= keep:
        return []

    def order(j):
        pos = int(positions[j])
        if pos >= next_position - recent:
            first = (2, 0.0)
        elif weights is None:
            first = (0, float(pos))
        else:
            w = float(weights[j])
            first = (1, 0.0) if w != w else (0, w + 0.0)
        return (-first[0], -first[1], j)

    kept = sorted(sorted(range(length), key=order)[:keep])
    holes = sorted(set(range(keep)) - set(kept))
    movers = [j for j in kept if j >= keep]
    assert len(holes) == len(movers)
    return list(zip(holes, movers))
