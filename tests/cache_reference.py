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

    Error of the kernels.  Scores and outputs are sums in fp32 on the tensor cores, which may cut off instead of rounding: up to 2 u (u the unit
    roundoff) per addition, where fp32 itself would have u.  A score is a sum of D exact products, scaled once: it is off by at most
    (D + 12) 2 u S / ln 2 in base 2 with S = max_j sum |q_i k_ji| / sqrt(D), a probability by a factor exp(+-2 u (D + 12) S); the exponential
    itself and its argument's subtraction stay inside the 12.  Sums over n tokens: chains of at most n / 4 + 64 additions.  A probability
    reaches the output as two 16-bit numbers: the second one's rounding leaves (eps / 2)^2 of it, and in fp16, whose second number can be
    subnormal, at least 2^-25 beside a largest probability of 1 or more (so beside a row sum L of 1 or more, L = sum exp(s_j - max s)).  Numerator and
    denominator: twice.  The result's rounding to 16 bits: eps / 2."""
    n, d = k1.shape
    if n == 0:
        z = torch.zeros(v.shape[1], dtype=torch.float64, device=v.device)
        return z, z[:0], z, z[:0]
    s1, s2 = (k1 @ q1) / math.sqrt(d), (k2 @ q2) / math.sqrt(d)
    p1, p2 = torch.softmax(s1, 0), torch.softmax(s2, 0)
    big = max(float((k1.abs() @ q1.abs()).max()), float((k2.abs() @ q2.abs()).max())) / math.sqrt(d)
    info = torch.finfo(io)
    rel = 4.0 * U32 * ((d + 12) * big + 64 + n / 4)
    a = p1 @ v - lam * (p2 @ v)
    da = (rel + 2 * (info.eps / 2) ** 2) * ((p1 + abs(lam) * p2) @ v.abs())
    if io == torch.float16:
        da = da + 2.0 ** -25 * (float(p1.max()) + abs(lam) * float(p2.max())) * v.abs().sum(0)      # (1 / L is the largest probability)
    if rms:
        r = 1.0 / math.sqrt(float((a * a).mean()) + eps)
        da = (1.0 - lambda_init) * r * (da + a.abs() * r * float((da * da).mean()) ** 0.5 + 8 * U32 * a.abs())
        a = a * r * (1.0 - lambda_init)
    if gain is not None:
        a, da = a * gain.double(), da * gain.double().abs() + 2 * U32 * (a * gain.double()).abs()
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
