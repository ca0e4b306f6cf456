"""The decoder's attention as sums of 16-bit pieces, on the CPU: which pieces and which products there are,
with any of them left out on request, and inputs on which each of them decides the result. Written apart
from the kernels; used by the tests alone.

A row sees two heavy keys, all others 100 and more below (a weight of 0), so that its sums have two terms and
an output is p1 v1 / (p0 + p1) with v0 = 0."""
from __future__ import annotations

import torch

LOG2E = 1.4426950408889634


def bf16_pieces(x: torch.Tensor, count: int):
    """f32 values as `count` bf16 ones (float64), the largest first."""
    got, rest = [], x.float()
    for _ in range(count):
        p = rest.bfloat16().float()
        got.append(p.double())
        rest = rest - p
    return got


def fp16_pieces(x: torch.Tensor):
    """Rows of f32 values as two fp16 pieces below a power of two of each row's largest (float64)."""
    x = x.double()
    e = torch.frexp(x.abs().amax(-1, keepdim=True))[1] - 14  # the largest lies in [2^13, 2^14)
    y = torch.ldexp(x, -e)
    hi = y.half().double()
    lo = (y - hi).float().half().double()
    return [torch.ldexp(hi, e), torch.ldexp(lo, e)]


def _product(a, b, which, drop, name):
    """sum over `which` (i, j) of a[i] b[j], but those of `drop`."""
    return sum(a[i] * b[j] for i, j in which if f"{name}{i}{j}" not in drop)


PROMPT_SCORES = ((0, 0), (0, 1), (1, 0))  # pieces of k, of q
PROMPT_VALUES = ((0, 0), (0, 1), (1, 0), (0, 2), (1, 1), (2, 0))  # of v, of p


def prompt_f32(q, k, v1, scale, drop=()):
    """p1 v1 / (p0 + p1) for rows q [r, c] over keys k [2, c]: [r, len(v1)]."""
    qs, ks = fp16_pieces(q), fp16_pieces(k)
    s = sum(_product([p[j] for p in ks], qs, PROMPT_SCORES, drop, "s").sum(-1)[:, None] * (torch.arange(2) == j) for j in range(2))
    return _softmax_pieces(s, bf16_pieces(v1, 3), PROMPT_VALUES, 3, scale, drop)


Q_PIECES, P_PIECES = {"f32": 3, "bf16": 1, "f16": 2}, {"f32": 3, "bf16": 2, "f16": 2}


def attend(kind, q, k, v1, scale, drop=()):
    """The same over cached keys and values, which bf16 holds exactly; q and p in pieces."""
    qs = bf16_pieces(q, Q_PIECES[kind])
    s = sum(sum(p * k[j].double() for i, p in enumerate(qs) if f"q{i}" not in drop).sum(-1)[:, None] * (torch.arange(2) == j)
            for j in range(2))
    n = P_PIECES[kind]
    return _softmax_pieces(s, [v1.double()], tuple((0, i) for i in range(n)), n, scale, drop)


def _softmax_pieces(s, vs, which, pieces, scale, drop):
    p = torch.exp2((s - s.amax(-1, keepdim=True)) * scale * LOG2E).float()
    ps = bf16_pieces(p, pieces)
    top = _product([x[None] for x in vs], [x[:, 1:] for x in ps], which, drop, "p")
    return top / p.double().sum(-1, keepdim=True)


def exact(q, k, v1, scale):
    s = (q.double()[:, None] * k.double()).sum(-1) * scale
    return torch.softmax(s, -1)[:, 1:] * v1.double()


# ------------------------------------------------------------------ inputs and bounds

def rough(shape, least, most, seed, kind=torch.float32):
    """Values of [least, most) whose every bit is random."""
    g = torch.Generator().manual_seed(seed)
    return (least + (most - least) * torch.rand(shape, generator=g, dtype=torch.float64)).to(kind)


def close_scores(rows, seed, kind=torch.float32):
    """q [rows, 2] and keys [2, 2]: scores near 75 (scale 1/8) that differ by up to 2, each the product of one
    channel with bits to the last."""
    k = torch.diag(rough((2,), 16.0, 31.0, seed + 1, kind).float())
    q = torch.empty(rows, 2)
    q[:, 0] = 600.0 / k[0, 0] + rough((rows,), -0.1, 0.1, seed + 2).float()
    q[:, 1] = 600.0 / k[1, 1] + rough((rows,), -0.1, 0.1, seed + 3).float()
    return q.to(kind), k


def score_bound(q, k, v1, scale, each):
    """Scores off by `each` of |q| |k|: p1 moves by p0 p1 of the two scores' errors, twice that for what is not
    linear in it."""
    s = (q.double()[:, None] * k.double()).sum(-1) * scale
    p = torch.softmax(s, -1)
    off = (q.double().abs()[:, None] * k.double().abs()).sum(-1).sum(-1) * scale * each
    return (p[:, :1] * p[:, 1:] * 2 * off[:, None]) * v1.double().abs()


# p1 v1 / (p0 + p1) from exact scores that differ by up to 2: the exponent's argument 2 2^-24 of 2.9, the
# exponential 2 2^-24, both in the quotient and in the sum (12); six products added (6), those of weight below
# 2^-24 (3), a sum of two (2), a quotient (2)
WEIGHT_BOUND = 25 * 2.0 ** -24


def close_cached_scores(rows, seed, kind):
    """q [rows, 2] over cached keys [2, 2] of 4 in one channel each: scores near 75 (scale 1/8) that differ by up
    to 2, q's bits to the last."""
    q = torch.stack([rough((rows,), 149.0, 151.0, seed + i, kind) for i in range(2)], 1)
    return q, torch.diag(torch.tensor([4.0, 4.0]))


def near_scores(rows, seed, kind):
    """q [rows, 1] whose score over a key of 4 (scale 1/8) is a multiple of 1/64 in (-2, 2): exact in every type."""
    return (torch.round(rough((rows, 1), -3.9, 3.9, seed).double() * 32) / 32).to(kind)


# as WEIGHT_BOUND, and 8 2^-24 for the waves' and the parts' join; p in two pieces: 2^-16
PART_BOUND = {"f32": 33 * 2.0 ** -24, "bf16": 33 * 2.0 ** -24 + 2.0 ** -16, "f16": 33 * 2.0 ** -24 + 2.0 ** -16}
