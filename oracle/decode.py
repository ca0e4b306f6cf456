"""A decoder's attention in float64 on the CPU: packed prompts, the 4-bit key-value cache (its
codes, pages and layouts, written token by token from their description in include/bq.h), attention
over it and eviction. Written apart from the kernels; used by the tests alone."""
from __future__ import annotations

import math

import torch

VALUES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def quantize(x: torch.Tensor):
    """x [..., dim] -> codes [..., dim] and scale bytes [..., dim / 32] (ints)."""
    g = x.double().reshape(*x.shape[:-1], -1, 32)
    bad = ~torch.isfinite(g).all(-1)
    g = torch.where(bad[..., None], torch.zeros_like(g), g)
    peak = g.abs().amax(-1)
    e = torch.full_like(peak, -126.0)
    for k in range(-126, 127):  # the least exponent that fits
        e = torch.where((peak > 6.0 * 2.0 ** (k - 1)) & (peak <= 6.0 * 2.0 ** k), torch.full_like(e, float(k)), e)
    y = g.abs() / (2.0 ** e)[..., None]
    table = torch.tensor(VALUES, dtype=torch.float64)
    dist = (y[..., None] - table).abs()
    near = dist == dist.amin(-1, keepdim=True)
    idx = torch.arange(8)
    # of two equally near codes the even one
    code = torch.where(near, torch.where(idx % 2 == 0, idx, idx + 8), torch.full_like(idx, 99)).amin(-1) % 8
    code = code + 8 * torch.signbit(g).long()
    byte = torch.where(bad, torch.full_like(e, 255.0), e + 127).long()
    return code.reshape(x.shape), byte


def value(code: torch.Tensor, byte: torch.Tensor) -> torch.Tensor:
    table = torch.tensor(VALUES + [-v for v in VALUES], dtype=torch.float64)
    s = torch.where(byte == 255, torch.full(byte.shape, math.nan, dtype=torch.float64), 2.0 ** (byte.double() - 127))
    return (table[code.long()].reshape(*byte.shape, 32) * s[..., None]).reshape(code.shape)


class Pages:
    """The four arrays on the CPU, written and read one token at a time."""

    def __init__(self, k, k_scales, v, v_scales):
        self.k, self.ks, self.v, self.vs = (t.cpu().clone() for t in (k, k_scales, v, v_scales))
        self.pages, self.heads, self.page, half = self.k.shape
        self.dim = 2 * half
        self.tb = 512 // self.dim

    def at(self, table, b, pos):
        i = pos // self.page
        if pos < 0 or i >= table.shape[1]:
            return None
        p = int(table[b, i])
        return (p, pos % self.page) if 0 <= p < self.pages else None

    def put(self, p, h, off, kc, kb, vc, vb):
        n, c = self.dim // 16, self.dim // 32
        for i in range(self.dim // 2):
            self.k[p, h, off, i] = int(kc[2 * i]) | int(kc[2 * i + 1]) << 4
        for i in range(c):
            self.ks[p, h, off // 32, off % 4, i, off % 32 // 4] = int(kb[i])
            self.vs[p, h, off // 32, i, off % 32] = int(vb[i])
        for s in range(16):
            for i in range(c):
                self.v[p, h, off // self.tb, s, off % self.tb, i] = int(vc[s * n + 2 * i]) | int(vc[s * n + 2 * i + 1]) << 4

    def get(self, p, h, off):
        """Codes and bytes of a token's key and value."""
        k = self.k[p, h, off].long()
        kc = torch.stack((k & 15, k >> 4), -1).flatten()
        v = self.v[p, h, off // self.tb, :, off % self.tb].flatten().long()
        vc = torch.stack((v & 15, v >> 4), -1).flatten()
        return (kc, self.ks[p, h, off // 32, off % 4, :, off % 32 // 4].long(), vc,
                self.vs[p, h, off // 32, :, off % 32].long())

    def append(self, new_k, new_v, table, lens, cu):
        for b in range(table.shape[0]):
            for i in range(int(cu[b]), int(cu[b + 1])):
                at = self.at(table, b, int(lens[b]) - int(cu[b + 1]) + i)
                if at is None:
                    continue
                (kc, kb), (vc, vb) = quantize(new_k[i]), quantize(new_v[i])
                for h in range(self.heads):
                    self.put(at[0], h, at[1], kc[h], kb[h], vc[h], vb[h])

    def read(self, table, lens, most):
        """Keys and values [B, heads, most, dim] in float64, zeros past the lengths and off the pages,
        and which places hold a token [B, most]."""
        B = table.shape[0]
        k = torch.zeros(B, self.heads, most, self.dim, dtype=torch.float64)
        v, there = torch.zeros_like(k), torch.zeros(B, most, dtype=torch.bool)
        for b in range(B):
            for t in range(min(int(lens[b]), most)):
                at = self.at(table, b, t)
                if at is None:
                    continue
                there[b, t] = True
                got = [self.get(at[0], h, at[1]) for h in range(self.heads)]
                k[b, :, t] = value(torch.stack([g[0] for g in got]), torch.stack([g[1] for g in got]))
                v[b, :, t] = value(torch.stack([g[2] for g in got]), torch.stack([g[3] for g in got]))
        return k, v, there


def softmax_rows(q, k, v, seen, scale):
    """softmax(scale q k^T) v of q [r, d] over k, v [n, d], row i over seen[i] [n], in float64; zeros
    for a row that sees nothing, or only scores of -infinity. Returns the output, the weights and sum_i
    p_i |v_i|."""
    q, k, v = q.double(), k.double(), v.double()
    out = torch.zeros(q.shape[0], v.shape[1], dtype=torch.float64)
    size = torch.zeros_like(out)
    p = torch.zeros(q.shape[0], k.shape[0], dtype=torch.float64)
    for i in range(q.shape[0]):
        at = seen[i].nonzero()[:, 0]
        if not len(at):
            continue
        s = (k[at] * q[i]).sum(-1) * scale
        top = s.max()
        w = torch.exp(s - (top if torch.isfinite(top) else 0.0))
        w = w / (w.sum() if w.sum() != 0 else 1.0)
        p[i, at] = w
        out[i] = (w[:, None] * v[at]).sum(0)
        size[i] = (w[:, None] * v[at].abs()).sum(0)
    return out, p, size


def score_error(q, k, scale, pieces):
    """A bound on the error that f32 accumulation leaves in a score, times 2 (numerator and sum):
    a sum of `pieces` dim exact products, each addition within 2^-24 of its partial sum, and the
    exponent's argument within 2^-22 of itself (a difference, a product, a reduced constant)."""
    if not q.numel() or not k.numel():
        return 0.0
    size = float((q.double().abs() @ k.double().abs().t().contiguous()).nan_to_num(0, 0, 0).max()) * scale
    return 2.0 * (size * (pieces * q.shape[1] + 4) * 2.0 ** -24 + 2 * size * 2.0 ** -22)


def evict(sums, n, keep, recent):
    """Which of n tokens stay, in order: the `recent` last ones and the keep - recent of the others of
    largest weight, ties to the earlier (sums [n] as python floats)."""
    if n <= keep:
        return list(range(n))
    old = n - recent
    rank = sorted(range(old), key=lambda i: (-math.inf if math.isnan(sums[i]) else -sums[i], not math.isnan(sums[i]), i))
    return sorted(rank[:keep - recent]) + list(range(old, n))
