"""Attention of chunks where a row's scores, times the scale and log2 e, lie on both sides of 2^20: from there on its
weights are relative to the maximum itself, below to a power of two, and parts of either kind are put together.

The scores are sums of a few products, multiples of 2^-7 below 2^16, that f32 holds whatever the order. What is
left, relative to sum_i p_i |v_i|: the exponent, c (s - m) of up to 2^6 by a c of 2^-24 and two roundings, to
3 2^-18 in all; exp2, sums and quotient as in test_gpu_kv4_chunk, with the 16-bit types' 2^-16 of p; and half a step
of the output."""
import math

import pytest
import torch

from borch_amd import kv4
from oracle import decode as D
from test_gpu_kv4 import HALF, LEAST, TYPES, starts, tables

pytestmark = pytest.mark.gpu

SCALE, FAR = 16.0, 2.0 ** 20
CODES = torch.tensor([0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n,rows,heads,group", [(200, 40, 1, 1), (200, 40, 1, 54), (9000, 2, 1, 8), (9000, 70, 1, 32)])
def test_chunk_maxima_on_both_sides(dev, sign, kind, dim, n, rows, heads, group):
    """In narrow tiles, wide ones, and shares of either: far maxima before and after near ones."""
    print(f"kv4 chunk far {sign} {kind} dim={dim} {n} tokens {rows} rows x {group}", flush=True)
    g = torch.Generator().manual_seed(61)
    k = torch.zeros(n, 1, dim)
    k[:, 0, 0] = k[:, 0, 1] = 2.0 if sign > 0 else 6.0  # far below the others
    k[:, 0, 9], k[:, 0, 40] = 6.0, 6.0                  # every block's scale 1
    if dim == 128:
        k[:, 0, 70] = k[:, 0, 100] = 6.0
    odd = torch.arange(3, n - rows, 23 if n < 1000 else 401)  # in all blocks of 32 and all shares
    k[odd, 0, :2] = 4.0
    k[odd, 0, 2:6] = CODES[torch.randint(0, 7, (len(odd), 4), generator=g)] * (torch.randint(0, 2, (len(odd), 4), generator=g) * 2 - 1)
    q = torch.zeros(rows, group, dim)
    q[..., 0], q[..., 1] = sign * 11264.0, sign * 92.5  # 4 (11264 + 92.5) = 45426, 2^20 / c = 45426.1
    q[..., 2:6] = torch.randint(1, 9, (rows, group, 4), generator=g) * 2.0 ** -6
    q = q.to(TYPES[kind])
    v = torch.randn(n, 1, dim, generator=g)
    table, pages = tables([n], 64, 62)
    c = kv4.Cache4.zeros(pages, 1, 64, dim, dev)
    ln = torch.tensor([n], dtype=torch.int32)
    c.append(k.to(dev), v.to(dev), table.to(dev), ln.to(dev), starts([n]).to(dev))
    held_k, held_v = (x[0, 0].cpu().double() for x in c.read(table.to(dev), ln.to(dev), n))
    assert torch.equal(held_k, k[:, 0].double())
    got = c.attend_chunk(q.to(dev), table.to(dev), ln.to(dev), starts([rows]).to(dev), scale=SCALE).cpu().double()
    qs = q.reshape(-1, dim).double()
    s = qs @ held_k.T
    assert torch.equal(s, s.float().double())
    tops = (s[:, odd] * SCALE / math.log(2)).abs()
    both = (tops > FAR + 1).any(1) & (tops < FAR - 1).any(1)
    assert float(both.double().mean()) > 0.9 and float((tops - FAR).abs().max()) < 2 ** 6
    seen = torch.arange(n) < (torch.arange(n - rows, n) + 1).repeat_interleave(group)[:, None]
    want, _, size = D.softmax_rows(qs, held_k, held_v, seen, SCALE)
    rel = 3 * 2.0 ** -18 + (3 * n + 64) * 2.0 ** -24 + (0.0 if kind == "f32" else 2.0 ** -16)
    off = (got.reshape(-1, dim) - want).abs()
    tol = size * rel + want.abs() * (HALF[kind] + 2.0 ** -24) + LEAST[kind]
    assert bool((off <= tol).all()), float((off / tol).max())
