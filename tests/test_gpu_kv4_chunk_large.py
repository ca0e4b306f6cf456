"""Attention of chunks over values near the end of f32's range: finite where the values are, as long as f32 holds
their sum. Tolerance as in test_gpu_kv4_chunk, with 2^-16 for the weights."""
import pytest
import torch

import test_gpu_kv4_chunk as C
from borch_amd import kv4
from test_gpu_kv4 import starts, tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n,rows,group", [(130, 12, 1), (300, 3, 5), (300, 140, 16), (9000, 2, 8), (9000, 70, 32)])
@pytest.mark.parametrize("where", ["spread", "last"])
def test_chunk_large_values(dev, monkeypatch, kind, dim, n, rows, group, where):
    """Scores that rise by less than the maximum may lag behind, and large values among the later tokens: in narrow
    tiles, wide ones, and shares of either."""
    print(f"kv4 chunk large values {kind} dim={dim} {n} tokens {rows} rows x {group} {where}", flush=True)
    monkeypatch.setitem(C.WEIGHT, "bf16", 2.0 ** -16)
    g = torch.Generator().manual_seed(71)
    k = torch.randn(n, 1, dim, generator=g) * 0.1
    rise = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])[(torch.arange(n) * 8) // n]
    k[:, 0, 0], k[:, 0, 1] = rise, 6.0
    q = torch.randn(rows, group, dim, generator=g) * 0.1
    q[..., 0] = torch.rand(rows, group, generator=g) * 0.9 * dim ** 0.5  # up to 5.4 for the last: 7.8 powers of two
    q[..., 1] = 0.0
    v = torch.randn(n, 1, dim, generator=g)
    at = torch.arange(n // 9, n - rows, n // 9) if where == "spread" else torch.arange(n - rows - 6, n - rows)
    v[at, 0, 5] = 1.2e37 * torch.rand(len(at), generator=g)
    v[at[:5], 0, 40] = -2.0e37
    v[at[-1], 0, 41] = 2.5e38  # held as 6 2^125
    q = q.to(C.TYPES[kind])
    table, pages = tables([n], 64, 72)
    c = kv4.Cache4.zeros(pages, 1, 64, dim, dev)
    ln, cu = torch.tensor([n], dtype=torch.int32), starts([rows])
    c.append(k.to(dev), v.to(dev), table.to(dev), ln.to(dev), starts([n]).to(dev))
    hk, hv, there = C.held(c, table, ln, n, dev)
    assert bool(torch.isfinite(hv).all()) and float(hv.max()) == 6 * 2.0 ** 125
    got = c.attend_chunk(q.to(dev), table.to(dev), ln.to(dev), cu.to(dev))
    assert bool(torch.isfinite(got).all())
    for _ in range(3):
        assert torch.equal(got, c.attend_chunk(q.to(dev), table.to(dev), ln.to(dev), cu.to(dev)))
    C.check(got, q, hk, hv, there, ln, cu, n, kind)
