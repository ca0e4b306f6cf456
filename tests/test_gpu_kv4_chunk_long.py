"""Attention of chunks where a share of the keys is long, so that its pages are looked up several times, and where
there are thousands of sequences, whose tiles are found in two steps. Tolerance as in test_gpu_kv4_chunk, with 2^-16
for the weights of the 16-bit types; the float64 products are taken on the GPU."""
import pytest
import torch

from borch_amd import _lib, kv4
from oracle import decode as D
from test_gpu_kv4 import HALF, LEAST, PIECES, TYPES, starts, tables

pytestmark = pytest.mark.gpu


def close(got, q, k, v, end, kind):
    """Rows q [r, dim] over k, v [n, dim] of which they see the first `end` [r]; or k, v [r, n, dim]."""
    q, n, dim = q.double(), k.shape[-2], k.shape[-1]
    s = ((k * q[:, None]).sum(-1) if k.dim() == 3 else q @ k.t().contiguous()) * dim ** -0.5
    p = torch.softmax(s.masked_fill(torch.arange(n, device=s.device) >= end[:, None], -torch.inf), -1)
    p = torch.where(end[:, None] > 0, p, torch.zeros_like(p))
    del s
    times = (lambda x: (p[..., None] * x).sum(1)) if k.dim() == 3 else (lambda x: p @ x)
    want, size = times(v), times(v.abs())
    err = D.score_error(q, k.reshape(-1, dim), dim ** -0.5, PIECES[kind])
    rel = err + (3 * n + 64) * 2.0 ** -24 + (0.0 if kind == "f32" else 2.0 ** -16)
    tol = size * rel + want.abs() * (HALF[kind] + 2.0 ** -24) + LEAST[kind] + n * 2.0 ** -126 * float(v.abs().max())
    off = (got.double() - want).abs()
    assert bool((off <= tol).all()), float((off / tol).max())


def cache_of(dev, lens, h, dim, page, g):
    table, pages = tables(lens, page, 81)
    c = kv4.Cache4.zeros(pages, h, page, dim, dev)
    x = torch.randn(sum(lens), 2 * h, dim, generator=g, device=dev)
    table, ln = table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev)
    c.append(x[:, :h], x[:, h:], table, ln, starts(lens).to(dev))
    return c, table, ln


def shares(c, kind, n, B, hq, most):
    """How many shares a tile may have: 0 where none is cut."""
    size = _lib.lib().bq_kv4_attend_chunk_ws_bytes(list(TYPES).index(kind), n, B, hq, c.heads, c.dim, most, c.pages * c.page)
    return size // (n * hq * (c.dim + 2) * 4)


@pytest.mark.parametrize("kind,dim,new,h,group", [("f32", 64, 1600, 8, 4), ("bf16", 64, 2048, 16, 3), ("f16", 64, 2048, 16, 3),
                                                  ("f32", 128, 1600, 8, 4), ("bf16", 128, 1600, 8, 4), ("f16", 128, 1600, 8, 4)])
def test_chunk_long_wide_shares(dev, kind, dim, new, h, group):
    """Wide tiles of 129 units of 64 keys in one share."""
    print(f"kv4 chunk long wide shares {kind} dim={dim}", flush=True)
    n = 8200
    g = torch.Generator(device=dev).manual_seed(82)
    c, table, ln = cache_of(dev, [n], h, dim, 32, g)
    assert shares(c, kind, new, 1, h * group, n) == 0
    q = (3 * torch.randn(new, h * group, dim, generator=g, device=dev)).to(TYPES[kind])
    got = c.attend_chunk(q, table, ln, starts([new]).to(dev), max_len=n)
    k, v = (x[0].double() for x in c.read(table, ln, n))
    end = torch.arange(n - new, n, device=dev) + 1
    for j in range(h * group):
        close(got[:, j], q[:, j], k[j // group], v[j // group], end, kind)


@pytest.mark.parametrize("kind,dim,B", [("f32", 64, 64), ("bf16", 64, 96), ("f16", 64, 96), ("f32", 128, 64), ("bf16", 128, 64),
                                        ("f16", 128, 64)])
def test_chunk_long_narrow_shares(dev, kind, dim, B):
    """Narrow tiles of 132 units and fewer, of which a wave takes every fourth half, in one share."""
    print(f"kv4 chunk long narrow shares {kind} dim={dim}", flush=True)
    h, lens = 8, [8420 - 3 * b for b in range(B)]
    g = torch.Generator(device=dev).manual_seed(83)
    c, table, ln = cache_of(dev, lens, h, dim, 32, g)
    new = [1 + b % 2 for b in range(B)]
    n = sum(new)
    assert shares(c, kind, n, B, h, max(lens)) == 0
    q = (3 * torch.randn(n, h, dim, generator=g, device=dev)).to(TYPES[kind])
    got = c.attend_chunk(q, table, ln, starts(new).to(dev), max_len=max(lens))
    k, v = (x.double() for x in c.read(table, ln, max(lens)))
    at = 0
    for b in range(B):
        end = torch.arange(lens[b] - new[b], lens[b], device=dev) + 1
        for j in range(h):
            close(got[at:at + new[b], j], q[at:at + new[b], j], k[b, j], v[b, j], end, kind)
        at += new[b]


@pytest.mark.parametrize("count", [4030, 4031, 4095, 4200, 8192])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_chunk_thousands_of_sequences(dev, kind, count):
    """Short sequences, many without new tokens, among them a few that take wide tiles."""
    print(f"kv4 chunk {count} sequences {kind}", flush=True)
    dim, group = 64, 2
    lens = [(i * 37) % 6 for i in range(count)]
    new = [min(m, (i * 5) % 3) for i, m in enumerate(lens)]
    for i in (0, 70, count // 2, count - 65, count - 1):
        lens[i], new[i] = 120, 100
    g = torch.Generator(device=dev).manual_seed(84)
    c, table, ln = cache_of(dev, lens, 1, dim, 32, g)
    cu = starts(new) + 2  # rows of no sequence before the first, and past the last
    n = sum(new) + 5
    q = (2 * torch.randn(n, group, dim, generator=g, device=dev)).to(TYPES[kind])
    got = c.attend_chunk(q, table, ln, cu.to(dev), max_len=120)
    assert not bool(got[:2].any()) and not bool(got[-3:].any())
    seq = torch.repeat_interleave(torch.arange(count), torch.tensor(new)).to(dev)
    end = (ln[seq] - cu.to(dev)[seq + 1] + torch.arange(2, n - 3, device=dev) + 1).repeat_interleave(group)
    k, v = (x[:, 0].double() for x in c.read(table, ln, 120))
    rows, mine, seq = q[2:n - 3].reshape(-1, dim), got[2:n - 3].reshape(-1, dim), seq.repeat_interleave(group)
    for i in range(0, len(rows), 2000):
        s = seq[i:i + 2000]
        close(mine[i:i + 2000], rows[i:i + 2000], k[s], v[s], end[i:i + 2000], kind)
