"""Attention of chunks of new tokens over the 4-bit cache, against float64 over what the cache holds.

Tolerance, relative to sum_i p_i |v_i|: the scores' f32 error twice (oracle's score_error; q as up to three
pieces), (3 n + 64) 2^-24 for the f32 sums over n tokens of up to three pieces, the joined parts and the
quotient; for f16 2^-16 (p as two bf16 pieces), for bf16 2^-8 (p rounded to bf16, half a step); and half a step
of the output."""
import math

import pytest
import torch

from borch_amd import kv4
from oracle import decode as D
from test_gpu_kv4 import HALF, LEAST, PIECES, TYPES, filled, starts

pytestmark = pytest.mark.gpu

WEIGHT = {"f32": 0.0, "bf16": 2.0 ** -8, "f16": 2.0 ** -16}


def queries(n, heads, dim, kind, seed):
    return torch.randn(n, heads, dim, generator=torch.Generator().manual_seed(seed)).to(TYPES[kind])


def check(got, q, k, v, there, lens, cu, most, kind, scale=None):
    """k, v [B, heads, >= most, dim] float64 and which places hold a token; rows of no sequence are zeros."""
    n, hq, dim = q.shape
    h = k.shape[1]
    group, got = hq // h, got.cpu().double()
    scale = 1.0 / math.sqrt(dim) if scale is None else scale
    of_none = torch.ones(n, dtype=torch.bool)
    for b in range(len(lens)):
        s, e = int(cu[b]), int(cu[b + 1])
        of_none[s:e] = False
        if s == e:
            continue
        end = torch.arange(s, e) + int(lens[b]) - e + 1
        end = end.clamp(0, min(int(lens[b]), most)).repeat_interleave(group)
        seen = there[b] & (torch.arange(there.shape[1]) < end[:, None])
        last = max(int(end.max()), 1)
        for j in range(h):
            qs = q[s:e, j * group:(j + 1) * group].reshape(-1, dim)
            want, _, size = D.softmax_rows(qs, k[b, j, :last], v[b, j, :last], seen[:, :last], scale)
            err = D.score_error(qs, k[b, j, :last], scale, PIECES[kind])
            rel = err + (3 * last + 64) * 2.0 ** -24 + WEIGHT[kind]
            tol = size * rel + want.abs() * (HALF[kind] + 2.0 ** -24) + LEAST[kind]
            tol = tol + last * 2.0 ** -126 * v[b, j, :last].nan_to_num(0, 0, 0).abs().amax(0)
            mine = got[s:e, j * group:(j + 1) * group].reshape(-1, dim)
            fine = torch.isfinite(want)
            assert torch.equal(want.isnan(), mine.isnan()), (b, j)
            assert torch.equal(want[~fine & ~want.isnan()], mine[~fine & ~want.isnan()]), (b, j)
            off = (mine - want).abs()
            assert bool((off[fine] <= tol[fine]).all()), (b, j, float((off[fine] / tol[fine]).max()))
    assert not bool(got[of_none].any())


def held(c, table, lens, most, dev):
    k, v = (x.cpu().double() for x in c.read(table.to(dev), lens.to(dev), most))
    return k, v, torch.arange(most)[None] < lens[:, None]


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens,new,h,group,page", [
    ([1], [1], 1, 1, 32), ([0, 31, 64, 33], [0, 31, 1, 2], 2, 3, 32), ([300, 5], [40, 5], 3, 1, 64),
    ([129, 0, 700], [129, 0, 33], 2, 4, 128), ([40, 3, 65], [11, 3, 65], 1, 6, 32), ([1000], [7], 1, 16, 256),
    ([200, 97], [64, 1], 2, 8, 96), ([260, 259, 1], [130, 257, 1], 1, 5, 64), ([513], [512], 1, 1, 64),
    # from here on wide tiles, beside narrow ones: more than 2048 rows in all, sequences of more than 64
    ([400, 33, 700], [140, 1, 3], 1, 16, 32), ([300, 90, 0], [129, 12, 0], 2, 18, 96), ([2100, 64], [2050, 3], 1, 1, 64),
    ([180] * 17 + [77, 300], [5] * 17 + [4, 127], 1, 16, 64), ([140, 129], [140, 129], 1, 8, 128)])
def test_chunk_against_float64(dev, kind, dim, lens, new, h, group, page):
    print(f"kv4 chunk {kind} dim={dim} lens={lens} new={new} heads={h}x{group} page={page}", flush=True)
    c, table, ln, _ = filled(dev, lens, h, dim, page, 31)
    most = max(lens)
    cu = starts(new)
    q = queries(sum(new), h * group + 2 * h, dim, kind, 5)
    k, v, there = held(c, table, ln, most, dev)
    qd, td, ld, cd = q.to(dev)[:, :h * group], table.to(dev), ln.to(dev), cu.to(dev)
    got = c.attend_chunk(qd, td, ld, cd, max_len=most)
    check(got, q[:, :h * group], k, v, there, ln, cu, most, kind)
    assert torch.equal(got, c.attend_chunk(qd.contiguous(), td, ld, cd, max_len=most))
    check(c.attend_chunk(qd, td, ld, cd), q[:, :h * group], k, v, there, ln, cu, most, kind)


@pytest.mark.parametrize("kind,dim,group", [("f32", 128, 1), ("bf16", 64, 2), ("f16", 128, 4), ("bf16", 128, 7),
                                            ("bf16", 64, 20), ("f32", 128, 20), ("f16", 64, 32)])
def test_chunk_in_shares(dev, kind, dim, group):
    """Few rows over a long axis: a row's keys in many shares, joined; beside them short sequences; a caller's
    max_len beyond every length; lengths cut by it."""
    print(f"kv4 chunk shares {kind} dim={dim} group={group}", flush=True)
    lens, new = [9000, 1, 2049, 40], [3, 1, 70, 40]
    c, table, ln, _ = filled(dev, lens, 1, dim, 64, 21, "bf16")
    cu = starts(new)
    q = queries(sum(new), group, dim, kind, 9)
    k, v, there = held(c, table, ln, 9000, dev)
    for most in (9000, None, 20000):
        got = c.attend_chunk(q.to(dev), table.to(dev), ln.to(dev), cu.to(dev), max_len=most)
        check(got, q, k, v, there, ln, cu, 9000, kind)
    got = c.attend_chunk(q.to(dev), table.to(dev), ln.to(dev), cu.to(dev), max_len=2048, scale=0.3)  # cut
    check(got, q, k[:, :, :2048], v[:, :, :2048], there[:, :2048], ln, cu, 2048, kind, scale=0.3)


@pytest.mark.parametrize("count,kind,dim", [(62, "f32", 64), (63, "bf16", 128), (200, "f16", 64), (700, "bf16", 64)])
def test_chunk_many_sequences(dev, count, kind, dim):
    """More sequences than lanes, most of them of a token or none, one of many rows and some in between."""
    print(f"kv4 chunk {count} sequences {kind} dim={dim}", flush=True)
    lens = [(i * 37) % 71 for i in range(count)]
    new = [min(n, (i * 5) % 3) for i, n in enumerate(lens)]
    lens[count // 2], new[count // 2] = 300, 200
    lens[count - 7], new[count - 7] = 90, 30
    c, table, ln, _ = filled(dev, lens, 1, dim, 32, 21)
    cu = starts(new) + 3  # rows of no sequence before the first, and past the last
    q = queries(sum(new) + 7, 4, dim, kind, 6)
    k, v, there = held(c, table, ln, 300, dev)
    got = c.attend_chunk(q.to(dev), table.to(dev), ln.to(dev), cu.to(dev), max_len=300)
    check(got, q, k, v, there, ln, cu, 300, kind)
    assert not bool(got[:3].any()) and not bool(got[-4:].any())


def test_chunk_rows_of_no_sequence(dev):
    """Rows before the first sequence and past the last one, and rows whose token lies before the cache's
    first: zeros."""
    print("kv4 chunk rows of no sequence", flush=True)
    lens = [40, 33, 3]
    c, table, ln, _ = filled(dev, lens, 2, 64, 32, 37)
    cu = torch.tensor([6, 9, 9, 14], dtype=torch.int32)  # five rows of a sequence of three tokens
    q = queries(19, 4, 64, "f32", 3)
    k, v, there = held(c, table, ln, 40, dev)
    got = c.attend_chunk(q.to(dev), table.to(dev), ln.to(dev), cu.to(dev))
    check(got, q, k, v, there, ln, cu, 40, "f32")
    assert not bool(got[9:11].any()) and bool(got[11:14].any(-1).all())
    none = torch.full((4,), 7, dtype=torch.int32)
    assert not bool(c.attend_chunk(q.to(dev), table.to(dev), ln.to(dev), none.to(dev)).any())


@pytest.mark.parametrize("group", [3, 32])
def test_chunk_entries_that_are_no_page(dev, group):
    print(f"kv4 chunk bad pages group={group}", flush=True)
    lens, new = [200, 140], [70, 9]
    c, table, ln, _ = filled(dev, lens, 2, 64, 32, 6)
    table = table.clone()
    table[0, 1], table[0, 2], table[1, 0] = -1, c.pages, 2 ** 31 - 1
    ln, cu = torch.tensor([200, 170], dtype=torch.int32), starts(new)  # past the table's pages too
    ref = D.Pages(c.k, c.k_scales, c.v, c.v_scales)
    k, v, there = ref.read(table, ln, 224)
    for kind in ("f32", "bf16"):
        q = queries(sum(new), 2 * group, 64, kind, 1)
        got = c.attend_chunk(q.to(dev), table.to(dev), ln.to(dev), cu.to(dev))
        check(got, q, k, v, there, ln, cu, 224, kind)


@pytest.mark.parametrize("dim,rows,group", [(64, 8, 1), (128, 8, 1), (128, 40, 1), (64, 100, 1), (64, 70, 32), (128, 100, 21)])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("bad", [0, 40, 97, 99, 101])
def test_chunk_what_is_not_seen_does_not_count(dev, dim, rows, group, which, bad):
    """A NaN among the tokens reaches the rows that see it, a value's in its 32 channels; NaN past the length,
    in the same page, reaches none. In narrow tiles and (more than 2048 rows) in wide ones."""
    print(f"kv4 chunk NaN dim={dim} rows={rows} group={group} {which}[{bad}]", flush=True)
    c, table, _, x = filled(dev, [160], 1, dim, 64, 23)
    ln, cu = torch.tensor([100], dtype=torch.int32), starts([rows])
    x = x.clone()
    x[bad, 0 if which == "k" else 1, 33] = math.nan
    c.append(x[:, :1].to(dev), x[:, 1:].to(dev), table.to(dev), torch.tensor([160], dtype=torch.int32, device=dev),
             starts([160]).to(dev))
    q = queries(rows, group, dim, "bf16", 2)
    ref = D.Pages(c.k, c.k_scales, c.v, c.v_scales)
    k, v, there = ref.read(table, ln, 100)
    got = c.attend_chunk(q.to(dev), table.to(dev), ln.to(dev), cu.to(dev)).cpu()
    check(got, q, k, v, there, ln, cu, 100, "bf16")
    sees = torch.arange(100 - rows, 100) >= bad
    sees = sees[:, None].expand(rows, group)
    if which == "v":
        assert torch.equal(got.isnan().any(-1), sees) and not got[:, :, :32].isnan().any()
    else:
        assert torch.equal(got.isnan().all(-1), sees) and torch.equal(got.isnan().any(-1), sees)


def test_chunk_infinite_values(dev):
    """A value that the cache holds as infinite, among the newest tokens: infinite where it is seen, not NaN
    where it is not."""
    print("kv4 chunk infinite values", flush=True)
    for dim, rows, group in ((64, 8, 1), (128, 50, 1), (128, 90, 1), (64, 90, 32), (128, 90, 24)):
        c, table, ln, x = filled(dev, [100], 1, dim, 64, 23)
        x = x.clone()
        x[95, 1, 5], x[97, 1, 40] = 3.3e38, -3.3e38
        c.append(x[:, :1].to(dev), x[:, 1:].to(dev), table.to(dev), ln.to(dev), starts([100]).to(dev))
        q = queries(rows, group, dim, "f32", 2)
        k, v, there = held(c, table, ln, 100, dev)
        assert bool(v.isinf().any())
        got = c.attend_chunk(q.to(dev), table.to(dev), ln.to(dev), starts([rows]).to(dev)).cpu()
        fine = got[:rows - 5]
        assert bool(torch.isfinite(fine).all())
        want = torch.zeros(5, group, dim)
        want[:, :, 5] = math.inf
        want[2:, :, 40] = -math.inf
        assert torch.equal(torch.where(got[rows - 5:].isinf(), got[rows - 5:], torch.zeros(())), want)
        assert not bool(got.isnan().any())


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,heads", [(3, 2), (40, 2), (130, 2), (130, 17)])
def test_chunk_queries_at_the_ends(dev, kind, rows, heads):
    """Infinite and NaN queries make their own rows NaN and no other; the largest finite ones and scores far
    beyond 2^20 decide by the largest score; zeros weigh all alike."""
    print(f"kv4 chunk extreme queries {kind} rows={rows} heads={heads}", flush=True)
    dim, n = 64, 200
    c, table, ln, _ = filled(dev, [n], 1, dim, 64, 29, "f32")
    q = queries(rows, heads, dim, kind, 4).float()
    q[0, 0, 3], q[1, 1, 7] = math.inf, math.nan
    q[2, 0] = 0.0
    q[1, 0] *= 1.0e4 if kind == "f16" else 1e9
    q = q.to(TYPES[kind])
    cu = starts([rows])
    k, v, there = held(c, table, ln, n, dev)
    got = c.attend_chunk(q.to(dev), table.to(dev), ln.to(dev), cu.to(dev)).cpu()
    assert bool(got[0, 0].isnan().all()) and bool(got[1, 1].isnan().all())
    others = torch.ones(rows, heads, dtype=torch.bool)
    others[0, 0] = others[1, 1] = False
    assert bool(torch.isfinite(got[others]).all())
    # a row whose scores are far apart takes the value of the largest
    end = n - rows + 2
    s = (k[0, 0, :end] * q[1, 0].double()).sum(-1)
    assert float(s.topk(2).values.diff().abs()) * dim ** -0.5 > 200
    best = v[0, 0, int(s.argmax())]
    assert bool(((got[1, 0].double() - best).abs() <= best.abs() * (HALF[kind] + WEIGHT[kind] + 2.0 ** -22)).all())
    clean = q.clone()
    clean[0, 0], clean[1, 1], clean[1, 0] = 0, 0, 0
    check(c.attend_chunk(clean.to(dev), table.to(dev), ln.to(dev), cu.to(dev)), clean, k, v, there, ln, cu, n, kind)


def test_chunk_agrees_with_attend(dev):
    """The same tokens through attend: both within their bounds of the same result."""
    print("kv4 chunk beside attend", flush=True)
    lens = [77, 130, 64]
    c, table, ln, _ = filled(dev, lens, 2, 128, 64, 41)
    q = queries(3 * 9, 8, 128, "f32", 8).to(dev)
    td, ld = table.to(dev), ln.to(dev)
    a = c.attend_chunk(q, td, ld, starts([9] * 3).to(dev))
    b = c.attend(q.view(3, 9, 8, 128), td, ld).view(27, 8, 128)
    assert float((a - b).abs().max()) <= 2.0 ** -16 * float(b.abs().max())


def test_chunk_strides_and_streams(dev):
    """Queries at odd addresses, in other orders and expanded; another stream than the current one's; a graph
    replayed over changed lengths."""
    print("kv4 chunk strides, streams, graph", flush=True)
    lens, new = [150, 90], [40, 33]
    c, table, ln, _ = filled(dev, lens, 2, 64, 32, 3)
    td, ld, cd = table.to(dev), ln.to(dev), starts(new).to(dev)
    long = queries(73, 128, 64, "f16", 7).to(dev)  # wide tiles
    assert torch.equal(c.attend_chunk(long.transpose(0, 1).contiguous().transpose(0, 1), td, ld, cd),
                       c.attend_chunk(long, td, ld, cd))
    q = queries(73, 4, 64, "f16", 6).to(dev)
    want = c.attend_chunk(q, td, ld, cd)
    odd = torch.empty(73 * 4 * 64 + 1, dtype=torch.float16, device=dev)[1:].view(73, 4, 64)
    odd.copy_(q)
    assert torch.equal(c.attend_chunk(odd, td, ld, cd), want)
    turned = q.permute(1, 2, 0).contiguous().permute(2, 0, 1)
    assert torch.equal(c.attend_chunk(turned, td, ld, cd), want)
    heads_first = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(c.attend_chunk(heads_first, td, ld, cd), want)
    one = q[:, :1].expand(73, 4, 64)
    assert torch.equal(c.attend_chunk(one, td, ld, cd), c.attend_chunk(one.contiguous(), td, ld, cd))
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        got = c.attend_chunk(q, td, ld, cd)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = c.attend_chunk(q, td, ld, cd, max_len=4096)
    for less in (0, 30, 7):
        ld.copy_(ln - less)
        graph.replay()
        eager = c.attend_chunk(q, td, ld, cd, max_len=4096)
        torch.cuda.synchronize()
        assert torch.equal(out, eager), less


def test_chunk_refusals(dev):
    c, table, ln, _ = filled(dev, [40], 2, 64, 32, 3)
    td, ld, cd = table.to(dev), ln.to(dev), starts([3]).to(dev)
    q = torch.zeros(3, 4, 64, device=dev)
    with pytest.raises(RuntimeError, match="key-value heads"):
        c.attend_chunk(q[:, :3], td, ld, cd)
    with pytest.raises(RuntimeError, match="key-value heads"):
        c.attend_chunk(q[None], td, ld, cd)
    with pytest.raises(TypeError, match="float64"):
        c.attend_chunk(q.double(), td, ld, cd)
    with pytest.raises(RuntimeError, match="cu"):
        c.attend_chunk(q, td, ld, torch.zeros(3, dtype=torch.int32, device=dev))
    with pytest.raises(TypeError, match="cu"):
        c.attend_chunk(q, td, ld, cd.long())
    with pytest.raises(RuntimeError, match="cpu"):
        c.attend_chunk(q.cpu(), td, ld, cd)
    with pytest.raises(RuntimeError, match="gradient"):
        c.attend_chunk(q.requires_grad_(), td, ld, cd)
    q = q.detach()
    for scale in (0.0, -1.0, math.nan, math.inf):
        with pytest.raises(ValueError, match="scale"):
            c.attend_chunk(q, td, ld, cd, scale=scale)
    with pytest.raises(ValueError, match="sizes"):
        c.attend_chunk(q, td, ld, cd, max_len=-1)
    assert c.attend_chunk(q[:0], td, ld, starts([0]).to(dev)).shape == (0, 4, 64)
