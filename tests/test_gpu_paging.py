"""Page tables on the GPU against the oracle's, step by step: whole numbers, compared exactly."""
import random

import pytest
import torch

from borch_amd import kv4, paging
from oracle import decode as D
from oracle.paging import Tables
from test_gpu_kv4 import same_pages, values

pytestmark = pytest.mark.gpu


def i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


class Both:
    """The tables on the GPU and the oracle's, kept equal."""

    def __init__(self, dev, sequences, width, pages, page):
        self.dev = dev
        self.gpu = paging.Pages.zeros(sequences, width, pages, page, dev)
        self.ref = Tables(self.gpu.table.tolist(), self.gpu.lens.tolist(), self.gpu.refs.tolist(), page)

    def same(self):
        assert self.gpu.lens.tolist() == self.ref.lens
        assert self.gpu.table.tolist() == self.ref.table
        assert self.gpu.refs.tolist() == self.ref.refs

    def cut(self, to):
        self.gpu.cut(i32(to, self.dev))
        self.ref.cut(to)
        self.same()

    def fork(self, parents):
        self.gpu.fork(i32(parents, self.dev))
        self.ref.fork(parents)
        self.same()

    def grow(self, more, rows):
        got = self.gpu.grow(i32(more, self.dev), rows)
        cu, slots, at, moves, ok = self.ref.grow(more, rows)
        assert got.ok.tolist() == [ok]
        assert got.cu.tolist() == cu and got.moves.tolist() == moves
        assert got.at.tolist() == at and got.slots.tolist() == slots
        self.same()
        return got


@pytest.mark.parametrize("sequences,width,pages,page", [
    (1, 4, 7, 32), (3, 9, 40, 16), (64, 20, 900, 64), (65, 33, 2500, 1), (300, 12, 5000, 96), (1100, 7, 9000, 33)])
def test_steps(dev, sequences, width, pages, page):
    """Prompts, steps, forks, cuts and requests that do not fit, in turn."""
    print(f"pages {sequences} sequences of {width}, {pages} of {page}", flush=True)
    r = random.Random(sequences)
    b = Both(dev, sequences, width, pages, page)
    fits = 0
    for step in range(14):
        kind = step % 7
        if kind == 0:
            b.cut([0 if r.random() < 0.5 else n for n in b.ref.lens])
            more = [r.randint(1, max(1, width * page // 3)) if n == 0 and r.random() < 0.8 else 0 for n in b.ref.lens]
        elif kind == 3:
            more = [r.randint(0, 2 * page) for _ in b.ref.lens]
        else:
            more = [1 if r.random() < 0.8 else 0 for _ in b.ref.lens]
        if kind in (2, 4, 5):
            b.fork([r.randrange(max(1, sequences // 3)) if r.random() < 0.4 else s for s in range(sequences)])
        if kind in (1, 6):
            b.cut([n - r.randint(0, page) for n in b.ref.lens])
        fits += b.grow(more, sum(more) + r.choice([0, 5])).ok.item()
    assert fits >= 7


@pytest.mark.parametrize("pages", [65536, 65537, 200001])
def test_many_pages(dev, pages):
    """Free pages far up, more than one block of them, around the size from which they are counted first."""
    print(f"pages of {pages}", flush=True)
    width = 2200
    b = Both(dev, 2, width, pages, 32)
    taken = pages - 4300
    b.gpu.refs[:taken] = 1
    holes = torch.tensor([5, 4095, 4096, 30000, taken - 5], device=dev)
    b.gpu.refs[holes] = 0
    b.ref.refs = b.gpu.refs.tolist()
    assert b.grow([32 * 2100, 32 * 2200], 32 * 4300).ok.item() == 1
    assert b.ref.table[0][:5] == holes.tolist()
    assert b.grow([32, 0], 32).ok.item() == 1
    assert b.grow([32 * 5, 0], 32 * 5).ok.item() == 0  # four are free, and four fit
    assert b.grow([32 * 4, 0], 32 * 4).ok.item() == 1
    assert b.grow([1, 0], 1).ok.item() == 0


@pytest.mark.parametrize("rows", [8192, 8193, 30000])
def test_many_rows(dev, rows):
    """Places written by the plan itself and by a launch of their own."""
    print(f"pages rows {rows}", flush=True)
    b = Both(dev, 5, 1200, 6000, 32)
    b.grow([3, 0, 40, 32, 1], 76)
    b.grow([rows - 700, 0, 77, 0, 500], rows)
    b.cut([0, 0, 117, 32, 0])
    b.grow([0, rows, 0, 0, 0], rows)


@pytest.mark.parametrize("pages", [9000, 65536, 70001])
def test_scattered_pages(dev, pages):
    """Free pages strewn among taken ones, shared last pages among those that grow, for many tokens and for few."""
    print(f"pages scattered {pages}", flush=True)
    r = random.Random(pages)
    sequences, page = 70, 8
    b = Both(dev, sequences, 300, pages, page)
    b.grow([r.randint(0, 100) for _ in range(sequences)], 7000)
    b.fork([s if r.random() < 0.5 else r.randrange(sequences) for s in range(sequences)])
    held = torch.tensor([n == 0 and r.random() < 0.7 for n in b.ref.refs], device=dev)
    b.gpu.refs += held.int()  # pages that others than these sequences hold
    b.ref.refs = b.gpu.refs.tolist()
    free = b.ref.refs.count(0)
    long = min(free // 20 * page, 1000)
    assert b.grow([r.choice([0, 1, page, long]) for _ in range(sequences)], 70000).ok.item() == 1
    b.fork([s if r.random() < 0.5 else r.randrange(sequences) for s in range(sequences)])
    assert b.grow([r.choice([0, 0, 1, 3 * page]) for _ in range(sequences)], 2000).ok.item() == 1


def test_most_sequences(dev):
    """As many sequences as there may be, most of them sharing pages that are partly filled."""
    print("pages of 8192 sequences", flush=True)
    r = random.Random(5)
    b = Both(dev, 8192, 3, 20000, 32)
    b.grow([r.randint(0, 40) for _ in range(8192)], 8192 * 40)
    b.fork([s if r.random() < 0.3 else r.randrange(8192) for s in range(8192)])
    assert b.grow([r.randint(0, 1) for _ in range(8192)], 8192).ok.item() == 1
    b.fork([r.randrange(3) if s % 2 else s for s in range(8192)])
    assert b.grow([1] * 8192, 8192).ok.item() == 1


def test_shared_pages(dev):
    """Who keeps a shared page: the lowest where all that share it grow; nobody where one does not, or has
    filled it."""
    print("pages shared", flush=True)
    b = Both(dev, 5, 4, 30, 32)
    b.grow([40, 64, 5, 0, 0], 109)
    b.fork([0, 1, 2, 0, 0])
    got = b.grow([1, 0, 0, 1, 1], 3)
    assert got.moves[0].tolist()[0] == -1 and got.moves[2].tolist() == [0, 0, 0, 8, 8]
    b.fork([1, 1, 2, 2, 2])
    assert b.grow([1, 1, 0, 1, 1], 4).moves[2].tolist() == [0, 0, 0, 5, 5]  # sequence 2 stays
    b.fork([0, 0, 2, 2, 3])
    b.cut([65, 50, 6, 3, 9])  # one page full for one, partly filled for another
    assert b.grow([1, 1, 0, 0, 0], 2).moves[2].tolist()[1] == 18
    b.fork([-1, 7, 2, 2, 2])
    assert b.ref.lens[:2] == [0, 0]
    b.cut([0] * 5)
    assert not any(b.ref.refs)


def test_no_room(dev):
    """Requests that do not fit as a whole change nothing."""
    print("pages no room", flush=True)
    b = Both(dev, 3, 3, 6, 32)
    b.grow([30, 33, 0], 63)
    for more, rows in (([1, 1, 128], 130), ([3, 64, 0], 66), ([1, -1, 1], 5), ([67, 0, 0], 200), ([0, 64, 0], 64),
                       ([3, 32, 64], 99)):
        assert b.grow(more, rows).ok.item() == 0, more
    assert b.grow([3, 31, 64], 98).ok.item() == 1
    b.fork([0, 0, 1])
    assert b.grow([1, 1, 0], 2).ok.item() == 1
    assert b.grow([0, 0, 0], 0).ok.item() == 1


def test_entries_that_are_no_page(dev):
    """Entries outside the pages count nowhere and give no slot."""
    print("pages bad entries", flush=True)
    b = Both(dev, 3, 3, 8, 32)
    b.grow([40, 10, 33], 83)
    for s, c, v in ((0, 1, -1), (1, 0, 2 ** 31 - 1), (2, 1, 8)):
        b.ref.refs[b.ref.table[s][c]] -= 1
        b.ref.table[s][c] = v
    b.gpu.table.copy_(i32(b.ref.table, dev))
    b.gpu.refs.copy_(i32(b.ref.refs, dev))
    got = b.grow([3, 1, 40], 44)
    assert got.slots[:4].tolist() == [-1] * 4
    b.fork([1, 0, 2])
    b.cut([5, 5, 5])
    b.cut([0, 0, 0])


def test_no_sequences(dev):
    p = paging.Pages.zeros(0, 4, 8, 32, dev)
    none = torch.empty(0, dtype=torch.int32, device=dev)
    p.cut(none)
    p.fork(none)
    got = p.grow(none, 3)
    assert got.cu.tolist() == [0] and got.at.tolist() == [-1] * 3 and got.ok.tolist() == [1]


@pytest.mark.parametrize("dim,heads,page", [(64, 1, 32), (128, 3, 64), (64, 2, 160)])
def test_copy_pages(dev, dim, heads, page):
    """What holds the tokens moves, in every cache; other places stay; moves of no page do nothing."""
    print(f"pages copy dim={dim} heads={heads} page={page}", flush=True)
    pages = 12
    caches, refs = [], []
    for i in range(70):  # more than one launch takes
        g = torch.Generator().manual_seed(i)
        c = kv4.Cache4.zeros(pages, heads, page, dim, dev)
        for t in (c.k, c.k_scales, c.v, c.v_scales):
            t.copy_(torch.randint(0, 255, t.shape, generator=g).to(torch.uint8))
        caches.append(c)
        refs.append(D.Pages(c.k, c.k_scales, c.v, c.v_scales))
    src, dst = [0, 3, -1, 5, 11, 2, pages, 4], [1, 6, 2, -1, 10, pages, 7, 8]
    tokens = [page, 1, 5, 9, page - 1, 7, 3, 0]
    moves = i32([src, dst, tokens], dev)
    paging.copy_pages(caches, moves)
    for c, ref in zip(caches, refs):
        for s, d, n in zip(src, dst, tokens):
            if not (0 <= s < pages and 0 <= d < pages):
                continue
            for off in range(-(-n // 32) * 32):
                for h in range(heads):
                    kc, kb, vc, vb = ref.get(s, h, off)
                    if c is caches[0] or c is caches[-1]:
                        ref.put(d, h, off, kc, kb, vc, vb)
        if c is caches[0] or c is caches[-1]:
            same_pages(c, ref)
        else:
            assert torch.equal(c.k[1], c.k[0]) and torch.equal(c.v_scales[6, :, 0], c.v_scales[3, :, 0])
    paging.copy_pages([], moves)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_append_slots(dev, kind):
    """Rows into given places: the same bytes as by tables; slots in no page are not written."""
    print(f"append slots {kind}", flush=True)
    dim, heads, page = 128, 3, 64
    p = paging.Pages.zeros(3, 4, 12, page, dev)
    p.refs[:2] = 1
    got = p.grow(i32([70, 0, 130], dev), 203)
    x = values(203, heads, dim, kind, 3).to(dev)
    a, b = (kv4.Cache4.zeros(12, heads, page, dim, dev) for _ in range(2))
    a.append(x[:, :heads], x[:, heads:], slots=got.slots)
    b.append(x[:, :heads], x[:, heads:], p.table, p.lens, got.cu)
    for name in ("k", "k_scales", "v", "v_scales"):
        assert torch.equal(getattr(a, name), getattr(b, name)), name
    assert bool(a.k.any())
    bad = torch.tensor([-1, 12 * page, 2 ** 40, -2 ** 40], dtype=torch.int64, device=dev)
    a.append(x[:4, :heads], x[:4, heads:], slots=bad)
    assert torch.equal(a.k, b.k) and torch.equal(a.v_scales, b.v_scales)
    with pytest.raises(RuntimeError, match="slots, or"):
        a.append(x[:4, :heads], x[:4, heads:], p.table, slots=bad)
    with pytest.raises(RuntimeError, match="slots, or"):
        a.append(x[:4, :heads], x[:4, heads:], p.table, p.lens)
    with pytest.raises(TypeError, match="int64"):
        a.append(x[:4, :heads], x[:4, heads:], slots=bad.int())
    with pytest.raises(RuntimeError, match="shape"):
        a.append(x[:3, :heads], x[:3, heads:], slots=bad)


def test_captured(dev):
    """A step captured and replayed, with eager work between: forks, growth and moves as the oracle has them."""
    print("pages captured", flush=True)
    b = Both(dev, 6, 8, 60, 32)
    b.grow([40, 31, 64, 1, 100, 7], 243)
    parents, more, to = (i32(x, dev) for x in ([0] * 6, [1] * 6, [200] * 6))
    cache = kv4.Cache4.zeros(60, 2, 32, 64, dev)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        b.gpu.cut(to)
        b.gpu.fork(parents)
        got = b.gpu.grow(more, 9)
        paging.copy_pages([cache], got.moves)
    r = random.Random(2)
    for step in range(5):
        p = [r.randrange(6) for _ in range(6)]
        m = [r.randint(0, 1) for _ in range(6)] if step < 4 else [2] * 6  # the last asks for too many rows
        t = [n - r.randint(0, 3) for n in b.ref.lens]
        for x, y in ((parents, p), (more, m), (to, t)):
            x.copy_(i32(y, dev))
        graph.replay()
        b.ref.cut(t)
        b.ref.fork(p)
        cu, slots, at, moves, ok = b.ref.grow(m, 9)
        b.same()
        assert (got.cu.tolist(), got.slots.tolist(), got.at.tolist(), got.moves.tolist(), got.ok.tolist()) == \
            (cu, slots, at, moves, [ok])


def test_streams(dev):
    """A step on another stream than the current one's; two states on two streams at once."""
    print("pages streams", flush=True)
    both = [Both(dev, 40, 9, 70000, 32) for _ in range(2)]
    sides = [torch.cuda.Stream(dev) for _ in range(2)]
    r = random.Random(3)
    steps = [([r.randint(0, 90) for _ in range(40)], [r.randrange(40) for _ in range(40)]) for _ in range(6)]
    given = [(i32(m, dev), i32(p, dev)) for m, p in steps]
    torch.cuda.synchronize()
    got = [[], []]
    for m, p in given:
        for b, side, g in zip(both, sides, got):
            with torch.cuda.stream(side):
                g.append(b.gpu.grow(m, 4000))
                b.gpu.fork(p)
    torch.cuda.synchronize()
    for b, g in zip(both, got):
        for (m, p), x in zip(steps, g):
            cu, slots, at, moves, ok = b.ref.grow(m, 4000)
            assert (x.cu.tolist(), x.slots.tolist(), x.at.tolist(), x.moves.tolist(), x.ok.tolist()) == \
                (cu, slots, at, moves, [ok])
            b.ref.fork(p)
        b.same()


def test_captured_many(dev):
    """Many pages and many tokens, whose launches share a workspace: captured, replayed with eager calls between."""
    print("pages captured, many", flush=True)
    b = Both(dev, 9, 2000, 70000, 8)
    b.grow([9000, 10, 0, 777, 0, 0, 64, 1, 3], 10000)
    parents, more, to = (i32(x, dev) for x in ([0] * 9, [1] * 9, [200] * 9))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        b.gpu.cut(to)
        b.gpu.fork(parents)
        got = b.gpu.grow(more, 9001)
    r = random.Random(7)
    for step in range(4):
        p = [r.randrange(9) for _ in range(9)]
        t = [n - r.randint(0, 5000) for n in b.ref.lens]
        m = [r.choice([0, 1, 300, 4000]) if sum(t) else 1 for _ in range(9)]
        m = [0 if sum(m[:i + 1]) > 9001 else n for i, n in enumerate(m)]
        for x, y in ((parents, p), (more, m), (to, t)):
            x.copy_(i32(y, dev))
        graph.replay()
        b.ref.cut(t)
        b.ref.fork(p)
        cu, slots, at, moves, ok = b.ref.grow(m, 9001)
        b.same()
        assert (got.cu.tolist(), got.slots.tolist(), got.at.tolist(), got.moves.tolist(), got.ok.tolist()) == \
            (cu, slots, at, moves, [ok])
        b.grow([5] * 9, 9000)  # eager, into what is free by now


def test_refusals(dev):
    p = paging.Pages.zeros(3, 4, 8, 32, dev)
    x = torch.zeros(3, dtype=torch.int32, device=dev)
    with pytest.raises(TypeError, match="int32"):
        p.cut(x.long())
    with pytest.raises(RuntimeError, match="shape"):
        p.fork(x[:2])
    with pytest.raises(RuntimeError, match="cpu"):
        p.grow(x.cpu(), 3)
    with pytest.raises(ValueError, match="rows"):
        p.grow(x, -1)
    with pytest.raises(RuntimeError, match="moves"):
        paging.copy_pages([kv4.Cache4.zeros(2, 1, 32, 64, dev)], x)
    with pytest.raises(RuntimeError, match="contiguous"):
        paging.Pages(p.table.t(), p.lens[:1].expand(4), p.refs, 32)
    with pytest.raises(NotImplementedError, match="8192"):
        q = paging.Pages.zeros(8193, 1, 8, 32, dev)
        q.cut(torch.zeros(8193, dtype=torch.int32, device=dev))
