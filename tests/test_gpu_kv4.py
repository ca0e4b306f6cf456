"""The 4-bit key-value cache against its description, token by token, and float64 (oracle/decode.py).

Codes, scales, places and kept tokens are compared exactly. Tolerance of attention, relative to
sum_i p_i |v_i|: the scores' f32 error twice (oracle's score_error; q as up to three pieces), (3 n +
64) 2^-24 for the f32 sums over n tokens of up to three pieces, the joined parts and the quotient, and
for the 16-bit types 2^-16 (p as two bf16 pieces) and half a step of the output. A token's received
weight: each of its r rows within the scores' error and (n + 64) 2^-24 of its p, and r + 1 additions."""
import math

import pytest
import torch

from borch_amd import kv4
from oracle import decode as D

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HALF = {"f32": 0.0, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
LEAST = {"f32": 2.0 ** -149, "bf16": 2.0 ** -133, "f16": 2.0 ** -24}
PIECES = {"f32": 3, "bf16": 1, "f16": 2}


def tables(lens, page, seed, spare=2, width=None):
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    width = max(need + [1]) if width is None else width
    order = torch.randperm(sum(need) + spare, generator=g)
    t = torch.full((len(lens), width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        t[b, :n] = order[at:at + n].int()
        at += n
    return t, sum(need) + spare


def starts(new):
    cu = [0]
    for m in new:
        cu.append(cu[-1] + m)
    return torch.tensor(cu, dtype=torch.int32)


def values(n, h, dim, kind, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, 2 * h, dim, generator=g) * torch.exp(2 * torch.randn(n, 2 * h, 1, generator=g))
    return x.to(TYPES[kind])


def filled(dev, lens, h, dim, page, seed, kind="f32"):
    table, pages = tables(lens, page, seed)
    c = kv4.Cache4.zeros(pages, h, page, dim, dev)
    x = values(sum(lens), h, dim, kind, seed)
    ln = torch.tensor(lens, dtype=torch.int32)
    c.append(x[:, :h].to(dev), x[:, h:].to(dev), table.to(dev), ln.to(dev), starts(lens).to(dev))
    return c, table, ln, x


def same_pages(c, ref):
    for name, a, b in (("k", c.k, ref.k), ("k_scales", c.k_scales, ref.ks), ("v", c.v, ref.v), ("v_scales", c.v_scales, ref.vs)):
        assert torch.equal(a.cpu(), b), name


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim,h,page,lens,new", [
    (128, 2, 32, [5, 33, 0, 40], [5, 33, 0, 40]), (64, 3, 64, [70, 1, 65], [70, 1, 65]),
    (128, 1, 96, [100, 97], [3, 50]), (64, 1, 32, [64, 31, 32], [1, 1, 1])])
def test_append_and_read(dev, kind, dim, h, page, lens, new):
    print(f"kv4 append {kind} dim={dim} heads={h} page={page} lens={lens} new={new}", flush=True)
    table, pages = tables(lens, page, 4)
    c = kv4.Cache4.zeros(pages, h, page, dim, dev)
    ref = D.Pages(c.k, c.k_scales, c.v, c.v_scales)
    x = values(sum(new), h, dim, kind, 8)
    ln, cu = torch.tensor(lens, dtype=torch.int32), starts(new)
    xd = x.to(dev)
    c.append(xd[:, :h], xd[:, h:], table.to(dev), ln.to(dev), cu.to(dev))
    ref.append(x[:, :h].float(), x[:, h:].float(), table, ln, cu)
    same_pages(c, ref)
    most = max(lens) + 3
    k, v = c.read(table.to(dev), ln.to(dev), most)
    wk, wv, _ = ref.read(table, ln, most)
    assert torch.equal(k.cpu().double(), wk) and torch.equal(v.cpu().double(), wv)
    k2, _ = c.read(table.to(dev), ln.to(dev), 2)  # cut short
    assert torch.equal(k2.cpu(), k.cpu()[:, :, :2])


def test_append_rows_of_no_sequence(dev):
    """Rows before the first sequence and past the last one: what the cache held stays."""
    print("kv4 append rows of no sequence", flush=True)
    lens, h, dim, page = [40, 33, 70], 2, 64, 32
    c, table, ln, _ = filled(dev, lens, h, dim, page, 37)
    ref = D.Pages(c.k, c.k_scales, c.v, c.v_scales)
    x = values(19, h, dim, "f32", 12)
    cu = torch.tensor([6, 9, 9, 14], dtype=torch.int32)
    c.append(x[:, :h].to(dev), x[:, h:].to(dev), table.to(dev), ln.to(dev), cu.to(dev))
    ref.append(x[:, :h], x[:, h:], table, ln, cu)
    same_pages(c, ref)


def test_append_extremes(dev):
    """Rounding ties, signed zeros, exponents at both ends, blocks that are not finite."""
    print("kv4 extremes", flush=True)
    rows = []
    for e in (-149, -140, -130, -127, -126, -125, -64, -3, 0, 1, 60, 120, 125):
        for peak in (1.0, 1.25, 1.5, 1.5000001, 1.75, 1.9999999):
            r = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 0.0, 0.125] * 4, dtype=torch.float64)[:32]
            r = r * torch.tensor([1.0, -1.0, 1.0, 1.0] * 8, dtype=torch.float64) * 2.0 ** (e - 2)
            r[3] = peak * 2.0 ** e
            rows.append(r.float())
    rows.append(torch.zeros(32))
    rows.append(-torch.zeros(32))
    for odd in (math.nan, math.inf, -math.inf):
        r = torch.ones(32)
        r[7] = odd
        rows.append(r)
    rows.append(torch.full((32,), torch.finfo(torch.float32).max))
    while len(rows) % 4:
        rows.append(torch.ones(32))
    x = torch.stack(rows).reshape(-1, 1, 128)
    n = x.shape[0]
    table, pages = tables([n], 32, 1)
    c = kv4.Cache4.zeros(pages, 1, 32, 128, dev)
    ref = D.Pages(c.k, c.k_scales, c.v, c.v_scales)
    ln, cu = torch.tensor([n], dtype=torch.int32), starts([n])
    c.append(x.to(dev), x.to(dev), table.to(dev), ln.to(dev), cu.to(dev))
    ref.append(x, x, table, ln, cu)
    same_pages(c, ref)
    k, v = c.read(table.to(dev), ln.to(dev), n)
    wk, wv, _ = ref.read(table, ln, n)
    for got, want in ((k, wk), (v, wv)):
        want = want.float()  # what f32 cannot hold is infinite
        assert torch.equal(got.cpu().isnan(), want.isnan())
        assert torch.equal(got.cpu().nan_to_num(), want.nan_to_num())


def test_entries_that_are_no_page(dev):
    print("kv4 bad pages", flush=True)
    lens = [100, 64]
    table, pages = tables(lens, 32, 6)
    table[0, 1], table[0, 2], table[1, 0] = -1, pages, 2 ** 31 - 1
    c = kv4.Cache4.zeros(pages, 2, 32, 64, dev)
    ref = D.Pages(c.k, c.k_scales, c.v, c.v_scales)
    x = values(sum(lens), 2, 64, "f32", 2)
    # lengths past the table's pages too
    ln, cu = torch.tensor([100, 70], dtype=torch.int32), starts(lens)
    td, ld = table.to(dev), ln.to(dev)
    c.append(x[:, :2].to(dev), x[:, 2:].to(dev), td, ld, cu.to(dev))
    ref.append(x[:, :2], x[:, 2:], table, ln, cu)
    same_pages(c, ref)
    k, v = c.read(td, ld, 128)
    wk, wv, there = ref.read(table, ln, 128)
    assert torch.equal(k.cpu().double(), wk) and torch.equal(v.cpu().double(), wv)
    q = torch.randn(2, 1, 4, 64, generator=torch.Generator().manual_seed(1))
    w = torch.zeros(2, 2, 128, device=dev)
    got = c.attend(q.to(dev), td, ld, weights=w)
    check_attend(got, w, q, wk, wv, there, ln, 128, "f32")


def check_attend(got, w, q, k, v, there, lens, most, kind, w0=None, scale=None):
    B, T, hq, dim = q.shape
    h = k.shape[1]
    scale = 1.0 / math.sqrt(dim) if scale is None else scale
    group, got = hq // h, got.cpu().double()
    for b in range(B):
        n = min(int(lens[b]), most)
        for j in range(h):
            qs = q[b, :, j * group:(j + 1) * group].reshape(-1, dim)
            end = [n - T + 1 + t for t in range(T) for _ in range(group)]
            seen = torch.stack([there[b] & (torch.arange(there.shape[1]) < max(e, 0)) for e in end])
            want, p, size = D.softmax_rows(qs, k[b, j], v[b, j], seen, scale)
            err = D.score_error(qs, k[b, j, :max(n, 1)], scale, PIECES[kind])
            rel = err + (3 * n + 64) * 2.0 ** -24 + (2.0 ** -16 if kind != "f32" else 0)
            tol = size * rel + want.abs() * (HALF[kind] + 2.0 ** -24) + LEAST[kind]
            tol = tol + n * 2.0 ** -126 * v[b, j].nan_to_num(0, 0, 0).abs().amax(0)
            mine = got[b, :, j * group:(j + 1) * group].reshape(-1, dim)
            fine = torch.isfinite(want)
            assert torch.equal(want.isnan(), mine.isnan()), (b, j)
            off = (mine - want).abs()
            assert bool((off[fine] <= tol[fine]).all()), (b, j, float(off[fine].max()), float(tol[fine].max()))
            if w is not None:
                add = w[b, j].cpu().double()
                first = torch.zeros_like(add) if w0 is None else w0[b, j].double()
                total = first.clone()
                total[:p.shape[1]] += p.sum(0)
                bound = p.sum(0) * (err + (n + 64 + len(end)) * 2.0 ** -24) + len(end) * 2.0 ** -126
                slack = total.abs() * 2.0 ** -23
                slack[:p.shape[1]] += bound
                ok = torch.isfinite(total)
                assert torch.equal(ok, torch.isfinite(add)), (b, j)
                assert bool(((add - total).abs()[ok] <= slack[ok]).all()), (b, j)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens,h,group,page,tokens,weights", [
    ([1], 1, 1, 32, 1, False), ([0, 31, 32, 33], 2, 3, 32, 1, True), ([300, 5], 3, 1, 64, 1, False),
    ([129, 0, 700], 2, 4, 128, 2, True), ([40, 3, 65], 1, 6, 32, 5, True), ([1000], 1, 16, 256, 3, True),
    ([90, 64], 2, 8, 96, 9, False)])
def test_attend_against_float64(dev, kind, dim, lens, h, group, page, tokens, weights):
    print(f"kv4 attend {kind} dim={dim} lens={lens} heads={h}x{group} page={page} tokens={tokens}", flush=True)
    c, table, ln, _ = filled(dev, lens, h, dim, page, 17)
    most = max(lens)
    ref = D.Pages(c.k, c.k_scales, c.v, c.v_scales)
    k, v, there = ref.read(table, ln, max(most, 1))
    g = torch.Generator().manual_seed(3)
    q = torch.randn(len(lens), tokens, h * group + 2 * h, dim, generator=g).to(TYPES[kind])
    w0 = torch.rand(len(lens), h, max(most, 1) + 5, generator=g)
    w = w0.to(dev) if weights else None
    qd = q.to(dev)[:, :, :h * group]  # the heads of a fused projection
    got = c.attend(qd, table.to(dev), ln.to(dev), max_len=most, weights=w)
    check_attend(got, w, q[:, :, :h * group], k, v, there, ln, most, kind, w0)
    assert torch.equal(c.attend(qd.contiguous(), table.to(dev), ln.to(dev)), c.attend(qd, table.to(dev), ln.to(dev)))


@pytest.mark.parametrize("kind,dim,tokens", [("f32", 128, 1), ("bf16", 64, 2), ("f16", 128, 1)])
def test_attend_long(dev, kind, dim, tokens):
    """Several chunks of a sequence, joined; a caller's max_len beyond every length."""
    print(f"kv4 attend long {kind} dim={dim}", flush=True)
    lens = [3000, 1, 2049]
    c, table, ln, _ = filled(dev, lens, 1, dim, 64, 21)
    k, v = (x.cpu().double() for x in c.read(table.to(dev), ln.to(dev), 3000))
    there = torch.arange(3000)[None] < ln[:, None]
    q = torch.randn(3, tokens, 4, dim, generator=torch.Generator().manual_seed(9)).to(TYPES[kind])
    wide = torch.full((3, 200), -1, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    for t, most in ((table, 3000), (wide, None), (wide, 9000)):
        w = torch.zeros(3, 1, 12800, device=dev)
        got = c.attend(q.to(dev), t.to(dev), ln.to(dev), max_len=most, weights=w)
        check_attend(got, w, q, k, v, there, ln, 3000, kind)
    got = c.attend(q.to(dev), table.to(dev), ln.to(dev), max_len=2048, scale=0.3)  # cut
    check_attend(got, None, q, k[:, :, :2048], v[:, :, :2048], there[:, :2048], ln, 2048, kind, scale=0.3)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("lens", [[300000], [3] * 31 + [100000] + [3] * 29])
def test_attend_in_many_parts(dev, kind, lens):
    """More parts of a row than the waves that join them take at once."""
    print(f"kv4 attend many parts {kind} {len(lens)}", flush=True)
    c, table, ln, _ = filled(dev, lens, 1, 64, 256, 43, "bf16")
    most = max(lens)
    q = torch.randn(len(lens), 1, 2, 64, generator=torch.Generator().manual_seed(5)).to(TYPES[kind])
    got = c.attend(q.to(dev), table.to(dev), ln.to(dev), max_len=most)
    for b in sorted({0, lens.index(most), len(lens) - 1}):
        k, v = (x.cpu().double() for x in c.read(table[b:b + 1].to(dev), ln[b:b + 1].to(dev), lens[b]))
        there = torch.ones(1, lens[b], dtype=torch.bool)
        check_attend(got[b:b + 1], None, q[b:b + 1], k, v, there, ln[b:b + 1], lens[b], kind)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("bad", [0, 40, 97, 98, 99])
def test_what_is_not_seen_does_not_count(dev, dim, which, bad):
    """A NaN among the newest tokens reaches the queries that see it, in its 32 channels; NaN past the
    length, in the same page, reaches none."""
    print(f"kv4 NaN dim={dim} {which}[{bad}]", flush=True)
    lens = [100]
    c, table, ln, x = filled(dev, [110], 1, dim, 64, 23)
    ln = torch.tensor(lens, dtype=torch.int32)
    q = torch.randn(1, 4, 3, dim, generator=torch.Generator().manual_seed(2))
    td, ld = table.to(dev), ln.to(dev)
    clean = c.attend(q.to(dev), td, ld)
    x = x.clone()
    x[bad, 0 if which == "k" else 1, 35] = math.nan
    x[100:] = math.nan
    c.append(x[:, :1].to(dev), x[:, 1:].to(dev), td, torch.tensor([110], dtype=torch.int32, device=dev),
             starts([110]).to(dev))
    ref = D.Pages(c.k, c.k_scales, c.v, c.v_scales)
    k, v, there = ref.read(table, ln, 100)
    w = torch.zeros(1, 1, 128, device=dev)
    got = c.attend(q.to(dev), td, ld, weights=w)
    check_attend(got, w, q, k, v, there, ln, 100, "f32")
    unseen = [t for t in range(4) if bad >= 97 + t]
    assert torch.equal(got[:, unseen], clean[:, unseen])


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens,tokens,group,most", [([1500, 0, 777], 7, 5, 800000), ([300, 511], 878, 16, 512)])
def test_attend_planned_for_much(dev, kind, dim, lens, tokens, group, most):
    """Plans of many places, that take 32 rows a workgroup, in shares and without; rows that see nothing."""
    print(f"kv4 attend planned {kind} dim={dim} lens={lens} tokens={tokens}", flush=True)
    c, table, ln, _ = filled(dev, lens, 1, dim, 64, 31)
    k, v = (x.cpu().double() for x in c.read(table.to(dev), ln.to(dev), max(lens)))
    there = torch.arange(max(lens))[None] < ln[:, None]
    q = torch.randn(len(lens), tokens, group, dim, generator=torch.Generator().manual_seed(7)).to(TYPES[kind])
    wide = torch.full((len(lens), most // 64), -1, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    w = torch.zeros(len(lens), 1, most, device=dev)
    got = c.attend(q.to(dev), wide.to(dev), ln.to(dev), max_len=most, weights=w)
    check_attend(got, w[:, :, :max(lens)], q, k, v, there, ln, max(lens), kind)
    assert not w[:, :, max(lens):].any()


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [32, 96])
def test_sums_over_pages(dev, kind, dim, page):
    """What tokens received, of several row tiles: small pages, entries that are no page among them."""
    print(f"kv4 sums over pages {kind} dim={dim} page={page}", flush=True)
    lens = [1300, 1025, 33]
    c, table, ln, _ = filled(dev, lens, 1, dim, page, 41)
    table[0, 3], table[1, 0], table[2, 0] = -1, c.pages, -7
    ref = D.Pages(c.k, c.k_scales, c.v, c.v_scales)
    k, v, there = ref.read(table, ln, 1300)
    q = torch.randn(3, 5, 7, dim, generator=torch.Generator().manual_seed(19)).to(TYPES[kind])
    w0 = torch.rand(3, 1, 1301, generator=torch.Generator().manual_seed(20))
    w = w0.to(dev)
    got = c.attend(q.to(dev), table.to(dev), ln.to(dev), max_len=1300, weights=w)
    check_attend(got, w, q, k, v, there, ln, 1300, kind, w0)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_attend_queries_at_the_ends(dev, kind, dim):
    """The types' largest queries over small keys; infinite ones: all scores -infinity (zeros), else NaN."""
    print(f"kv4 attend ends {kind} dim={dim}", flush=True)
    n, top = 45, torch.finfo(TYPES[kind]).max
    small = 2.0 ** -126 if kind != "f16" else 2.0 ** -14
    x = values(n, 1, dim, "f32", 3)
    x[:, 0] = torch.where(x[:, 0] < 0, -1.0, 1.0) * small * 2
    x[:, 0, 5] = small * 2
    table, pages = tables([n], 32, 2)
    c = kv4.Cache4.zeros(pages, 1, 32, dim, dev)
    ln = torch.tensor([n], dtype=torch.int32)
    c.append(x[:, :1].to(dev), x[:, 1:].to(dev), table.to(dev), ln.to(dev), starts([n]).to(dev))
    k, v, there = D.Pages(c.k, c.k_scales, c.v, c.v_scales).read(table, ln, n)
    q = torch.zeros(1, 2, 2, dim)
    q[0, 0, 0, 9], q[0, 0, 1, 40], q[0, 1, 0, 0], q[0, 1, 1, 5] = top, -top, top, top
    q[0, 1, 0, 63] = top / 4
    q = q.to(TYPES[kind])
    check_attend(c.attend(q.to(dev), table.to(dev), ln.to(dev), scale=0.25), None, q, k, v, there, ln, n, kind, scale=0.25)
    odd = torch.zeros(1, 1, 3, dim)
    odd[0, 0, 0, 5], odd[0, 0, 1, 5], odd[0, 0, 2, 9] = -math.inf, math.inf, math.inf  # k of channel 5: all above 0
    w = torch.zeros(1, 1, n, device=dev)
    got = c.attend(odd.to(TYPES[kind]).to(dev)[:, :, :1], table.to(dev), ln.to(dev), max_len=n, weights=w).cpu()
    assert not got.any() and not w.any()
    got = c.attend(odd.to(TYPES[kind]).to(dev), table.to(dev), ln.to(dev)).cpu()
    assert not got[:, :, 0].any() and bool(got[:, :, 1:].isnan().all())


def check_evict(dev, c, table, lens, sums, keep, recent, spare_seed=5):
    B, h = len(lens), c.heads
    ln = torch.tensor(lens, dtype=torch.int32)
    used = set(table[table >= 0].tolist())
    free = [p for p in range(c.pages) if p not in used]
    per = -(-keep // c.page)
    new = torch.tensor(free[:B * per], dtype=torch.int32).reshape(B, per)
    ref = D.Pages(c.k, c.k_scales, c.v, c.v_scales)
    kept, weights, left = c.evict(sums.to(dev), table.to(dev), ln.to(dev), new.to(dev), keep, recent)
    want = torch.full((B, h, keep), -1, dtype=torch.int32)
    wsum = torch.zeros(B, h, keep)
    for b in range(B):
        for j in range(h):
            n = min(lens[b], sums.shape[2])
            at = D.evict(sums[b, j].tolist(), n, keep, recent)
            want[b, j, :len(at)] = torch.tensor(at, dtype=torch.int32)
            wsum[b, j, :len(at)] = sums[b, j][at]
            for to, src in enumerate(at):
                s, d = ref.at(table, b, src), ref.at(new, b, to)
                kc, kb, vc, vb = ref.get(s[0], j, s[1])
                ref.put(d[0], j, d[1], kc, kb, vc, vb)
    assert torch.equal(left.cpu(), torch.tensor([min(n, keep, sums.shape[2]) for n in lens], dtype=torch.int32))
    assert torch.equal(kept.cpu(), want)
    assert torch.equal(weights.cpu().nan_to_num(7.0), wsum.nan_to_num(7.0))
    same_pages(c, ref)


def roomy(dev, lens, h, dim, page, keep, seed):
    table, pages = tables(lens, page, seed)
    pages += len(lens) * -(-keep // page)
    c = kv4.Cache4.zeros(pages, h, page, dim, dev)
    x = values(sum(lens), h, dim, "f32", seed)
    c.append(x[:, :h].to(dev), x[:, h:].to(dev), table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev),
             starts(lens).to(dev))
    return c, table


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens,h,page,keep,recent", [
    ([100, 40, 0, 65], 2, 32, 40, 8), ([200], 1, 64, 64, 64), ([90, 33], 3, 32, 33, 0), ([5], 1, 32, 1, 0),
    ([3000, 1100], 1, 64, 300, 17)])
def test_evict(dev, dim, lens, h, page, keep, recent):
    print(f"kv4 evict dim={dim} lens={lens} heads={h} page={page} keep={keep} recent={recent}", flush=True)
    c, table = roomy(dev, lens, h, dim, page, keep, 7)
    g = torch.Generator().manual_seed(keep)
    sums = torch.exp(2 * torch.randn(len(lens), h, max(lens), generator=g))
    sums = torch.where(sums < 0.5, torch.round(sums * 8) / 8, sums)  # many equal
    check_evict(dev, c, table, lens, sums, keep, recent)


@pytest.mark.parametrize("name", ["equal", "zeros", "signs", "odd", "short"])
def test_evict_orders(dev, name):
    print(f"kv4 evict {name}", flush=True)
    lens, keep, recent = [150, 97], 50, 10
    c, table = roomy(dev, lens, 2, 64, 32, keep, 11)
    g = torch.Generator().manual_seed(1)
    sums = torch.randn(2, 2, 150, generator=g)
    if name == "equal":
        sums = torch.full_like(sums, 0.3)
    elif name == "zeros":
        sums = torch.where(sums > 0, torch.zeros_like(sums), -torch.zeros_like(sums))
    elif name == "odd":
        sums[:, :, 5:9] = math.inf
        sums[:, :, 30:33] = math.nan
        sums[:, :, 60:70] = -math.inf
        sums[:, :, 88:95] = torch.tensor(1e-42)
    elif name == "short":  # fewer weights than tokens: the length is cut
        sums = sums[:, :, :80].contiguous()
    check_evict(dev, c, table, lens, sums, keep, recent)


@pytest.mark.parametrize("name", ["spread", "ties", "equal", "one"])
def test_evict_long_rows(dev, name):
    """Rows of several parts: the list of one digit, one that does not hold them all, ties across the
    parts' borders, rows that keep all or end early."""
    print(f"kv4 evict long {name}", flush=True)
    lens, keep, recent, dim = [30000, 17000, 900, 8193], 2500, 100, 64
    table, pages = tables(lens, 1024, 3)
    pages += 4 * 3
    c = kv4.Cache4.zeros(pages, 1, 1024, dim, dev)
    for t in (c.k, c.v):  # any codes: all are values
        t.copy_(torch.randint(0, 256, t.shape, generator=torch.Generator().manual_seed(2), dtype=torch.uint8))
    g = torch.Generator().manual_seed(6)
    sums = torch.exp(2 * torch.randn(4, 1, 30000, generator=g))
    if name == "ties":
        sums = torch.round(sums * 2) / 2
    elif name == "equal":
        sums = torch.full_like(sums, 0.25)
    elif name == "one":  # all in one digit, none equal
        sums = 1.0 + torch.rand(sums.shape, generator=g) / 8
    if name == "spread":
        keep, recent = 2500, 2500  # none of the old stay
    kept, weights, left = c.evict(sums.to(dev), table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev),
                                  torch.tensor(sorted(set(range(pages)) - set(table.flatten().tolist())),
                                               dtype=torch.int32)[:12].reshape(4, 3).to(dev), keep, recent)
    for b, n in enumerate(lens):
        at = D.evict(sums[b, 0].tolist(), n, keep, recent)
        want = torch.full((keep,), -1, dtype=torch.int32)
        want[:len(at)] = torch.tensor(at, dtype=torch.int32)
        assert torch.equal(kept[b, 0].cpu(), want), b
        assert torch.equal(weights[b, 0, :len(at)].cpu(), sums[b, 0][at]) and not weights[b, 0, len(at):].any()
    assert left.tolist() == [2500, 2500, 900, 2500]


def test_evict_long_rows_moved(dev):
    print("kv4 evict long moved", flush=True)
    c, table = roomy(dev, [17500], 1, 64, 256, 600, 5)
    sums = torch.exp(2 * torch.randn(1, 1, 17500, generator=torch.Generator().manual_seed(8)))
    check_evict(dev, c, table, [17500], sums, 600, 50)


def test_evict_rows_of_odd_length(dev):
    """Rows of weights that start at no multiple of 16 bytes, in one workgroup and in parts."""
    print("kv4 evict odd rows", flush=True)
    c, table = roomy(dev, [1001, 700], 2, 64, 32, 100, 13)
    sums = torch.exp(2 * torch.randn(2, 2, 1001, generator=torch.Generator().manual_seed(2)))
    check_evict(dev, c, table, [1001, 700], sums, 100, 7)
    wide = torch.exp(2 * torch.randn(2, 2, 20003, generator=torch.Generator().manual_seed(3)))
    wide[:, :, :1001] = sums
    c, table = roomy(dev, [1001, 700], 2, 64, 32, 100, 13)
    check_evict(dev, c, table, [1001, 700], wide, 100, 7)


def test_evict_strided_sums(dev):
    print("kv4 evict strided", flush=True)
    c, table = roomy(dev, [70, 80], 2, 64, 32, 32, 3)
    wide = torch.rand(2, 3, 200, generator=torch.Generator().manual_seed(4))
    check_evict(dev, c, table, [70, 80], wide[:, 1:, :80], 32, 4)


def test_graph_and_other_stream(dev):
    """A decode step (append, attend with weights) captured, replayed on new inputs against eager."""
    print("kv4 graph", flush=True)
    lens = [70, 300]
    c, table, ln, _ = filled(dev, lens, 2, 128, 64, 29)
    d = kv4.Cache4(*(t.clone() for t in (c.k, c.k_scales, c.v, c.v_scales)))
    td, ld, cu = table.to(dev), ln.to(dev), starts([1, 1]).to(dev)
    x = torch.zeros(2, 12, 128, device=dev, dtype=torch.bfloat16)
    w, w2 = torch.zeros(2, 2, 320, device=dev), torch.zeros(2, 2, 320, device=dev)

    def step(cache, sums):
        cache.append(x[:, 8:10], x[:, 10:], td, ld, cu)
        return cache.attend(x[:, None, :8], td, ld, max_len=300, weights=sums)

    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        step(c, w)
    st.synchronize()
    step(d, w2)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(c, w)
    for seed in (1, 2, 3):
        x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(seed)).to(dev))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step(d, w2))
        assert torch.equal(w, w2)
        assert torch.equal(c.k, d.k) and torch.equal(c.v_scales, d.v_scales)


def test_refusals(dev):
    c, table, ln, x = filled(dev, [40], 2, 64, 32, 1)
    td, ld = table.to(dev), ln.to(dev)
    q = torch.zeros(1, 1, 4, 64, device=dev)
    with pytest.raises(TypeError):
        c.attend(q.double(), td, ld)
    with pytest.raises(RuntimeError):
        c.attend(q[:, :, :3], td, ld)
    with pytest.raises(RuntimeError):
        c.attend(q[0], td, ld)
    with pytest.raises(TypeError, match="int32"):
        c.attend(q, td.long(), ld)
    with pytest.raises(RuntimeError, match="lens"):
        c.attend(q, td, torch.cat((ld, ld)))
    with pytest.raises(RuntimeError):
        c.attend(q, td, ld, weights=torch.zeros(1, 2, 10, device=dev))
    with pytest.raises(ValueError, match="scale"):
        c.attend(q, td, ld, scale=0.0)
    with pytest.raises(ValueError):
        c.attend(q, td, ld, max_len=-1)
    n = x[:, :2].to(dev)
    with pytest.raises(TypeError):
        c.append(n, n.half(), td, ld, starts([40]).to(dev))
    with pytest.raises(RuntimeError):
        c.append(n[:, :1], n[:, :1], td, ld, starts([40]).to(dev))
    with pytest.raises(RuntimeError, match="cu"):
        c.append(n, n, td, ld, starts([20, 20]).to(dev))
    with pytest.raises(ValueError):
        c.read(td, ld, -1)
    sums = torch.zeros(1, 2, 40, device=dev)
    with pytest.raises(ValueError, match="latest"):
        c.evict(sums, td, ld, td, 8, 9)
    with pytest.raises(ValueError, match="keep"):
        c.evict(sums, td, ld, td, 0)
    with pytest.raises(ValueError, match="hold"):
        c.evict(sums, td, ld, td, 65)
    with pytest.raises(RuntimeError):
        c.evict(sums[:, :1], td, ld, td, 8)
    with pytest.raises(RuntimeError, match="k_scales"):
        kv4.Cache4(c.k, c.k_scales[:, :1].contiguous(), c.v, c.v_scales)
    with pytest.raises(NotImplementedError):
        kv4.Cache4.zeros(1, 1, 48, 64, dev)
    with pytest.raises(RuntimeError, match="contiguous"):
        kv4.Cache4(c.k.transpose(0, 1), c.k_scales, c.v, c.v_scales)
