"""prompt_attention in f32 where the tolerance does not hide a lost bit: scores and values that are exact.

A score is one channel's product, a whole number of sixteenths that two fp16 pieces hold; few keys carry
weight, so that the sums are short. Tolerance of an output, relative to sum_i p_i |v_i|, for differences of scores
d <= 4 from the row's largest and h keys within it (all others are 200 below: a weight of 0): the exponent's
argument within 3 2^-24 of itself (log2(e) as a constant, its product with the scale, the product), 3 * 4 2^-24 in p
and once more in its sum, the exponential's 2^-23 likewise, h additions in each of the sums, and 16 2^-24 for the
six products of pieces (what the three others would add is below 2^-24), the joined parts and the quotient:
(24 + 4 + 2 h + 16) 2^-24."""
import pytest
import torch

from borch_amd import attention as A
from oracle import decode as D

pytestmark = pytest.mark.gpu

HEAVY = [(3, 0.0), (17, -1.0), (36, -1.0), (61, -0.5), (64, -4.0), (100, -0.25), (130, -2.0), (190, -1.5), (239, 0.0),
         (299, -3.0)]


@pytest.mark.parametrize("dim,n,heads", [(64, 300, 2), (128, 300, 2), (64, 300, 600), (128, 300, 600), (64, 150, 2), (128, 96, 2)])
@pytest.mark.parametrize("top", [0.0, 1000.0, 2.0 ** 14, -(2.0 ** 14), 2.0 ** 17])
@pytest.mark.parametrize("causal", [True, False])
def test_f32_weights_of_large_scores(dev, dim, n, heads, top, causal):
    """Every form: one wave or two a query (their halves joined), tiles split where they are used. The weights
    are of both halves of a tile and of several tiles, whose maxima differ."""
    print(f"prompt f32 exact dim={dim} n={n} heads={heads} top={top} causal={causal}", flush=True)
    g = torch.Generator().manual_seed(dim + n)
    v = torch.randn(n, 1, dim, generator=g)
    score = torch.full((n,), top - 200.0)
    heavy = [(i, d) for i, d in HEAVY if i < n]
    for i, d in heavy:
        score[i] = top + d
    q, k = torch.zeros(n, heads, dim), torch.zeros(n, 1, dim)
    q[:, :, 5], k[:, 0, 5] = 1.0, score * 8.0
    cu = torch.tensor([0, n], dtype=torch.int32)
    got = A.prompt_attention(q.to(dev), k.to(dev), v.to(dev), cu.to(dev), causal=causal, scale=0.125).cpu().double()
    seen = torch.ones(n, n, dtype=torch.bool)
    want, _, size = D.softmax_rows(q[:, 0], k[:, 0], v[:, 0], seen.tril() if causal else seen, 0.125)
    rows = slice(heavy[0][0], n)  # before: rows of flat scores, whose sums are long
    tol = (44 + 2 * len(heavy)) * 2.0 ** -24
    for j in sorted({0, 1, heads - 1}):
        off = ((got[:, j] - want).abs() / size)[rows if causal else slice(None)].max()
        assert float(off) <= tol, f"off by {float(off):.3g}, tolerance {tol:.3g}"


@pytest.mark.parametrize("dim,n", [(64, 192), (128, 96)])
def test_tiles_split_where_they_are_used(dev, dim, n):
    """Several tiles in one buffer, filled again by all waves: every head and every run the same bits."""
    print(f"prompt f32 tiles in one buffer dim={dim}", flush=True)
    g = torch.Generator().manual_seed(n)
    q, k, v = (torch.randn(n, 1, dim, generator=g).to(dev) for _ in range(3))
    cu = torch.tensor([0, n], dtype=torch.int32, device=dev)
    base = A.prompt_attention(q, k, v, cu, causal=False)
    for _ in range(5):
        got = A.prompt_attention(q.expand(n, 512, dim), k, v, cu, causal=False)
        assert torch.equal(got, base.expand(n, 512, dim))


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("at", [0, 63, 64, 200])
def test_scores_that_decide_a_row(dev, kind, dim, at):
    """A key whose scores are NaN or +infinity leaves NaN in every channel of the rows that see it, though keys
    of -infinity and values that are not finite follow; the same key with scores of -infinity leaves the rest."""
    print(f"prompt deciding scores {kind} dim={dim} at={at}", flush=True)
    g = torch.Generator().manual_seed(dim)
    n = 260
    q, k, v = (torch.randn(n, h, dim, generator=g) for h in (2, 1, 1))
    q[:, 0, 3], q[:, 1, 3] = q[:, 0, 3].abs() + 0.1, -q[:, 1, 3].abs() - 0.1
    k[at, 0, 3] = torch.inf  # head 0: +infinity, head 1: -infinity
    k[at + 5, 0, 3] = -torch.inf if at else torch.inf
    v[at + 7, 0, 9] = torch.inf
    q, k, v = q.to(kind), k.to(kind), v.to(kind)
    cu = torch.tensor([0, n], dtype=torch.int32)
    got = A.prompt_attention(q.to(dev), k.to(dev), v.to(dev), cu.to(dev)).cpu()
    seen = torch.ones(n, n, dtype=torch.bool).tril()
    for j in range(2):
        want = D.softmax_rows(q[:, j], k[:, 0], v[:, 0], seen, dim ** -0.5)[0]
        assert torch.equal(got[:, j].isnan(), want.isnan()) and torch.equal(got[:, j].isposinf(), want.isposinf())
        assert bool(got[at:, 0].isnan().all())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n,heads", [(90, 1), (300, 1), (300, 264)])
@pytest.mark.parametrize("above", [2.0 ** 10, 2.0 ** 14, 2.0 ** 20, 2.0 ** 30, 2.0 ** 45])
@pytest.mark.parametrize("which", ["q", "k"])
def test_f32_channel_above_its_row(dev, dim, n, heads, above, which):
    """A channel far above the others of its rows, over rows that are as small there (or 0). A score (times log2 e)
    is within 3 2^-22 of sum |q||k| and 3 dim 2^-24 of it for the products' sums, and within 2^-17 or 2^-22 of the
    row's largest for what small channels lose; twice the largest of them in the output, (n + 44) 2^-24 as above."""
    print(f"prompt f32 channel above dim={dim} n={n} heads={heads} above={above} of {which}", flush=True)
    g = torch.Generator().manual_seed(dim + n)
    q, k, v = (torch.randn(n, 1, dim, generator=g) for _ in range(3))
    high, low = (q, k) if which == "q" else (k, q)
    high[..., 5] *= above
    low[..., 5] /= above
    low[::2, :, 5] = 0
    cu = torch.tensor([0, n], dtype=torch.int32)
    got = A.prompt_attention(q.expand(n, heads, dim).to(dev), k.to(dev), v.to(dev), cu.to(dev), causal=False, scale=0.125)
    got = got[:, heads - 1].cpu().double()
    want, _, size = D.softmax_rows(q[:, 0], k[:, 0], v[:, 0], torch.ones(n, n, dtype=torch.bool), 0.125)
    top = (q[:, 0].double() @ k[:, 0].double().t().contiguous()).amax(1, keepdim=True).abs() * 0.125
    each = (q[:, 0].double().abs() @ k[:, 0].double().abs().t().contiguous()).amax(1, keepdim=True) * 0.125
    off = each * (3 * 2.0 ** -22 + 3 * dim * 2.0 ** -24) + torch.clamp_min(top * 2.0 ** -22, 2.0 ** -17)
    tol = size * (2 * off + (n + 44) * 2.0 ** -24)
    assert bool(((got - want).abs() <= tol).all()), float(((got - want).abs() / tol).max())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n,heads", [(90, 1), (300, 1), (300, 264)])
def test_f32_channel_above_that_is_not_seen(dev, dim, n, heads):
    """Keys and queries with such a channel change no bit of the rows before them, nor of the next sequence."""
    print(f"prompt f32 channel above unseen dim={dim} n={n} heads={heads}", flush=True)
    g = torch.Generator().manual_seed(dim + n)
    q, k, v = (torch.randn(n, h, dim, generator=g) for h in (heads, 1, 1))
    cu = torch.tensor([0, n - 20, n], dtype=torch.int32, device=dev)
    clean = A.prompt_attention(q.to(dev), k.to(dev), v.to(dev), cu)
    for at in (37, 66):
        k[at, 0, 5] = 2.0 ** 40
        got = A.prompt_attention(q.to(dev), k.to(dev), v.to(dev), cu)
        assert torch.equal(got[:37], clean[:37]) and torch.equal(got[n - 20:], clean[n - 20:])
        assert not torch.equal(got[at], clean[at])
    q[40] *= 2.0 ** 60
    got = A.prompt_attention(q.to(dev), k.to(dev), v.to(dev), cu)
    assert torch.equal(got[:37], clean[:37]) and torch.equal(got[n - 20:], clean[n - 20:])
