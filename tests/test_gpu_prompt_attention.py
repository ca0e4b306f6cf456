"""prompt_attention against float64, sequence by sequence (oracle/decode.py).

Tolerance of an output, relative to sum_i p_i |v_i|: the scores' f32 error twice (oracle's
score_error; f32 sums three pieces' six products), (n + 16) 2^-24 for the f32 sums over n tokens and
the quotient, half a step of the 16-bit types for each p (2^-8 bf16, 2^-11 fp16; fp16's least subnormal 2^-24 of
the row's largest), and then half a step of the output itself. Below f32's normal numbers: n weights off
by 2^-126 of the row's largest, and the output by its type's least subnormal."""
import math

import pytest
import torch

from borch_amd import attention as A
from oracle import decode as D

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
LEAST = {"f32": 2.0 ** -149, "bf16": 2.0 ** -133, "f16": 2.0 ** -24}
HALF = {"f32": 0.0, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def data(lens, hq, h, dim, kind, seed, spread=1.0, before=0, after=0):
    g = torch.Generator().manual_seed(seed)
    n = before + sum(lens) + after
    x = (torch.randn(n, hq + 2 * h, dim, generator=g) * spread).to(TYPES[kind])
    cu = [before]
    for m in lens:
        cu.append(cu[-1] + m)
    return x, torch.tensor(cu, dtype=torch.int32)


def expected(x, cu, hq, h, causal, kind, scale=None):
    n, _, dim = x.shape
    scale = 1.0 / math.sqrt(dim) if scale is None else scale
    q, k, v = x[:, :hq].cpu(), x[:, hq:hq + h].cpu(), x[:, hq + h:].cpu()
    want = torch.zeros(n, hq, dim, dtype=torch.float64)
    tol = torch.zeros_like(want)
    for b in range(len(cu) - 1):
        at = slice(int(cu[b]), int(cu[b + 1]))
        m = at.stop - at.start
        seen = torch.ones(m, m, dtype=torch.bool)
        seen = seen.tril() if causal else seen
        for j in range(hq):
            kk, vv = k[at, j * h // hq], v[at, j * h // hq]
            out, _, size = D.softmax_rows(q[at, j], kk, vv, seen, scale)
            rel = D.score_error(q[at, j], kk, scale, 6 if kind == "f32" else 1) + (m + 16) * 2.0 ** -24 + HALF[kind]
            want[at, j] = out
            least = 2.0 ** -24 if kind == "f16" else 2.0 ** -126
            tol[at, j] = size * rel + out.abs() * (HALF[kind] + 2.0 ** -24) + LEAST[kind]
            tol[at, j] += m * least * vv.double().nan_to_num(0, 0, 0).abs().amax(0) if m else 0
    return want, tol


def check(got, want, tol, rows=slice(None)):
    got, want, tol = got.cpu().double()[rows], want[rows], tol[rows]
    fine = torch.isfinite(want)
    assert torch.equal(fine, torch.isfinite(got))
    assert torch.equal(want.isnan(), got.isnan())
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf])
    off = (got - want).abs()
    assert bool((off[fine] <= tol[fine]).all()), f"off by {float((off - tol)[fine].max()):.3g} over the tolerance"


def run(dev, x, cu, hq, h, causal, **more):
    x = x.to(dev)
    return A.prompt_attention(x[:, :hq], x[:, hq:hq + h], x[:, hq + h:], cu.to(dev), causal=causal, **more)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens,hq,h,causal", [
    ([1], 1, 1, True), ([2, 1, 3], 4, 2, True), ([31, 32, 33], 3, 1, True), ([63, 64, 65], 2, 2, False),
    ([127, 128, 129], 8, 8, True), ([0, 5, 0, 0, 200, 0], 6, 2, True), ([300, 1, 17], 5, 5, False), ([257], 16, 2, True),
    ([1] * 70 + [40], 2, 1, True)])
def test_against_float64(dev, kind, dim, lens, hq, h, causal):
    print(f"prompt {kind} dim={dim} lens={lens[:8]} heads={hq}/{h} causal={causal}", flush=True)
    x, cu = data(lens, hq, h, dim, kind, sum(lens) + hq)
    want, tol = expected(x, cu, hq, h, causal, kind)
    check(run(dev, x, cu, hq, h, causal), want, tol)


@pytest.mark.parametrize("kind,dim,spread,scale", [("f32", 64, 6.0, None), ("f32", 128, 0.02, None), ("bf16", 128, 5.0, None),
                                                   ("f16", 64, 4.0, 0.5), ("f32", 64, 1.0, 3.0)])
def test_score_sizes_and_scales(dev, kind, dim, spread, scale):
    print(f"prompt {kind} dim={dim} spread={spread} scale={scale}", flush=True)
    x, cu = data([70, 133], 4, 2, dim, kind, 5, spread)
    want, tol = expected(x, cu, 4, 2, True, kind, scale)
    check(run(dev, x, cu, 4, 2, True, scale=scale), want, tol)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_operands_apart_and_misaligned(dev, kind):
    print(f"prompt operands apart {kind}", flush=True)
    x, cu = data([50, 77], 4, 2, 64, kind, 9)
    base = run(dev, x, cu, 4, 2, True)
    xd = x.to(dev)
    q, k, v = xd[:, :4].contiguous(), xd[:, 4:6].contiguous(), xd[:, 6:].contiguous()
    assert torch.equal(A.prompt_attention(q, k, v, cu.to(dev)), base)
    # heads first, tokens last but one
    t = [y.permute(1, 0, 2).contiguous().permute(1, 0, 2) for y in (q, k, v)]
    assert torch.equal(A.prompt_attention(*t, cu.to(dev)), base)
    # a storage offset that breaks 16-byte alignment, channels apart
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device=dev)[1:].view(q.shape).copy_(q)
    wide = torch.empty(*k.shape, 2, dtype=k.dtype, device=dev)
    wide[..., 0] = k
    assert torch.equal(A.prompt_attention(odd, wide[..., 0], v, cu.to(dev)), base)


def test_rows_of_no_sequence_are_zeros(dev):
    print("prompt rows outside", flush=True)
    x, cu = data([40, 90], 2, 1, 64, "f32", 3, before=130, after=7)
    want, tol = expected(x, cu, 2, 1, True, "f32")
    got = run(dev, x, cu, 2, 1, True)
    check(got, want, tol)
    assert not got[:130].any() and not got[-7:].any()


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("at", [0, 70, 149])
def test_values_that_are_not_finite(dev, kind, dim, what, at):
    """A value that is not finite reaches the queries that see it, as float64 has it, and no other."""
    print(f"prompt {kind} dim={dim} v[{at}]={what}", flush=True)
    x, cu = data([20, 150, 30], 2, 1, dim, kind, 31)
    clean = run(dev, x, cu, 2, 1, True)
    x[20 + at, 3, 5] = what
    x[20 + at, 3, 40] = -what
    want, tol = expected(x, cu, 2, 1, True, kind)
    got = run(dev, x, cu, 2, 1, True)
    unseen = [i for i in range(200) if i < 20 + at or i >= 170]
    assert torch.equal(got[unseen], clean[unseen])
    check(got, want, tol)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("what", [math.nan, math.inf])
def test_keys_that_are_not_finite(dev, kind, what):
    print(f"prompt {kind} k={what}", flush=True)
    x, cu = data([20, 150, 30], 2, 1, 64, kind, 33)
    clean = run(dev, x, cu, 2, 1, True)
    x[20 + 99, 2, 7] = what
    got = run(dev, x, cu, 2, 1, True)
    unseen = [i for i in range(200) if i < 119 or i >= 170]
    assert torch.equal(got[unseen], clean[unseen])
    want, tol = expected(x, cu, 2, 1, True, kind)
    # a score of +inf or NaN leaves NaN; one of -inf takes the token out
    check(got, want, tol)


def many_heads(x, heads):
    """The 2 query heads and 1 key-value head of x with the query heads repeated to `heads`: enough
    workgroups for the form that takes 128 queries each."""
    return torch.cat([x[:, :2]] * (heads // 2) + [x[:, 2:]], 1)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim,causal", [(64, True), (128, True), (128, False)])
def test_many_heads(dev, kind, dim, causal):
    print(f"prompt many heads {kind} dim={dim} causal={causal}", flush=True)
    x, cu = data([20, 385, 1, 130], 2, 1, dim, kind, 41)
    want, tol = expected(x, cu, 2, 1, causal, kind)
    got = run(dev, many_heads(x, 300), cu, 300, 1, causal)
    for j in (0, 148, 298):
        check(got[:, j:j + 2], want, tol)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("what", [None, math.nan, math.inf])
@pytest.mark.parametrize("lens,causal", [([600, 450], True), ([333, 7, 500], False), ([64] * 8, True)])
def test_f32_forms(dev, dim, what, lens, causal):
    """f32 prompts of several tiles, long and short sequences on average: one wave or two a query."""
    print(f"prompt f32 forms dim={dim} lens={lens} causal={causal} {what}", flush=True)
    x, cu = data(lens, 2, 1, dim, "f32", 61)
    if what is not None:
        at = lens[0] // 2 + 5
        clean = run(dev, x, cu, 2, 1, causal)
        x[at, 3, 9] = what
        unseen = [i for i in range(sum(lens)) if i >= lens[0] or (causal and i < at)]
        got = run(dev, x, cu, 2, 1, causal)
        assert torch.equal(got[unseen], clean[unseen])
    want, tol = expected(x, cu, 2, 1, causal, "f32")
    check(run(dev, x, cu, 2, 1, causal), want, tol)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("what,at", [(math.nan, 70), (math.inf, 149), (-math.inf, 3)])
def test_many_heads_not_finite(dev, kind, what, at):
    print(f"prompt many heads {kind} v[{at}]={what}", flush=True)
    x, cu = data([20, 150, 30], 2, 1, 128, kind, 43)
    clean = run(dev, many_heads(x, 600), cu, 600, 1, True)
    x[20 + at, 3, 5] = what
    x[20 + at, 3, 100] = -what
    want, tol = expected(x, cu, 2, 1, True, kind)
    got = run(dev, many_heads(x, 600), cu, 600, 1, True)
    unseen = [i for i in range(200) if i < 20 + at or i >= 170]
    assert torch.equal(got[unseen], clean[unseen])
    check(got[:, 4:6], want, tol)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("which", [2, 3])
@pytest.mark.parametrize("what,at", [(math.nan, 40), (math.inf, 59), (-math.inf, 0)])
def test_short_f32_not_finite(dev, dim, which, what, at):
    """Short f32 prompts, whose tiles are split where they are used."""
    print(f"prompt short dim={dim} operand {which}[{at}]={what}", flush=True)
    x, cu = data([20, 60, 10], 2, 1, dim, "f32", 59)
    clean = run(dev, x, cu, 2, 1, True)
    x[20 + at, which, 5] = what
    want, tol = expected(x, cu, 2, 1, True, "f32")
    got = run(dev, x, cu, 2, 1, True)
    unseen = [i for i in range(90) if i < 20 + at or i >= 80]
    assert torch.equal(got[unseen], clean[unseen])
    check(got, want, tol)


@pytest.mark.parametrize("dim,n", [(64, 192), (64, 193), (128, 96), (128, 97)])
def test_f32_either_side_of_the_split(dev, dim, n):
    print(f"prompt f32 dim={dim} n={n}", flush=True)
    x, cu = data([n - 33, 33], 6, 2, dim, "f32", n)
    for causal in (True, False):
        want, tol = expected(x, cu, 6, 2, causal, "f32")
        check(run(dev, x, cu, 6, 2, causal), want, tol)


@pytest.mark.parametrize("lens", [[40, 30], [400, 333]])
@pytest.mark.parametrize("dim", [64, 128])
def test_f32_small_values(dev, dim, lens):
    """Values that bf16 pieces cannot hold whole; flat scores, so that the tolerance is the sums' alone."""
    print(f"prompt f32 small values dim={dim} lens={lens}", flush=True)
    x, cu = data(lens, 2, 1, dim, "f32", 67)
    x[:, :2] = 0
    x[:, 3] *= 2.0 ** -119
    want, tol = expected(x, cu, 2, 1, True, "f32")
    check(run(dev, x, cu, 2, 1, True), want, tol)


@pytest.mark.parametrize("qs,ks", [(2.0 ** 100, 2.0 ** -98), (2.0 ** -120, 2.0 ** 118), (2.0 ** -140, 2.0 ** 30),
                                   (2.0 ** -10, 2.0 ** 8)])
def test_f32_rows_of_any_size(dev, qs, ks):
    """Rows of q and k near f32's ends, rows of unlike size side by side, channels far below their row's
    largest: the pieces follow each row."""
    print(f"prompt f32 q * {qs} k * {ks}", flush=True)
    x, cu = data([90, 140], 2, 1, 64, "f32", 47)
    x[:, :2, 3] *= 2.0 ** -15
    x[:, 2, 7] *= 2.0 ** -13
    x[:, :2] *= qs * 2.0 ** torch.randint(-3, 1, (230, 1, 1), generator=torch.Generator().manual_seed(1))
    x[:, 2] *= ks * 2.0 ** torch.randint(-3, 1, (230, 1), generator=torch.Generator().manual_seed(2))
    want, tol = expected(x, cu, 2, 1, True, "f32")
    check(run(dev, x, cu, 2, 1, True), want, tol)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_scores_beyond_the_rounded_shift(dev, kind):
    """Scores so large that the product of the maximum and the scale is taken apart from its rounding."""
    print(f"prompt large scores {kind}", flush=True)
    size = 2.0 ** 16 if kind == "bf16" else 2.0 ** 14
    x, cu = data([70, 40], 2, 1, 64, kind, 53)
    x[:, :3] = (x[:, :3].float() * size).clamp(-60000, 60000).to(TYPES[kind]) if kind == "f16" else x[:, :3] * size
    want, tol = expected(x, cu, 2, 1, True, kind)
    check(run(dev, x, cu, 2, 1, True), want, tol)
    check(run(dev, many_heads(x, 600), cu, 600, 1, True)[:, :2], want, tol)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_graph_and_other_stream(dev, kind):
    print(f"prompt graph {kind}", flush=True)
    x, cu = data([40, 210, 7], 4, 2, 128, kind, 13)
    xs, cs = x.to(dev), cu.to(dev)
    args = (xs[:, :4], xs[:, 4:6], xs[:, 6:], cs)
    base = A.prompt_attention(*args).clone()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        y = A.prompt_attention(*args)
    st.synchronize()
    assert torch.equal(y, base)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = A.prompt_attention(*args)
    for seed in (1, 2, 3):
        x2, _ = data([40, 210, 7], 4, 2, 128, kind, seed)
        xs.copy_(x2.to(dev))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, A.prompt_attention(*args))


def test_refusals(dev):
    q = torch.zeros(4, 4, 64, device=dev)
    k = torch.zeros(4, 2, 64, device=dev)
    cu = torch.tensor([0, 4], dtype=torch.int32, device=dev)
    with pytest.raises(TypeError):
        A.prompt_attention(q.double(), k.double(), k.double(), cu)
    with pytest.raises(TypeError):
        A.prompt_attention(q, k.half(), k.half(), cu)
    with pytest.raises(RuntimeError, match="query heads"):
        A.prompt_attention(q, torch.zeros(4, 3, 64, device=dev), torch.zeros(4, 3, 64, device=dev), cu)
    with pytest.raises(RuntimeError, match="shapes"):
        A.prompt_attention(q, k[:3], k[:3], cu)
    with pytest.raises(NotImplementedError):
        A.prompt_attention(q[..., :32], k[..., :32], k[..., :32], cu)
    with pytest.raises(TypeError, match="int32"):
        A.prompt_attention(q, k, k, cu.long())
    with pytest.raises(ValueError, match="scale"):
        A.prompt_attention(q, k, k, cu, scale=-1.0)
    with pytest.raises(RuntimeError):
        A.prompt_attention(q, k.cpu(), k.cpu(), cu)
    assert A.prompt_attention(q[:0], k[:0], k[:0], cu[:1]).shape == (0, 4, 64)
