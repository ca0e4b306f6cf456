"""A beam search's selection against the oracle's: parents, tokens and ends exactly, scores to f32's rounding.

Tolerance of the scores: each f64 exponential is within 1.1e-12 < 2^-39 of itself, so the sum is and its logarithm within
2^-39, and an f32 score is that rounded
once, half a step of 2^-24 (the oracle's and the other f64 errors are far below). The inputs
of the exact comparisons have no two candidates of different beams within 1e-9 of one another, other than equals."""
import math

import pytest
import torch

from borch_amd import beams
from oracle import beams as O

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def check(dev, logits, scores, done=None, end=-1):
    got = beams.beam_select(logits.to(dev), scores.to(dev), None if done is None else done.to(dev), end)
    B, W = scores.shape
    x = logits.double().tolist()
    for b in range(B):
        was = [False] * W if done is None else done[b].tolist()
        want = O.select(x[b * W:(b + 1) * W], scores[b].double().tolist(), was, end)
        assert got.parents[b].tolist() == [b * W + c[1] for c in want], b
        assert got.tokens[b].tolist() == [c[2] for c in want], b
        assert got.done[b].tolist() == [c[3] for c in want], b
        for mine, (key, w, v, _) in zip(got.scores[b].tolist(), want):
            assert mine == key or abs(mine - key) <= abs(key) * 2.0 ** -24 + 2.0 ** -149 + 2.0 ** -39, (b, mine, key)
    return got


def random_case(B, W, V, kind, seed):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(B * W, V, generator=g) * 3).to(TYPES[kind])
    scores = -5 - torch.rand(B, W, generator=g) * 3
    return logits, scores


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,W,V", [(1, 1, 1), (1, 1, 50), (2, 4, 3), (1, 3, 64), (3, 5, 257), (2, 8, 1025), (1, 16, 3001),
                                   (5, 2, 10007), (1, 64, 70), (1, 33, 2500), (130, 3, 90)])
def test_select(dev, kind, B, W, V):
    print(f"beams {kind} {B} x {W} of {V}", flush=True)
    check(dev, *random_case(B, W, V, kind, V))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_select_ended(dev, kind):
    """Beams that have ended keep their score and one candidate; ending is told; all ended stay in order."""
    print(f"beams ended {kind}", flush=True)
    B, W, V = 4, 5, 700
    logits, scores = random_case(B, W, V, kind, 2)
    logits[:, 13] += 9
    scores -= torch.tensor([0.0, 2.0, 1.0, 9.0, 3.0])
    done = torch.tensor([[0, 1, 0, 0, 1], [1, 1, 1, 1, 1], [0, 0, 0, 0, 0], [1, 0, 1, 1, 1]], dtype=torch.bool)
    got = check(dev, logits, scores, done, 13)
    assert bool(got.done[1].all()) and got.tokens[1].tolist() == [13] * W
    assert torch.equal(got.scores[1].cpu(), scores[1].sort(descending=True).values)
    check(dev, logits, scores, None, 13)
    check(dev, logits, scores)


def test_select_first_step(dev):
    """All beams alike, all but the first at -infinity; a vocabulary smaller than the beams."""
    print("beams first step", flush=True)
    logits, scores = random_case(3, 4, 900, "f32", 7)
    scores[:, 0], scores[:, 1:] = 0, -math.inf
    got = check(dev, logits, scores)
    assert got.parents.tolist() == [[4 * b] * 4 for b in range(3)]
    logits, scores = random_case(1, 6, 2, "f32", 8)
    scores[:, 0], scores[:, 1:] = 0, -math.inf
    got = check(dev, logits, scores)  # two candidates, then the lowest of the others
    assert got.parents.tolist() == [[0, 0, 1, 1, 2, 2]] and got.tokens.tolist()[0][2:] == [0, 1, 0, 1]


@pytest.mark.parametrize("V", [40, 5000])
def test_select_ties(dev, V):
    """Equal logits by the lower token, equal beams by the lower beam, -0 and 0 alike; few distinct values over
    the whole vocabulary."""
    print(f"beams ties {V}", flush=True)
    g = torch.Generator().manual_seed(V)
    row = torch.randint(0, 3, (V,), generator=g).float()
    check(dev, row.repeat(6, 1), torch.full((2, 3), -1.5))
    check(dev, torch.zeros(8, V), torch.zeros(1, 8))
    signed = torch.where(torch.arange(V) % 2 == 0, -0.0, 0.0).repeat(4, 1)
    assert check(dev, signed, torch.zeros(1, 4)).tokens.tolist() == [[0, 1, 2, 3]]
    up = torch.arange(V, dtype=torch.float32).repeat(4, 1) * 2.0 ** -10  # every one beats the last
    check(dev, up, torch.tensor([[0.0, -0.25, -3.0, -0.125]]))


def test_select_masks_and_odd_values(dev):
    """Banned tokens, beams with nothing left, NaN and infinities among logits and scores."""
    print("beams odd values", flush=True)
    B, W, V = 6, 4, 3000
    logits, scores = random_case(B, W, V, "f32", 3)
    logits[:, ::3] = -math.inf
    logits[0:4] = -math.inf                       # nothing anywhere: the lowest
    logits[4, :], logits[5, :V - 1] = -math.inf, -math.inf  # one beam with none, one with one token
    logits[9, 2999] = math.nan
    logits[10, 0], logits[11, 5] = math.inf, -math.inf
    scores[3, 1], scores[3, 2] = math.nan, math.inf
    scores[4] = -math.inf
    logits[20:24, 2:] = -math.inf
    got = check(dev, logits, scores)
    assert got.parents[0].tolist() == [0] * 4 and got.tokens[0].tolist() == [0, 1, 2, 3]
    assert bool((got.scores[0] == -math.inf).all()) and not bool(got.scores.isnan().any())
    done = torch.zeros(B, W, dtype=torch.bool)
    done[0, 2], done[3, 1], done[4, 3], done[2, 2] = True, True, True, True
    check(dev, logits, scores, done, 7)
    big = torch.full((2, 300), 3.0e38)
    big[0, 5], big[1, 7] = 3.4e38, -3.4e38
    check(dev, big, torch.tensor([[0.0, -1.0]]))
    check(dev, big * 1e-40, torch.tensor([[0.0, -1.0]]))


def test_select_near_beams(dev):
    """Candidates of two beams that f32 scores cannot tell apart come out in their order."""
    print("beams near", flush=True)
    V = 4000
    g = torch.Generator().manual_seed(5)
    row = torch.randn(V, generator=g)
    logits = torch.stack((row, row))
    logits[0, 17], logits[1, 17] = 6.0, 6.0
    for t in (1e-5, -1e-5):  # changes a sum of about 6600 by 1e-5, the score near -20 by 1.5e-9
        x = logits.double()
        x[1, 50] = math.log(math.exp(float(x[0, 50])) + t)
        x = x.float()
        got = check(dev, x, torch.tensor([[-20.0, -20.0]]))
        sums = torch.logsumexp(x.double(), 1)
        assert got.parents[0, 0].item() == int(sums.argmin())
        assert got.scores[0, 0] == got.scores[0, 1]


def test_select_strides_streams_graph(dev):
    print("beams strides, streams, graph", flush=True)
    logits, scores = random_case(3, 4, 777, "bf16", 9)
    want = beams.beam_select(logits.to(dev), scores.to(dev))
    wide = torch.full((12, 1001), 50.0, dtype=torch.bfloat16)
    wide[:, 3:780] = logits
    same = lambda a, b: all(torch.equal(x, y) for x, y in zip(a, b))  # noqa: E731
    assert same(beams.beam_select(wide.to(dev)[:, 3:780], scores.to(dev)), want)
    assert same(beams.beam_select(logits.t().contiguous().to(dev).t(), scores.to(dev)), want)
    assert same(beams.beam_select(logits.to(dev), scores.t().contiguous().to(dev).t()), want)
    one = logits[:1].to(dev).expand(12, 777)
    assert same(beams.beam_select(one, scores.to(dev)), beams.beam_select(one.contiguous(), scores.to(dev)))
    x, s = logits.to(dev), scores.to(dev)
    done = torch.zeros(3, 4, dtype=torch.bool, device=dev)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        got = beams.beam_select(x, s, done, 5)
    side.synchronize()
    assert same(got[:3], want[:3])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = beams.beam_select(x, s, done, 5)
    for i in range(4):
        x.copy_(random_case(3, 4, 777, "bf16", 20 + i)[0])
        done[1, i] = True
        graph.replay()
        eager = beams.beam_select(x, s, done, 5)
        torch.cuda.synchronize()
        assert same(out, eager)


def test_select_refusals(dev):
    logits, scores = (t.to(dev) for t in random_case(2, 3, 40, "f32", 1))
    done = torch.zeros(2, 3, dtype=torch.bool, device=dev)
    assert all(t.shape == (0, 3) for t in beams.beam_select(logits[:0], scores[:0]))
    for bad in ((logits[:5], scores), (logits[:, :0], scores), (logits, scores.view(-1)), (logits[:0], scores[:, :0])):
        with pytest.raises(RuntimeError, match="beam_select"):
            beams.beam_select(*bad)
    with pytest.raises(TypeError, match="float64"):
        beams.beam_select(logits.double(), scores)
    with pytest.raises(TypeError, match="scores"):
        beams.beam_select(logits, scores.half())
    with pytest.raises(TypeError, match="scores"):
        beams.beam_select(logits, scores.cpu())
    with pytest.raises(TypeError, match="done"):
        beams.beam_select(logits, scores, done.int(), 3)
    with pytest.raises(TypeError, match="done"):
        beams.beam_select(logits, scores, done[:1], 3)
    for end in (-1, 40):
        with pytest.raises(ValueError, match="end token"):
            beams.beam_select(logits, scores, done, end)
    with pytest.raises(NotImplementedError, match="64"):
        beams.beam_select(torch.zeros(65, 9, device=dev), torch.zeros(1, 65, device=dev))
    with pytest.raises(RuntimeError, match="gradient"):
        beams.beam_select(logits.requires_grad_(), scores)


def test_select_parts_of_nothing_but(dev):
    """A part of the vocabulary that is all NaN, all -infinity, or all beyond what f64's exponentials hold, beside
    ordinary ones; logits that start and end anywhere in 16 bytes."""
    print("beams parts", flush=True)
    V = 9001
    logits, scores = random_case(1, 6, V, "f32", 11)
    logits[0, 4096:] = math.nan
    logits[1, 4096:] = -math.inf
    logits[2, :6000] = -5000.0
    logits[3, 5000:] += 2000.0
    logits[4] = -3.0e4 + logits[4]
    check(dev, logits, scores)
    for off in range(9):
        for kind in ("f32", "bf16"):
            wide = random_case(1, 3, 2100, kind, off)[0]
            x = wide.to(dev)[:, off:off + 2050 + off]
            got = beams.beam_select(x, torch.zeros(1, 3, device=dev))
            want = O.select(wide[:, off:off + 2050 + off].double().tolist(), [0.0] * 3, [False] * 3, -1)
            assert got.tokens.tolist() == [[c[2] for c in want]] and got.parents.tolist() == [[c[1] for c in want]], (off, kind)
