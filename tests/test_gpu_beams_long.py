"""A beam search's selection over inputs whose parts are as long as they get, or many: the loops that short
vocabularies do not reach. Tolerances as in test_gpu_beams; the oracle takes some of many requests."""
import math

import pytest
import torch

from borch_amd import _lib, beams
from oracle import beams as O
from test_gpu_beams import TYPES

pytestmark = pytest.mark.gpu


def same(got, b, want, W):
    assert got.parents[b].tolist() == [b * W + c[1] for c in want], b
    assert got.tokens[b].tolist() == [c[2] for c in want], b
    assert got.done[b].tolist() == [c[3] for c in want], b
    for mine, (key, w, v, _) in zip(got.scores[b].tolist(), want):
        assert mine == key or abs(mine - key) <= abs(key) * 2.0 ** -24 + 2.0 ** -149 + 2.0 ** -39, (b, mine, key)


def parts_of(kind, B, W, V):
    return _lib.lib().bq_beam_select_ws_bytes(list(TYPES).index(kind), B, W, V) // ((16 + 8 * W) * B * W)


@pytest.mark.parametrize("V", [2 ** 31 - 8193, 2 ** 31 - 20011])
def test_select_longest(dev, V):
    """As many tokens as a call takes, the best of them first, last and in between."""
    print(f"beams longest {V}", flush=True)
    logits = torch.full((1, V), -math.inf, dtype=torch.float16, device=dev)
    places = torch.cat([torch.arange(40), torch.arange(V // 2, V // 2 + 40), torch.arange(V - 50000, V, 331),
                        torch.arange(V - 40, V)]).unique()
    x = (torch.randn(len(places), generator=torch.Generator().manual_seed(3)) * 3).half()
    x[-1], x[0], x[60] = 9.0, 8.5, 8.0
    logits[0, places.to(dev)] = x.to(dev)
    got = beams.beam_select(logits, torch.tensor([[-1.5]], device=dev), None, V - 1)
    (key, _, at, _), = O.select([x.double().tolist()], [-1.5], [False], -1)
    assert places[at] == V - 1
    same(got, 0, [(key, 0, V - 1, True)], 1)


@pytest.mark.parametrize("kind,B,W,V,pitch,parts,pieces", [
    # of each: how many parts a beam has, and 16-byte pieces a lane takes of the first of them (16 at most)
    ("f32", 64, 8, 33000, 33001, 4, 9), ("bf16", 64, 8, 33000, 33000, 4, 5), ("f32", 256, 8, 16361, 16363, 1, 16),
    ("bf16", 1024, 2, 32737, 32739, 1, 16), ("f16", 1024, 2, 32740, 32740, 1, 16), ("f32", 512, 4, 20001, 20001, 2, 10),
    ("bf16", 128, 16, 40000, 40001, 2, 10), ("f32", 1, 1, 140001, 140001, 69, 2), ("bf16", 1, 2, 300007, 300010, 147, 1),
    ("f16", 1, 1, 2000003, 2000003, 977, 1), ("f32", 2, 1, 3000001, 3000001, 1024, 3)])
def test_select_long_parts(dev, kind, B, W, V, pitch, parts, pieces):
    print(f"beams long parts {kind} {B} x {W} of {V}", flush=True)
    assert parts_of(kind, B, W, V) == parts
    size = 4 if kind == "f32" else 2
    assert (-(-V // parts) * size // 16 + 255) // 256 == pieces
    g = torch.Generator(device=dev).manual_seed(V)
    wide = (torch.randn(B * W, pitch, generator=g, device=dev) * 3).to(TYPES[kind])
    logits = wide[:, pitch - V:]
    scores = -5 - torch.rand(B, W, generator=g, device=dev) * 3
    done = torch.rand(B, W, generator=g, device=dev) < 0.1
    got = beams.beam_select(logits, scores, done, 17)
    for b in {0, B // 3, B - 1}:
        x = logits[b * W:(b + 1) * W].cpu().double().tolist()
        same(got, b, O.select(x, scores[b].cpu().double().tolist(), done[b].tolist(), 17), W)
    # the others' parents, tokens and scores by 64-bit sorting, where no two of the best are close
    key = torch.log_softmax(logits.double(), -1) + scores.double().view(-1, 1)
    key = torch.where(done.view(-1, 1), torch.where(torch.arange(V, device=dev) == 17, scores.double().view(-1, 1), -math.inf), key)
    best, at = key.view(B, W * V).topk(W + 1)
    clear = ((best[:, :-1] - best[:, 1:]) > 1e-9).all(1)
    assert kind != "f32" or float(clear.double().mean()) > 0.9
    w, v = at[:, :W] // V, at[:, :W] % V
    assert torch.equal(got.tokens[clear].long(), v[clear])
    assert torch.equal((got.parents - torch.arange(B, device=dev)[:, None] * W)[clear].long(), w[clear])
    assert bool(((got.scores.double() - best[:, :W]).abs() <= best[:, :W].abs() * 2.0 ** -24 + 2.0 ** -39).all())


def test_select_long_parts_odd_values(dev):
    """NaN, infinities and logits beyond f64's exponentials at the far end of long parts, where the best are too."""
    print("beams long parts, odd values", flush=True)
    B, W, V = 1024, 2, 16365
    g = torch.Generator(device=dev).manual_seed(5)
    logits = torch.randn(B * W, V, generator=g, device=dev)
    scores = -torch.rand(B, W, generator=g, device=dev)
    logits[0, V - 3], logits[2, V - 1], logits[5, V - 2] = math.nan, math.inf, 3000.0
    logits[6], logits[8, 100:] = -math.inf, -math.inf
    logits[10, V - 70:] += 12.0
    assert parts_of("f32", B, W, V) == 1
    got = beams.beam_select(logits, scores)
    for b in range(7):
        same(got, b, O.select(logits[b * W:(b + 1) * W].cpu().double().tolist(), scores[b].cpu().double().tolist(), [False] * W, -1), W)
