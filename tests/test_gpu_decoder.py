"""The decoder example: prompts, steps over the 4-bit cache and an eviction, against the same network
with float64 attention over the values that the caches hold.

Tolerance: both sides run the same f32 Linears on inputs that differ by the attention's f32 error. Each
of the L layers' attention outputs is within (scores' error + 3 n + 64) 2^-24 of its scale (test_gpu_kv4;
under 2e-5 at these sizes), and each of about 5 L f32 products of K <= 512 terms may change its rounding by
(K + 2) 2^-24 = 3.1e-5 of its scale: 2 layers stay within 10 * 5e-5 of the largest logit."""
import pytest
import torch

import borch_amd as bt
from borch_amd.decoder import Decoder, DecoderState

pytestmark = pytest.mark.gpu


def model_of(dev, seed=0, **more):
    torch.manual_seed(seed)
    return Decoder(layers=2, d=128, heads=4, kv_heads=2, dim=64, mlp=256, vocab=97, context=512, **more).to(dev).eval()


def plain_step(m, state, ids, at):
    """step() with attention in float64 over read()."""
    x = m.embed(ids) + m.places(at)
    for layer, cache in zip(m.layers, state.caches):
        q, _, _ = layer.heads_of(x)
        k, v = (t.double() for t in cache.read(state.table, state.lens, state.longest))
        B, hq, dim = q.shape
        h = k.shape[1]
        s = (k[:, :, None] * q.double().reshape(B, h, hq // h, 1, dim)).sum(-1) / dim ** 0.5
        seen = torch.arange(state.longest, device=q.device) < state.lens[:, None]
        p = torch.softmax(s.masked_fill(~seen[:, None, None], -torch.inf), -1)
        o = (p[..., None] * v[:, :, None]).sum(-2).reshape(B, hq, dim).float()
        x = layer.close(x, o)
    return m.head(m.ln(x))


@torch.no_grad()
def test_decoder(dev):
    print("decoder", flush=True)
    m = model_of(dev)
    lens = [150, 3, 64]
    state = DecoderState(m, 3, 256)
    ids = torch.randint(0, 97, (sum(lens),), generator=torch.Generator().manual_seed(1)).to(dev)
    logits = m.prompt(state, ids, lens)
    # each prompt alone gives the same
    at = 0
    for i, n in enumerate(lens):
        one = DecoderState(m, 1, 256)
        assert torch.allclose(m.prompt(one, ids[at:at + n], [n]), logits[i:i + 1], rtol=0, atol=5e-4 * float(logits.abs().max()))
        at += n
    for t in range(8):
        if t == 4:
            state.evict(1000)  # more than any holds: nothing leaves
            assert state.held == [154, 7, 68]
            state.evict(40, 8)
            assert state.held == [40, 7, 40] and state.lens.tolist() == state.held
            assert all(float(s[:, :, 40:].abs().max()) == 0 for s in state.sums)
        nxt = logits.argmax(-1)
        places = torch.tensor(state.next, device=dev)
        logits = m.step(state, nxt)
        want = plain_step(m, state, nxt, places)
        off = float((logits - want).abs().max())
        assert off <= 5e-4 * float(want.abs().max()), (t, off)
    # what all tokens received is what all queries gave: one a step, layer and head, times the group
    total = [float(s[1].sum()) for s in state.sums]  # never cut: 8 steps, 2 heads, 2 queries each
    assert all(abs(x - 8 * 4) < 1e-3 for x in total)


@torch.no_grad()
def test_decoder_int8(dev):
    """The same with every Linear in int8: the layers convert, and the path runs through them."""
    print("decoder int8", flush=True)
    m = model_of(dev, 2)
    assert bt.quantize_for_int8(m) == 9
    state = DecoderState(m, 2, 128)
    ids = torch.arange(50, device=dev) % 97
    logits = m.prompt(state, ids, [20, 30])
    for _ in range(3):
        logits = m.step(state, logits.argmax(-1))
    assert torch.isfinite(logits).all() and state.held == [23, 33]
    with pytest.raises(RuntimeError, match="already"):
        m.prompt(state, ids, [20, 30])
    with pytest.raises(RuntimeError, match="128"):
        DecoderState(m, 1, 128).begin([129])
