"""The decoder example evicts straight after a prompt: by what the prompt's last tokens gave.

Tolerance of a sum against float64 over the values that the cache holds: W queries of 2 heads, each weight within
twice its score's f32 error (scores below 30 here: products of three pieces, 192 additions of at most 2^-24 of it,
under 4e-4) and W * 2 additions of at most 2^-24 of the sum: 1e-3 of the sum, and 1e-6 for what is nearly 0."""
import pytest
import torch

from borch_amd.decoder import Decoder, DecoderState
from oracle import decode as D

pytestmark = pytest.mark.gpu


@torch.no_grad()
@pytest.mark.parametrize("window", [1, 16])
def test_evict_after_a_prompt(dev, window):
    print(f"decoder evict after a prompt, window {window}", flush=True)
    torch.manual_seed(3)
    m = Decoder(layers=2, d=128, heads=4, kv_heads=2, dim=64, mlp=256, vocab=97, context=512).to(dev).eval()
    lens, keep, recent = [150, 9, 300], 40, 8
    ids = torch.randint(0, 97, (sum(lens),), generator=torch.Generator().manual_seed(1)).to(dev)
    plain = m.prompt(DecoderState(m, 3, 320), ids, lens)
    state = DecoderState(m, 3, 320)
    assert torch.equal(m.prompt(state, ids, lens, window=window), plain)  # the logits are as without

    # the first layer's sums
    at = torch.cat([torch.arange(n) for n in lens]).to(dev)
    q = m.layers[0].heads_of(m.embed(ids) + m.places(at))[0].double().cpu()
    k = state.caches[0].read(state.table, state.lens, 300)[0].double().cpu()
    start = 0
    for b, n in enumerate(lens):
        rows = q[start:start + n][-window:]
        end = torch.arange(max(0, n - window), n) + 1
        for h in range(2):
            s = torch.stack([r[2 * h:2 * h + 2] @ k[b, h, :n].t().contiguous() for r in rows]) / 8
            s = s.masked_fill(torch.arange(n) >= end[:, None, None], -torch.inf)
            want = torch.softmax(s, -1).sum((0, 1))
            got = state.sums[0][b, h].double().cpu()
            assert bool(((got[:n] - want).abs() <= 1e-3 * want + 1e-6).all()) and not got[n:].any()
        start += n

    sums = [s.cpu().clone() for s in state.sums]
    state.evict(keep, recent)
    assert state.held == [40, 9, 40]
    for before, after in zip(sums, state.sums):
        for b, n in enumerate(lens):
            for h in range(2):
                stay = D.evict(before[b, h].tolist(), n, keep, recent)
                assert torch.equal(after[b, h, :len(stay)].cpu(), before[b, h][stay])
    assert torch.isfinite(m.step(state, plain.argmax(-1))).all()
