"""The decoder with its page tables on the GPU: texts read in pieces, against the same network with float64
attention over the values that the caches hold; a beam search against hypotheses read each from the start.

Tolerance, as for the decoder's steps (test_gpu_decoder): both sides run the same f32 Linears on inputs that differ
by the attention's f32 error, and 2 layers stay within 10 * 5e-5 of the largest logit. Where the caches are filled
by other pieces, a value that lies at a border of the 4-bit rounding may fall to the other side: the search's two
sides read the prompt in one piece and its tokens one by one, so that their Linears see rows of the same values."""
import pytest
import torch

import borch_amd as bt
from borch_amd.beams import beam_select
from borch_amd.decoder import PagedState
from oracle import beams as O
from test_gpu_decoder import model_of

pytestmark = pytest.mark.gpu


def plain_read(m, state, ids, seq, at):
    """read() of rows of sequences `seq` at places `at`, with attention in float64 over what the caches hold."""
    x = m.embed(ids) + m.places(at)
    most = state.pages.width * state.pages.page
    for layer, cache in zip(m.layers, state.caches):
        q, _, _ = layer.heads_of(x)
        k, v = (t.double()[seq] for t in cache.read(state.pages.table, state.pages.lens, most))
        n, hq, dim = q.shape
        h = k.shape[1]
        s = (k[:, :, None] * q.double().reshape(n, h, hq // h, 1, dim)).sum(-1) / dim ** 0.5
        seen = torch.arange(most, device=q.device) <= at[:, None]
        p = torch.softmax(s.masked_fill(~seen[:, None, None], -torch.inf), -1)
        x = layer.close(x, (p[..., None] * v[:, :, None]).sum(-2).reshape(n, hq, dim).float())
    return m.head(m.ln(x))


@torch.no_grad()
def test_read_in_pieces(dev):
    """Prompts, pieces and single tokens in one call; a sequence that waits; one that ends and makes room; a call
    that finds none."""
    print("decoder read", flush=True)
    m = model_of(dev)
    state = PagedState(m, 3, pages=14, width=5, page=32)
    g = torch.Generator().manual_seed(1)
    lens = [0, 0, 0]
    for step, counts in enumerate(([40, 0, 7], [1, 64, 30], [33, 1, 1], [0, 50, 1], [1, 1, 1])):
        rows = sum(counts)
        ids = torch.randint(0, 97, (rows + 2,), generator=g).to(dev)
        if step == 3:
            state.pages.cut(torch.tensor([0, 999, 20], dtype=torch.int32, device=dev))
            lens = [0, lens[1], 20]
        logits = m.read(state, ids, torch.tensor(counts, dtype=torch.int32, device=dev))
        seq = torch.tensor([s for s in range(3) for _ in range(counts[s])], device=dev)
        at = torch.tensor([lens[s] + i for s in range(3) for i in range(counts[s])], device=dev)
        lens = [n + c for n, c in zip(lens, counts)]
        assert state.pages.lens.tolist() == lens and state.ok.item() == 1
        want = plain_read(m, state, ids[:rows], seq, at)
        end = 0
        for s in range(3):
            end += counts[s]
            if counts[s]:
                off = float((logits[s] - want[end - 1]).abs().max())
                assert off <= 5e-4 * float(want.abs().max()), (step, s, off)
    before = state.pages.table.clone()
    m.read(state, torch.zeros(200, dtype=torch.long, device=dev), torch.tensor([0, 0, 141], dtype=torch.int32, device=dev))
    assert state.ok.item() == 0 and torch.equal(state.pages.table, before) and state.pages.lens.tolist() == lens


@torch.no_grad()
@pytest.mark.parametrize("int8", [False, True])
def test_search(dev, int8):
    print(f"decoder search int8={int8}", flush=True)
    m = model_of(dev, 3)
    if int8:
        assert bt.quantize_for_int8(m) == 9
    lens, W, steps, end = [37, 64, 5], 4, 6, 11
    ids = torch.randint(0, 97, (sum(lens),), generator=torch.Generator().manual_seed(4)).to(dev)
    state = PagedState(m, len(lens) * W, pages=60, width=4, page=32)
    tokens, scores = m.search(state, ids, lens, W, steps, end)
    at = 0
    for b, n in enumerate(lens):
        prompt = ids[at:at + n]
        at += n

        def logits_of(hypothesis):
            one = PagedState(m, 1, pages=4, width=4, page=32)
            y = m.read(one, prompt, torch.tensor([n], dtype=torch.int32, device=dev))
            for t in hypothesis:
                y = m.read(one, torch.tensor([t], device=dev), torch.ones(1, dtype=torch.int32, device=dev))
            return y[0].double().tolist()

        found, done, total = [[]] * W, [False] * W, [0.0] + [-torch.inf] * (W - 1)
        for _ in range(steps):
            rows = [[0.0] * 97 if d or s == -torch.inf else logits_of(h) for h, d, s in zip(found, done, total)]
            best = O.select(rows, total, done, end)
            found, total, done = [found[c[1]] + [c[2]] for c in best], [c[0] for c in best], [c[3] for c in best]
        assert tokens[b].tolist() == found, b
        assert all(abs(x - y) < 2e-3 for x, y in zip(scores[b].tolist(), total))


@torch.no_grad()
def test_search_refusals(dev):
    m = model_of(dev)
    with pytest.raises(RuntimeError, match="places for 512"):
        PagedState(m, 2, pages=30, width=17, page=32)
    state = PagedState(m, 4, pages=3, width=2, page=32)
    ids = torch.zeros(60, dtype=torch.long, device=dev)
    counts = torch.tensor([3, 0, 0, 0], dtype=torch.int32, device=dev)
    for bad in (ids[:0], ids.cpu(), ids.view(2, 30)):
        with pytest.raises(RuntimeError, match="read: ids"):
            m.read(state, bad, counts)
    with pytest.raises(RuntimeError, match="end token 97"):
        m.search(state, ids, [60], 4, 2, end=97)
    with pytest.raises(RuntimeError, match="65 beams"):
        m.search(PagedState(m, 65, pages=3, width=2, page=32), ids, [60], 65, 2)
    assert not bool(state.pages.lens.any())
    with pytest.raises(RuntimeError, match="4 sequences"):
        m.search(state, ids, [60], 3, 2)
    with pytest.raises(RuntimeError, match="prompts of 50"):
        m.search(state, ids, [50], 4, 2)
    with pytest.raises(RuntimeError, match="64 a sequence"):
        m.search(state, ids, [60], 4, 6)
    with pytest.raises(RuntimeError, match="3 pages"):
        m.search(state, ids, [60], 4, 4)


@torch.no_grad()
def test_search_captured(dev):
    """A step of the search captured: fork, growth, copies, the model over the caches and the selection, replayed with
    the host's own work between, against the same search call by call."""
    print("decoder search captured", flush=True)
    m = model_of(dev, 3)
    lens, W, steps, end = [37, 63], 3, 6, 11
    S = len(lens) * W
    ids = torch.randint(0, 97, (sum(lens),), generator=torch.Generator().manual_seed(8)).to(dev)
    want, scores = m.search(PagedState(m, S, pages=40, width=4, page=32), ids, lens, W, steps, end)
    state = PagedState(m, S, pages=40, width=4, page=32)
    counts = torch.tensor([37, 0, 0, 63, 0, 0], dtype=torch.int32, device=dev)
    logits = m.read(state, ids, counts)
    have = torch.tensor([[0.0, -torch.inf, -torch.inf]] * 2, device=dev)
    done, one = torch.zeros(2, W, dtype=torch.bool, device=dev), torch.ones(S, dtype=torch.int32, device=dev)
    tokens = torch.zeros(S, steps + 1, dtype=torch.int32, device=dev)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = beam_select(logits, have, done, end)
        parents, new = got.parents.view(-1), got.tokens.view(-1)
        tokens.copy_(torch.cat([tokens[parents][:, 1:], new[:, None]], 1))
        state.pages.fork(parents)
        next_logits = m.read(state, new, one)
        for to, x in ((logits, next_logits), (have, got.scores), (done, got.done)):
            to.copy_(x)
    for step in range(steps):
        graph.replay()
        assert state.ok.item() == 1
        assert state.pages.lens.tolist() == [38 + step] * W + [64 + step] * W
    assert torch.equal(tokens[:, 1:].view(2, W, steps), want)
    assert float((have - scores).abs().max()) < 2e-3
