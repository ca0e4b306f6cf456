"""A beam that has ended takes no further pages, copies or attention, and gives back what it held."""
import pytest
import torch

import borch_amd as bt
from borch_amd.beams import beam_select
from borch_amd.decoder import PagedState
from test_gpu_decoder import model_of

pytestmark = pytest.mark.gpu


def every_beam(m, state, ids, lens, W, steps, end):
    """The search with all beams lengthened at each step, those that have ended too."""
    B, S = len(lens), len(lens) * W
    counts = torch.zeros(B, W, dtype=torch.int32, device=ids.device)
    counts[:, 0] = torch.tensor(lens, dtype=torch.int32)
    scores = torch.tensor([[0.0] + [-torch.inf] * (W - 1)] * B, device=ids.device)
    done = torch.zeros(B, W, dtype=torch.bool, device=ids.device)
    tokens = torch.zeros(S, 0, dtype=torch.int32, device=ids.device)
    logits = m.read(state, ids, counts.view(-1))
    for _ in range(steps):
        scores, parents, new, done = beam_select(logits, scores, done, end)
        tokens = torch.cat([tokens[parents.view(-1)], new.view(-1, 1)], 1)
        state.pages.fork(parents.view(-1))
        logits = m.read(state, new.view(-1), torch.ones(S, dtype=torch.int32, device=ids.device))
        assert state.ok.item() == 1
    return tokens.view(B, W, steps), scores, done


@torch.no_grad()
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("push", [20.0, 3.0, 1.5])
def test_search_ends(dev, int8, push):
    """An end token that is likely: at once, after some steps, now and then."""
    print(f"decoder search ended int8={int8} push={push}", flush=True)
    m = model_of(dev, 3)
    end, W, steps, lens = 11, 4, 30, [30, 61, 7]
    m.head.bias.data[end] += push
    if int8:
        assert bt.quantize_for_int8(m) == 9
    ids = torch.randint(0, 97, (sum(lens),), generator=torch.Generator().manual_seed(6)).to(dev)
    state = PagedState(m, len(lens) * W, pages=60, width=4, page=32)
    want, scores, done = every_beam(m, PagedState(m, len(lens) * W, pages=90, width=4, page=32), ids, lens, W, steps, end)
    got, mine = m.search(state, ids, lens, W, steps, end)
    assert bool(done.any())
    assert torch.equal(got, want)
    assert float((mine - scores).abs().max()) < 2e-3
    # the tables are those of the last token read: of the beams before the last selection
    before, _ = m.search(PagedState(m, len(lens) * W, pages=60, width=4, page=32), ids, lens, W, steps - 1, end)
    over = (before == end).any(-1).view(-1)
    assert bool(over.any())
    assert not bool(state.pages.lens[over].any()) and bool((state.pages.table[over] == -1).all())
    held = state.pages.table[state.pages.table >= 0].long().bincount(minlength=60)
    assert torch.equal(held, state.pages.refs.long())


@torch.no_grad()
def test_search_ends_early_in_few_pages(dev):
    """All beams have ended after two steps: no page more than those steps take, however many steps follow."""
    print("decoder search in few pages", flush=True)
    m = model_of(dev, 3)
    end, W, steps = 11, 4, 60
    m.head.bias.data[end] += 20.0
    ids = torch.randint(0, 97, (30,), generator=torch.Generator().manual_seed(6)).to(dev)
    got, _ = m.search(PagedState(m, W, pages=4, width=4, page=32), ids, [30], W, steps, end)
    assert bool((got[:, :, 2:] == end).all())
