"""Searches in a state that other calls have used: as in a fresh one."""
import pytest
import torch

from borch_amd.decoder import PagedState
from test_gpu_decoder import model_of

pytestmark = pytest.mark.gpu


@torch.no_grad()
def test_search_in_a_used_state(dev):
    """Twice in a row, after a call that found no room, after a text that was read: the same beams and scores as in a
    fresh state each time, whose pages hold exactly what they need."""
    print("decoder search in a used state", flush=True)
    m = model_of(dev, 3)
    W, steps, end = 4, 5, 11
    g = torch.Generator().manual_seed(9)
    prompts = [torch.randint(0, 97, (n,), generator=g).to(dev) for n in (33, 40, 70)]
    state = PagedState(m, W, pages=12, width=4, page=32)
    m.read(state, prompts[2], torch.tensor([0, 70, 0, 0], dtype=torch.int32, device=dev))
    for ids in (prompts[0], prompts[0], prompts[1]):
        want, scores = m.search(PagedState(m, W, pages=12, width=4, page=32), ids, [len(ids)], W, steps, end)
        got, mine = m.search(state, ids, [len(ids)], W, steps, end)
        assert torch.equal(got, want) and torch.equal(mine, scores)
    few = PagedState(m, W, pages=4, width=4, page=32)
    with pytest.raises(RuntimeError, match="4 pages"):
        m.search(few, prompts[2], [70], W, steps, end)
    want, scores = m.search(PagedState(m, W, pages=4, width=4, page=32), prompts[0][:20], [20], W, steps, end)
    got, mine = m.search(few, prompts[0][:20], [20], W, steps, end)
    assert torch.equal(got, want) and torch.equal(mine, scores)
