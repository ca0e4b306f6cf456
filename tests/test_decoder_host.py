"""The decoder example's bookkeeping on the CPU: what it refuses before any launch, and that a refusal
changes nothing."""
import pytest
import torch

from borch_amd.decoder import Decoder, DecoderState


def state_of(sequences=1, tokens=256, context=64, page=32):
    m = Decoder(layers=1, d=32, heads=2, kv_heads=1, dim=64, mlp=32, vocab=11, context=context)
    return m, DecoderState(m, sequences, tokens, page)


def books(s):
    return ([list(p) for p in s.pages], sorted(s.free), list(s.held), list(s.next), s.table.tolist(), s.lens.tolist())


def test_texts_past_the_places():
    m, s = state_of()
    before = books(s)
    with pytest.raises(RuntimeError, match="places for 64"):
        s.begin([200])
    with pytest.raises(RuntimeError, match="places for 64"):
        s.begin([65])
    with pytest.raises(RuntimeError, match="places for 64"):
        m.prompt(s, torch.zeros(65, dtype=torch.long), [65])
    assert books(s) == before
    assert s.begin([62]).tolist() == [0, 62]
    assert s.grow()[1].tolist() == [62] and s.grow()[1].tolist() == [63]  # the last place
    before = books(s)
    with pytest.raises(RuntimeError, match="places for 64"):
        s.grow()
    assert books(s) == before


def test_a_short_cache_does_not_lengthen_the_text():
    """Cached tokens leave, the text goes on: the next place counts, not what is held."""
    _, s = state_of(2)
    s.begin([60, 3])
    s.held = [5, 3]  # as an eviction leaves them
    for _ in range(4):
        s.grow()
    assert s.held == [9, 7] and s.next == [64, 7]
    with pytest.raises(RuntimeError, match="65 tokens"):
        s.grow()


def test_ids_that_do_not_fit():
    """One id for several sequences would have been taken for each; a prompt's would have failed halfway."""
    m, s = state_of(2)
    before = books(s)
    for ids in (torch.zeros(4, dtype=torch.long), torch.zeros(1, dtype=torch.long), torch.zeros(1, 5, dtype=torch.long)):
        with pytest.raises(RuntimeError, match="prompts of 5"):
            m.prompt(s, ids, [2, 3])
    assert books(s) == before
    s.begin([2, 3])
    before = books(s)
    for ids in (torch.zeros(1, dtype=torch.long), torch.zeros(3, dtype=torch.long), torch.zeros(2, 1, dtype=torch.long)):
        with pytest.raises(RuntimeError, match="2 sequences"):
            m.step(s, ids)
    assert books(s) == before


@pytest.mark.parametrize("keep,recent", [(8, 9), (8, -1), (0, 0), (-5, 0)])
def test_refused_evictions_lose_no_page(keep, recent):
    _, s = state_of(2)
    s.begin([60, 3])
    before = books(s)
    with pytest.raises(ValueError, match="evict"):
        s.evict(keep, recent)
    assert books(s) == before


def test_evictions_with_nothing_to_go_by():
    """Sums that are all 0 would have kept the earliest tokens as ties."""
    m, s = state_of(2)
    s.begin([60, 3])
    before = books(s)
    with pytest.raises(RuntimeError, match="received"):
        s.evict(20, 8)
    assert books(s) == before
    s.evict(60, 8)  # nothing leaves
    assert books(s) == before
    with pytest.raises(ValueError, match="window"):
        m.prompt(s, torch.zeros(5, dtype=torch.long), [2, 3], window=-1)
