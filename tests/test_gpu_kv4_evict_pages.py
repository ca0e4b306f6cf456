"""Evictions from tables with entries that are no page: a kept token of such an entry reads as zeros afterwards as
before, whatever the new pages held."""
import pytest
import torch

from borch_amd import kv4
from oracle import decode as D

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128])
def test_tokens_of_no_page(dev, dim):
    print(f"kv4 evict from no page dim={dim}", flush=True)
    lens, h, page, keep, recent, pages = [150, 97], 2, 32, 70, 20, 16
    c = kv4.Cache4.zeros(pages, h, page, dim, dev)
    g = torch.Generator().manual_seed(dim)
    for t in (c.k, c.v):  # every page holds something, the new ones too
        t.copy_(torch.randint(0, 256, t.shape, generator=g, dtype=torch.uint8))
    for t in (c.k_scales, c.v_scales):
        t.copy_(torch.randint(100, 140, t.shape, generator=g, dtype=torch.uint8))
    table = torch.tensor([[0, -1, 2, 3, pages], [4, 5, 6, -9, -1]], dtype=torch.int32)
    new = torch.tensor([[7, 8, 9], [10, -1, 12]], dtype=torch.int32)
    sums = torch.rand(2, h, 150, generator=g)
    ref = D.Pages(c.k, c.k_scales, c.v, c.v_scales)
    kept, weights, left = c.evict(sums.to(dev), table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), new.to(dev),
                                  keep, recent)
    zero, one = torch.zeros(dim, dtype=torch.long), torch.ones(dim // 32, dtype=torch.long)
    holes = 0
    for b, n in enumerate(lens):
        for j in range(h):
            at = D.evict(sums[b, j].tolist(), n, keep, recent)
            assert kept[b, j].tolist() == at and torch.equal(weights[b, j].cpu(), sums[b, j][at])
            for to, src in enumerate(at):
                s, d = ref.at(table, b, src), ref.at(new, b, to)
                if d is not None:
                    ref.put(d[0], j, d[1], *(ref.get(s[0], j, s[1]) if s else (zero, one, zero, one)))
                holes += s is None
    assert holes > 40 and left.tolist() == [keep, keep]
    for name, a, b in (("k", c.k, ref.k), ("k_scales", c.k_scales, ref.ks), ("v", c.v, ref.v), ("v_scales", c.v_scales, ref.vs)):
        assert torch.equal(a.cpu(), b), name
    k, v = c.read(new.to(dev), left, keep)
    gone = torch.tensor([[[ref.at(table, b, int(i)) is None for i in kept[b, j]] for j in range(h)] for b in range(2)])
    assert not k.cpu()[gone].any() and not v.cpu()[gone].any()
