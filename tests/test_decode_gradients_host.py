"""Operands that require a gradient are refused by the decoder's attention, which keeps no graph; under no_grad
they are taken as any other (here: refused for lying on the CPU)."""
import pytest
import torch

from borch_amd import _lib, attention, kv4


def test_operands_that_require_a_gradient():
    x = torch.zeros(4, 2, 64)
    r = torch.zeros(4, 2, 64, requires_grad=True)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    c = kv4.Cache4.zeros(2, 2, 32, 64, "cpu")
    t, n = torch.zeros(1, 1, dtype=torch.int32), torch.tensor([4], dtype=torch.int32)
    w, s = torch.zeros(1, 2, 32, requires_grad=True), torch.zeros(1, 2, 4, requires_grad=True)
    calls = [lambda: attention.prompt_attention(r, x, x, cu), lambda: attention.prompt_attention(x, r, x, cu),
             lambda: attention.prompt_attention(x, x, r * 2, cu), lambda: c.append(r, x, t, n, cu),
             lambda: c.append(x, r, t, n, cu), lambda: c.attend(r[None, :1], t, n),
             lambda: c.attend(x[None, :1], t, n, weights=w), lambda: c.evict(s, t, n, t, 2)]
    for call in calls:
        with pytest.raises(RuntimeError, match="gradient"):
            call()
        with torch.no_grad(), pytest.raises(_lib.Int8Unavailable, match="cpu"):
            call()
