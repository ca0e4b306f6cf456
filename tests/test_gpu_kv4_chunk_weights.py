"""The weights of attention of chunks over the 4-bit cache, in all types, to more than the outputs' own bits.

The tolerance is test_gpu_kv4_chunk's, but for bf16 2^-16 of sum_i p_i |v_i| as for f16: p as two bf16 pieces, the
second rounded, 2^-8 of what is at most 2^-8 of p. Sequences of a few tokens, so that the sums' (3 n + 64) 2^-24
stays below it, and values of both signs, so that many outputs are far smaller than their terms."""
import pytest
import torch

import test_gpu_kv4_chunk as C
from test_gpu_kv4 import filled, starts

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens,group", [([8, 5, 12], 2), ([9] * 40, 16), ([33, 7] * 30, 12)])  # narrow tiles; wide ones; both
def test_chunk_weights(dev, monkeypatch, kind, dim, lens, group):
    print(f"kv4 chunk weights {kind} dim={dim} {len(lens)} sequences group={group}", flush=True)
    monkeypatch.setitem(C.WEIGHT, "bf16", 2.0 ** -16)
    c, table, ln, _ = filled(dev, lens, 1, dim, 32, 51)
    cu = starts(lens)
    q = C.queries(sum(lens), group, dim, kind, 52)
    k, v, there = C.held(c, table, ln, max(lens), dev)
    got = c.attend_chunk(q.to(dev), table.to(dev), ln.to(dev), cu.to(dev))
    C.check(got, q, k, v, there, ln, cu, max(lens), kind)
