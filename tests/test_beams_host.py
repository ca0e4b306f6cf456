"""A beam search's selection on the CPU: the library's refusals before any launch, and the oracle against torch."""
import math

import pytest
import torch

from borch_amd import _lib, beams
from oracle import beams as O

ARG, UNSUPPORTED = _lib.BQ_ERR_ARG, _lib.BQ_ERR_UNSUPPORTED


def test_select_refusals():
    lib = _lib.lib()
    need = lib.bq_beam_select_ws_bytes(0, 2, 3, 40)
    assert need > 0

    def call(x=16, type=0, B=2, W=3, V=40, scores=16, done=None, end=-1, out=16, parents=16, tokens=16, ws=16, size=need):
        return lib.bq_beam_select(x, type, B, W, V, V, scores, done, end, out, parents, tokens, None, ws, size, None)

    assert call(type=3) == ARG and call(B=-1) == ARG and call(W=0) == ARG and call(V=0) == ARG
    assert call(W=65) == UNSUPPORTED and "64" in _lib.last_error()
    assert call(V=2 ** 31) == ARG and call(B=2 ** 24) == ARG and call(B=2 ** 22, W=64, V=10 ** 6) == ARG
    assert call(done=16) == ARG and "end token" in _lib.last_error()
    assert call(B=0, x=None) == 0
    for name in ("x", "scores", "out", "parents", "tokens"):
        assert call(**{name: None}) == ARG and "null" in _lib.last_error()
    assert call(ws=None) == ARG and call(size=need - 1) == ARG and call(ws=24) == ARG
    assert lib.bq_beam_select_ws_bytes(0, 0, 3, 40) == 0 == lib.bq_beam_select_ws_bytes(0, 1, 65, 40)


def test_cpu_tensors_are_refused():
    with pytest.raises(_lib.Int8Unavailable):
        beams.beam_select(torch.zeros(4, 9), torch.zeros(2, 2))


def test_oracle_against_torch():
    g = torch.Generator().manual_seed(0)
    x, s = torch.randn(3, 50, generator=g, dtype=torch.float64), torch.tensor([-1.0, -2.0, -0.5], dtype=torch.float64)
    got = O.select(x.tolist(), s.tolist(), [False] * 3, 7)
    key = (torch.log_softmax(x, -1) + s[:, None]).flatten()
    want = key.topk(3)
    assert [c[1] * 50 + c[2] for c in got] == want.indices.tolist()
    assert max(abs(c[0] - k) for c, k in zip(got, want.values.tolist())) < 1e-12
    got = O.select(x.tolist(), s.tolist(), [False, False, True], 7)
    assert got[0] == (-0.5, 2, 7, True)
    dead = O.select([[math.nan] * 4, [-math.inf] * 4], [0.0, 0.0], [False] * 2, 1)
    assert [c[:3] for c in dead] == [(-math.inf, 0, 0), (-math.inf, 0, 1)]
