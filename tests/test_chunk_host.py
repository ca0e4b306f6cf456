"""Attention of chunks over the 4-bit cache on the CPU: the library's refusals before any launch."""
import ctypes
import math

import pytest
import torch

from borch_amd import _lib, kv4

ARG, UNSUPPORTED = _lib.BQ_ERR_ARG, _lib.BQ_ERR_UNSUPPORTED


def desc(pages=2, heads=2, page=32, dim=64, ptr=16):
    return _lib.Kv4Desc(ptr, ptr, ptr, ptr, pages, heads, page, dim)


def test_chunk_refusals():
    lib = _lib.lib()
    full = desc()

    def call(d=full, q=16, type=0, n=3, hq=4, strides=(256, 64), B=1, width=2, lens=16, cu=16, max_len=64, scale=0.1,
             out=16, ws=None, ws_bytes=0, table=16):
        return lib.bq_kv4_attend_chunk(ctypes.byref(d) if d else None, q, type, n, hq, *strides, table, B, width, lens, cu,
                                       max_len, scale, out, ws, ws_bytes, None)

    assert call(d=None) == ARG and call(d=desc(dim=96)) == UNSUPPORTED and call(d=desc(page=48)) == UNSUPPORTED
    assert call(type=3) == ARG and call(type=-1) == ARG
    assert call(n=-1) == ARG and call(hq=0) == ARG and call(max_len=-1) == ARG and call(B=-1) == ARG
    assert call(n=2 ** 31) == ARG and call(max_len=2 ** 31) == ARG and call(hq=70000) == ARG
    assert call(hq=3) == ARG and "query heads" in _lib.last_error()
    for s in (0.0, -1.0, math.nan, math.inf):
        assert call(scale=s) == ARG
    assert call(n=0, q=None, cu=None, lens=None, out=None) == 0
    for name in ("q", "cu", "lens", "out"):
        assert call(**{name: None}) == ARG and "null" in _lib.last_error()
    assert call(table=None) == ARG
    assert call(q=24) == ARG and call(out=8) == ARG and "aligned" in _lib.last_error()
    assert call(strides=(255, 64)) == ARG and call(type=1, strides=(256, 68)) == ARG
    assert call(n=2 ** 30, hq=64) == ARG and "large" in _lib.last_error()
    tokens = full.pages * full.page
    need = lib.bq_kv4_attend_chunk_ws_bytes(0, 3, 1, 4, 2, 64, 100000, tokens)
    assert need > 0 and call(max_len=100000, width=4000) == ARG and "workspace" in _lib.last_error()
    assert call(max_len=100000, width=4000, ws=16, ws_bytes=need - 1) == ARG
    assert call(max_len=100000, width=4000, ws=24, ws_bytes=need) == ARG
    assert lib.bq_kv4_attend_chunk_ws_bytes(0, 3, 1, 4, 2, 64, 100, tokens) == 0 == lib.bq_kv4_attend_chunk_ws_bytes(0, 0, 1, 4, 2, 64, 10 ** 6, tokens)
    assert lib.bq_kv4_attend_chunk_ws_bytes(0, 3, 1, 1, 2, 64, 10 ** 6, tokens) == 0


def test_chunk_on_the_cpu():
    c = kv4.Cache4.zeros(2, 2, 32, 64, "cpu")
    t, n = torch.zeros(1, 1, dtype=torch.int32), torch.tensor([4], dtype=torch.int32)
    with pytest.raises(_lib.Int8Unavailable):
        c.attend_chunk(torch.zeros(4, 2, 64), t, n, torch.tensor([0, 4], dtype=torch.int32))
