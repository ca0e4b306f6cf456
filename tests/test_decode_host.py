"""A decoder's attention on the CPU: the library's refusals before any launch, the refusal of CPU
tensors, and the oracle's codes against torch's own casts and closed forms."""
import ctypes
import math

import pytest
import torch

from borch_amd import _lib, attention, kv4
from oracle import decode as D

ARG, UNSUPPORTED = _lib.BQ_ERR_ARG, _lib.BQ_ERR_UNSUPPORTED


def desc(pages=0, heads=2, page=32, dim=64, ptr=None):
    return _lib.Kv4Desc(ptr, ptr, ptr, ptr, pages, heads, page, dim)


def test_prompt_refusals():
    f = _lib.lib().bq_prompt_attention

    def call(type=0, n=4, hq=4, h=2, dim=64, strides=(256, 64, 128, 64, 128, 64), B=1, scale=0.1, ptr=None):
        return f(ptr, ptr, ptr, type, n, hq, h, dim, *strides, ptr, B, 1, scale, ptr, None, 0, None)

    assert call(type=3) == ARG
    assert call(dim=96) == UNSUPPORTED
    assert call(n=-1) == ARG and call(B=-1) == ARG and call(h=0) == ARG
    assert call(hq=3) == ARG and "query heads" in _lib.last_error()
    for s in (0.0, -1.0, math.nan, math.inf):
        assert call(scale=s) == ARG
    assert call() == ARG and "null" in _lib.last_error()
    assert call(n=0) == 0
    assert call(ptr=8) == ARG and "aligned" in _lib.last_error()
    assert call(ptr=16, strides=(255, 64, 128, 64, 128, 64)) == ARG
    assert call(ptr=16, n=4000) == ARG and "workspace" in _lib.last_error()
    ws = _lib.lib().bq_prompt_attention_ws_bytes
    assert ws(0, 4000, 2, 64) > 0 == ws(1, 4000, 2, 64) == ws(0, 4, 2, 64)
    assert call(ptr=16, type=1, strides=(256, 64, 2 ** 23 + 8, 64, 128, 64)) == UNSUPPORTED
    assert call(ptr=16, n=2 ** 31 - 10000, hq=4096, h=2) == ARG and "large" in _lib.last_error()


def test_cache_refusals():
    lib = _lib.lib()
    for d, rc in ((desc(dim=96), UNSUPPORTED), (desc(page=48), UNSUPPORTED), (desc(page=0), UNSUPPORTED),
                  (desc(pages=-1), ARG), (desc(heads=0), ARG), (desc(pages=1), ARG), (desc(pages=1, ptr=8), ARG)):
        assert lib.bq_kv4_read(ctypes.byref(d), None, 0, 0, None, 4, None, None, None) == rc
    d = desc()
    r = ctypes.byref(d)
    assert lib.bq_kv4_read(None, None, 0, 0, None, 4, None, None, None) == ARG
    assert lib.bq_kv4_read(r, None, 1, 1, None, 4, None, None, None) == ARG  # no table
    assert lib.bq_kv4_read(r, 16, 1, 1, None, -1, None, None, None) == ARG
    assert lib.bq_kv4_read(r, 16, 1, 2 ** 31, None, 4, None, None, None) == ARG
    assert lib.bq_kv4_read(r, 16, 0, 1, None, 4, None, None, None) == 0
    assert lib.bq_kv4_append(r, None, None, 5, 1, 1, 1, 1, 1, 16, 1, 1, None, None, None) == ARG
    assert lib.bq_kv4_append(r, None, None, 0, -1, 64, 64, 64, 64, 16, 1, 1, None, None, None) == ARG
    full = desc(pages=2, ptr=16)
    assert lib.bq_kv4_append(ctypes.byref(full), 16, 16, 1, 1, 4, 64, 64, 64, 16, 1, 1, 16, 16, None) == ARG
    assert "aligned" in _lib.last_error()


def test_attend_and_evict_refusals():
    lib = _lib.lib()
    full = desc(pages=2, ptr=16)
    r = ctypes.byref(full)

    def attend(type=0, tokens=1, hq=4, max_len=64, scale=0.1, ws=None, ws_bytes=0, q=16, weights=None):
        return lib.bq_kv4_attend(r, q, type, tokens, hq, 256, 256, 64, 16, 1, 2, 16, max_len, scale, 16, weights, 64, 64,
                                 ws, ws_bytes, None)

    assert attend(type=7) == ARG and attend(tokens=-1) == ARG and attend(max_len=-1) == ARG
    assert attend(hq=3) == ARG and attend(scale=0.0) == ARG and attend(scale=math.nan) == ARG
    assert attend(tokens=0) == 0
    assert attend(q=None) == ARG and attend(q=24) == ARG
    assert attend(weights=16) == ARG and "workspace" in _lib.last_error()
    assert attend(tokens=2 ** 21) == ARG
    need = lib.bq_kv4_attend_ws_bytes(1, 2, 2, 64, 100000, 0)
    assert need > 0 and attend(max_len=100000, ws=16, ws_bytes=need - 1) == ARG
    assert lib.bq_kv4_attend_ws_bytes(0, 2, 2, 64, 100, 1) == 0

    def evict(keep=4, recent=0, most=8, new_width=1, ptr=None):
        return lib.bq_kv4_evict(r, ptr, 16, 8, most, 16, 1, 2, ptr, 16, new_width, keep, recent, ptr, ptr, ptr, None, 0, None)

    assert evict(keep=0) == ARG and evict(recent=5) == ARG and evict(recent=-1) == ARG
    assert evict(keep=33) == ARG and "hold" in _lib.last_error()
    assert evict(most=-1) == ARG and evict() == ARG
    assert lib.bq_kv4_evict_ws_bytes(1, 2, 16384, 8) == 0 < lib.bq_kv4_evict_ws_bytes(1, 2, 16385, 8)
    assert evict(most=20000, ptr=16) == ARG and "workspace" in _lib.last_error()


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 2, 64)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(_lib.Int8Unavailable):
        attention.prompt_attention(x, x, x, cu)
    c = kv4.Cache4.zeros(2, 2, 32, 64, "cpu")
    t, n = torch.zeros(1, 1, dtype=torch.int32), torch.tensor([4], dtype=torch.int32)
    for call in (lambda: c.append(x, x, t, n, cu), lambda: c.read(t, n, 4), lambda: c.attend(x[None, :1], t, n),
                 lambda: c.evict(torch.zeros(1, 2, 4), t, n, t, 2)):
        with pytest.raises(_lib.Int8Unavailable):
            call()
    with pytest.raises(NotImplementedError):
        kv4.Cache4.zeros(2, 2, 48, 64, "cpu")
    with pytest.raises(TypeError):
        kv4.Cache4(c.k.float(), c.k_scales, c.v, c.v_scales)


def test_oracle_codes():
    """Each code of each scale comes back as itself; ties go to the even code; the pages return what
    was put."""
    for e in (-126, -20, 0, 100):
        x = torch.tensor([v * s for v in D.VALUES for s in (1.0, -1.0)] * 2, dtype=torch.float64) * 2.0 ** e
        code, byte = D.quantize(x)
        assert int(byte[0]) == e + 127
        assert torch.equal(D.value(code, byte), x)
    x = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0] + [0.0] * 24)
    assert D.quantize(x)[0][:8].tolist() == [0, 2, 2, 4, 4, 6, 6, 7]
    assert int(D.quantize(torch.full((32,), math.nan))[1][0]) == 255
    c = kv4.Cache4.zeros(3, 2, 32, 128, "cpu")
    p = D.Pages(c.k, c.k_scales, c.v, c.v_scales)
    k, v = torch.randn(9, 2, 128), torch.randn(9, 2, 128)
    table, lens = torch.tensor([[2, 0]], dtype=torch.int32), torch.tensor([36], dtype=torch.int32)
    p.append(k, v, table, lens, torch.tensor([0, 9]))
    rk, rv, there = p.read(table, lens, 36)
    assert torch.equal(rk[0, :, 27:], D.value(*D.quantize(k)).transpose(0, 1)) and bool(there.all())
    assert torch.equal(rv[0, :, 27:], D.value(*D.quantize(v)).transpose(0, 1))
    assert D.evict([3.0, 1.0, 3.0, math.nan, 0.0], 5, 3, 1) == [0, 3, 4]


def test_oracle_attention_against_torch():
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(7, 64, dtype=torch.float64, generator=g) for _ in range(3))
    out, p, _ = D.softmax_rows(q, k, v, torch.ones(7, 7, dtype=torch.bool).tril(), 0.125)
    want = torch.nn.functional.scaled_dot_product_attention(q[None], k[None], v[None], is_causal=True)[0]
    assert torch.allclose(out, want, atol=1e-12) and torch.allclose(p.sum(1), torch.ones(7, dtype=torch.float64))
    none = D.softmax_rows(q, k, v, torch.zeros(7, 7, dtype=torch.bool), 0.125)[0]
    assert not none.any()
