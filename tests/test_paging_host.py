"""Page tables on the CPU: the library's refusals before any launch, and the oracle's rules by hand."""
import ctypes

import pytest
import torch

from borch_amd import _lib, kv4, paging
from oracle.paging import Tables

ARG, UNSUPPORTED = _lib.BQ_ERR_ARG, _lib.BQ_ERR_UNSUPPORTED


def desc(table=16, lens=16, refs=16, sequences=2, width=3, pages=9, page=32):
    return ctypes.byref(_lib.PagesDesc(table, lens, refs, sequences, width, pages, page))


@pytest.mark.parametrize("name", ["cut", "fork", "grow"])
def test_tables_are_checked(name):
    lib = _lib.lib()

    def call(d, x=16):
        if name == "grow":
            return lib.bq_pages_grow(d, x, 4, 16, 16, 16, 16, 16, None, 0, None)
        return getattr(lib, "bq_pages_" + name)(d, x, None)

    assert call(None) == ARG
    for bad in (dict(sequences=-1), dict(width=-1), dict(pages=-1), dict(page=0), dict(page=1 << 21), dict(width=1 << 20),
                dict(width=1 << 17, page=1 << 15), dict(pages=(1 << 24) + 1), dict(table=None), dict(lens=None),
                dict(refs=None)):
        assert call(desc(**bad)) == ARG, bad
    assert call(desc(sequences=8193)) == UNSUPPORTED and "8192" in _lib.last_error()
    assert call(desc(), None) == ARG and "null" in _lib.last_error()
    if name != "grow":
        assert call(desc(sequences=0, table=None, lens=None), None) == 0


def test_grow_is_checked():
    lib = _lib.lib()

    def call(d=None, more=16, rows=4, cu=16, slots=16, at=16, moves=16, ok=16, ws=None, size=0):
        return lib.bq_pages_grow(d or desc(), more, rows, cu, slots, at, moves, ok, ws, size, None)

    assert call(rows=-1) == ARG and call(rows=2 ** 31) == ARG
    for name in ("more", "cu", "slots", "at", "moves", "ok"):
        assert call(**{name: None}) == ARG, name
    need = lib.bq_pages_grow_ws_bytes(2, 70000)
    assert need > 0 == lib.bq_pages_grow_ws_bytes(2, 65536)
    assert call(desc(pages=70000)) == ARG and "workspace" in _lib.last_error()
    assert call(desc(pages=70000), ws=16, size=need - 1) == ARG and call(desc(pages=70000), ws=18, size=need) == ARG


def test_copies_and_slots_are_checked():
    lib = _lib.lib()
    c = (_lib.Kv4Desc * 2)(_lib.Kv4Desc(16, 16, 16, 16, 2, 1, 32, 64), _lib.Kv4Desc(16, 16, 16, 16, 2, 1, 32, 96))
    at = ctypes.addressof(c)
    assert lib.bq_kv4_copy_pages(at, -1, 16, 1, None) == ARG and lib.bq_kv4_copy_pages(at, 1, 16, -1, None) == ARG
    assert lib.bq_kv4_copy_pages(None, 1, 16, 1, None) == ARG and lib.bq_kv4_copy_pages(at, 1, None, 1, None) == ARG
    assert lib.bq_kv4_copy_pages(at, 2, 16, 1, None) == UNSUPPORTED
    assert lib.bq_kv4_copy_pages(at, 0, None, 1, None) == 0 == lib.bq_kv4_copy_pages(at, 1, None, 0, None)

    def append(k=16, type=0, n=3, strides=(64, 64, 64, 64), slots=16):
        return lib.bq_kv4_append_slots(at, k, 16, type, n, *strides, slots, None)

    assert append(type=3) == ARG and append(n=-1) == ARG and append(slots=None) == ARG and append(k=None) == ARG
    assert append(k=24) == ARG and append(strides=(63, 64, 64, 64)) == ARG and append(n=0, slots=None) == 0


def test_cpu_tensors_are_refused():
    p = paging.Pages.zeros(2, 3, 9, 32, "cpu")
    x = torch.zeros(2, dtype=torch.int32)
    for call in (lambda: p.cut(x), lambda: p.fork(x), lambda: p.grow(x, 4),
                 lambda: paging.copy_pages([kv4.Cache4.zeros(2, 1, 32, 64, "cpu")], torch.zeros(3, 2, dtype=torch.int32))):
        with pytest.raises(_lib.Int8Unavailable):
            call()
    with pytest.raises(TypeError, match="lens"):
        paging.Pages(p.table, p.lens.long(), p.refs, 32)
    with pytest.raises(RuntimeError, match="width"):
        paging.Pages(p.table, p.lens[:1], p.refs, 32)
    with pytest.raises(ValueError, match="page"):
        paging.Pages(p.table, p.lens, p.refs, 0)


def test_oracle_by_hand():
    t = Tables([[-1] * 3 for _ in range(3)], [0, 0, 0], [1, 0, 0, 1, 0, 0, 0, 0], 4)
    cu, slots, at, moves, ok = t.grow([5, 0, 2], 8)
    assert ok and cu == [0, 5, 5, 7] and at == [0, 1, 2, 3, 4, 0, 1, -1]
    assert slots == [4, 5, 6, 7, 8, 16, 17, -1] and t.table == [[1, 2, -1], [-1] * 3, [4, -1, -1]]
    t.fork([0, 0, 2])
    assert t.refs == [1, 2, 2, 1, 1, 0, 0, 0] and t.lens == [5, 5, 2]
    _, slots, _, moves, ok = t.grow([1, 1, 0], 2)
    assert ok and moves == [[-1, 2, -1], [-1, 5, -1], [0, 1, 0]] and slots == [9, 21]
    t.cut([4, 0, 9])
    assert t.table == [[1, -1, -1], [-1] * 3, [4, -1, -1]] and t.refs == [1, 1, 0, 1, 1, 0, 0, 0]
    before = [list(r) for r in t.table]
    assert t.grow([9, 0, 0], 9)[4] == 0 and t.grow([0, 0, 1], 0)[4] == 0 and t.table == before
