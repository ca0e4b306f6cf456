"""Page tables of a paged cache, kept on the GPU (``bq_pages_*``, ``include/bq.h``): which pages hold which
sequence's tokens, and the places of new ones, without a look from the host in between, so that a step that
lengthens, forks or ends sequences can be captured into a graph.

    pages = Pages.zeros(sequences=8, width=64, pages=1024, page=64, device="cuda")
    got = pages.grow(lengths, rows)       # places for `rows` new tokens, packed
    cache.append(k, v, slots=got.slots)   # of each layer
    cache.attend_chunk(q, pages.table, pages.lens, got.cu)
    pages.fork(parents)                   # a beam search: sequences go on from others'
    copy_pages(caches, pages.grow(ones, 8).moves)
    pages.cut(lengths)                    # rejected drafts, or 0: sequences that have ended

A page may be named by several sequences; none of them writes to it while they do. A new token's page that is
shared and partly filled is replaced when its sequence grows, and ``copy_pages`` moves what it holds."""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Sequence

import torch

from ._lib import Kv4Desc, PagesDesc, check, lib, require_device
from .attention import ints, on
from .int8 import _stream
from .kv4 import Cache4

__all__ = ["Grown", "Pages", "copy_pages"]


class Grown(NamedTuple):
    """What ``Pages.grow`` gives, on the device: ``cu`` int32 ``[sequences + 1]``, the first row of each
    sequence's new tokens and the end; ``slots`` int64 and ``at`` int32 ``[rows]``, each token's place in the
    cache (page times page size plus place) and in its sequence, -1 past the last; ``moves`` int32 ``[3,
    sequences]``, for ``copy_pages``; ``ok`` int32 ``[1]``, 0 where there was no room."""
    cu: torch.Tensor
    slots: torch.Tensor
    at: torch.Tensor
    moves: torch.Tensor
    ok: torch.Tensor


class Pages:
    """``table [sequences, width]`` names each sequence's pages in order (-1 past the last), ``lens
    [sequences]`` its tokens, ``refs [pages]`` how many entries name a page (0: it is free); int32, contiguous,
    on one device, changed in place. ``page``: tokens a page. ``Pages.zeros`` makes empty ones."""

    def __init__(self, table: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor, page: int):
        if table.dim() != 2 or lens.shape != table.shape[:1] or refs.dim() != 1:
            raise RuntimeError(f"Pages: table {tuple(table.shape)}, lens {tuple(lens.shape)}, refs {tuple(refs.shape)} are "
                               "[sequences, width], [sequences] and [pages]")
        for name, t in (("table", table), ("lens", lens), ("refs", refs)):
            if t.dtype is not torch.int32:
                raise TypeError(f"Pages: {name} is int32, got {t.dtype}")
            if not t.is_contiguous():
                raise RuntimeError(f"Pages: {name} has to be contiguous")
            if t.device != table.device:
                raise RuntimeError(f"Pages: {name} is on {t.device}, table on {table.device}")
        if page < 1:
            raise ValueError(f"Pages: {page} tokens a page")
        self.table, self.lens, self.refs, self.page = table, lens, refs, page
        self.sequences, self.width = table.shape
        self.pages = refs.shape[0]
        self.device, self._index = table.device, table.get_device()
        self._desc = PagesDesc(table.data_ptr(), lens.data_ptr(), refs.data_ptr(), self.sequences, self.width, self.pages, page)
        self._ref = ctypes.addressof(self._desc)

    @classmethod
    def zeros(cls, sequences: int, width: int, pages: int, page: int, device) -> "Pages":
        """``sequences`` empty sequences of up to ``width`` pages each, ``pages`` pages, all free."""
        i32 = dict(dtype=torch.int32, device=device)
        return cls(torch.full((sequences, width), -1, **i32), torch.zeros(sequences, **i32), torch.zeros(pages, **i32), page)

    def cut(self, to: torch.Tensor) -> None:
        """Sequences back to ``to`` int32 ``[sequences]`` tokens where they have more (0 and below: they end);
        pages that no sequence needs any more are free."""
        require_device(self.device)
        to = ints(to, self.lens.shape, "to", self._index)
        with on(self._index):
            check(lib().bq_pages_cut(self._ref, to.data_ptr(), _stream(to)))

    def fork(self, parents: torch.Tensor) -> None:
        """Every sequence ``s`` becomes what sequence ``parents[s]`` was (int32 ``[sequences]``; empty where
        that is none): the pages are shared, nothing is copied."""
        require_device(self.device)
        parents = ints(parents, self.lens.shape, "parents", self._index)
        with on(self._index):
            check(lib().bq_pages_fork(self._ref, parents.data_ptr(), _stream(parents)))

    def grow(self, more: torch.Tensor, rows: int) -> Grown:
        """Places for ``more`` int32 ``[sequences]`` new tokens each, packed one sequence after another into
        ``rows`` rows: free pages in ascending order, sequence after sequence. All find room or nothing changes
        (``ok`` 0, ``cu`` zeros): ``more`` and the lengths 0 or above, the pages within ``width`` and free,
        the tokens within ``rows``. A last page that is partly filled and shared is replaced by a free one,
        save for the lowest of the sequences that share it where all that name it grow; ``moves`` says what
        ``copy_pages`` has to move before the new tokens are written."""
        require_device(self.device)
        S = self.sequences
        more = ints(more, self.lens.shape, "more", self._index)
        if rows < 0:
            raise ValueError(f"grow: {rows} rows")
        # one allocation for four of them: 1.5 us less
        cu, at, moves, ok = torch.empty(4 * S + 2 + rows, dtype=torch.int32, device=self.device).split_with_sizes(
            (S + 1, rows, 3 * S, 1))
        got = Grown(cu, torch.empty(rows, dtype=torch.int64, device=self.device), at, moves.view(3, S), ok)
        need = lib().bq_pages_grow_ws_bytes(S, self.pages)
        ws = torch.empty(need, dtype=torch.uint8, device=self.device) if need else None
        with on(self._index):
            check(lib().bq_pages_grow(self._ref, more.data_ptr(), rows, got.cu.data_ptr(), got.slots.data_ptr(),
                                      got.at.data_ptr(), got.moves.data_ptr(), got.ok.data_ptr(),
                                      ws.data_ptr() if need else None, need, _stream(more)))
        return got


def copy_pages(caches: Sequence[Cache4], moves: torch.Tensor) -> None:
    """The ``moves`` of ``Pages.grow`` in every one of ``caches`` (a model's layers, on one device): of each the
    first tokens of a page, 32 at a time, to another page."""
    caches = list(caches)
    if not caches:
        return
    index = caches[0]._index
    require_device(caches[0].device)
    if moves.dim() != 2 or moves.shape[0] != 3:
        raise RuntimeError(f"copy_pages: moves {tuple(moves.shape)} are [3, sequences]")
    moves = ints(moves, moves.shape, "moves", index)
    if any(c._index != index for c in caches):
        raise RuntimeError(f"copy_pages: caches on {sorted({str(c.device) for c in caches})}")
    descs = (Kv4Desc * len(caches))(*(c._desc for c in caches))
    with on(index):
        check(lib().bq_kv4_copy_pages(ctypes.addressof(descs), len(caches), moves.data_ptr(), moves.shape[1], _stream(moves)))
