"""A decoder's key-value cache held in 4 bits (``bq_kv4_*``, ``include/bq.h``): new tokens quantized
into its pages, attention of the newest tokens or of chunks of a prompt over it, eviction of the tokens that
received least.

A value is one of +-{0, 1/2, 1, 3/2, 2, 3, 4, 6} times the power of two that 32 neighbouring channels
of a token share: 4.25 bits a channel, 136 bytes for the keys and values of a token and a head of
128, where f32 takes 1024. The arrays' layouts are described at ``bq_kv4_cache``."""
from __future__ import annotations

import ctypes
import functools

import torch

from ._lib import Kv4Desc, check, lib, require_device
from .attention import ints, no_graph, on, rows, type_of
from .int8 import _stream

__all__ = ["Cache4"]


@functools.lru_cache(maxsize=1024)
def _attend_ws_bytes(*sizes) -> int:
    return int(lib().bq_kv4_attend_ws_bytes(*sizes))


@functools.lru_cache(maxsize=1024)
def _chunk_ws_bytes(*sizes) -> int:
    return int(lib().bq_kv4_attend_chunk_ws_bytes(*sizes))


class Cache4:
    """The pages of a 4-bit cache: ``k``, ``k_scales``, ``v``, ``v_scales`` uint8 with ``[pages,
    heads]`` first (``Cache4.zeros`` makes them). The caller keeps, on the device and in int32,
    ``table [sequences, width]`` (each sequence's pages in order) and ``lens [sequences]`` (its cached
    tokens). An entry that is no page holds nothing: not written, read as zeros, not attended to. Inference
    only: operands that require a gradient are refused."""

    def __init__(self, k: torch.Tensor, k_scales: torch.Tensor, v: torch.Tensor, v_scales: torch.Tensor):
        for name, t in (("k", k), ("k_scales", k_scales), ("v", v), ("v_scales", v_scales)):
            if t.dtype != torch.uint8:
                raise TypeError(f"Cache4: {name} is uint8, got {t.dtype}")
            if not t.is_contiguous() or t.data_ptr() % 16:
                raise RuntimeError(f"Cache4: {name} has to be contiguous and 16-byte aligned")
            if t.device != k.device:
                raise RuntimeError(f"Cache4: {name} is on {t.device}, k on {k.device}")
        if k.dim() != 4:
            raise RuntimeError("Cache4: k is [pages, heads, page, dim / 2]")
        pages, heads, page, half = k.shape
        dim = 2 * half
        if dim not in (64, 128):
            raise NotImplementedError(f"Cache4: head width {dim} (64 or 128)")
        if page < 32 or page % 32:
            raise NotImplementedError(f"Cache4: {page} tokens a page (a multiple of 32)")
        for name, t, want in (("k_scales", k_scales, self._shapes(page, dim)[1]), ("v", v, self._shapes(page, dim)[2]),
                              ("v_scales", v_scales, self._shapes(page, dim)[3])):
            if tuple(t.shape) != (pages, heads, *want):
                raise RuntimeError(f"Cache4: {name}: expected the shape {(pages, heads, *want)}, got {tuple(t.shape)}")
        self.k, self.k_scales, self.v, self.v_scales = k, k_scales, v, v_scales
        self.pages, self.heads, self.page, self.dim = pages, heads, page, dim
        self.device, self._index = k.device, k.get_device()
        self._desc = Kv4Desc(k.data_ptr(), k_scales.data_ptr(), v.data_ptr(), v_scales.data_ptr(), pages, heads, page,
                             dim)
        self._ref = ctypes.addressof(self._desc)

    @staticmethod
    def _shapes(page, dim):
        tb = 512 // dim
        return ((page, dim // 2), (page // 32, 4, dim // 32, 8), (page // tb, 16, tb, dim // 32),
                (page // 32, dim // 32, 32))

    @classmethod
    def zeros(cls, pages: int, heads: int, page: int, dim: int, device) -> "Cache4":
        """``pages`` pages of ``page`` tokens (a multiple of 32), every value 0."""
        if dim not in (64, 128) or page < 32 or page % 32:
            raise NotImplementedError(f"Cache4: heads of {dim} (64 or 128), {page} tokens a page (a multiple of 32)")
        k, ks, v, vs = ((pages, heads, *s) for s in cls._shapes(page, dim))
        u8 = dict(dtype=torch.uint8, device=device)
        return cls(torch.zeros(k, **u8), torch.ones(ks, **u8), torch.zeros(v, **u8), torch.ones(vs, **u8))

    def _table(self, table, lens, what):
        shape = table.shape
        if len(shape) != 2:
            raise RuntimeError(f"{what}: table is [sequences, pages]")
        return ints(table, shape, "table", self._index), ints(lens, shape[:1], "lens", self._index), *shape

    def append(self, new_k: torch.Tensor, new_v: torch.Tensor, table: torch.Tensor | None = None,
               lens: torch.Tensor | None = None, cu: torch.Tensor | None = None,
               slots: torch.Tensor | None = None) -> None:
        """``new_k``, ``new_v [n, heads, dim]`` (f32, bf16 or f16) into the cache: sequence ``b``'s the
        rows ``cu[b] .. cu[b + 1]``, the last ones of its ``lens[b]`` tokens (``lens`` counts them). Or, in
        place of the three, ``slots`` int64 ``[n]``: row ``i`` into place ``slots[i] % page`` of page ``slots[i]
        // page`` (``paging.Pages.grow`` gives them, for all layers at once); a slot in no page is not
        written, and none is named twice."""
        no_graph("append", new_k, new_v)
        require_device(self.device)
        code = type_of(new_k, "append")
        if new_v.dtype is not new_k.dtype:
            raise TypeError(f"append: keys are {new_k.dtype}, values {new_v.dtype}")
        shape = new_k.shape
        if new_v.shape != shape or shape[1:] != (self.heads, self.dim):
            raise RuntimeError(f"append: keys {tuple(new_k.shape)}, values {tuple(new_v.shape)}, "
                               f"the cache holds {self.heads} heads of {self.dim}")
        if new_k.get_device() != self._index or new_v.get_device() != self._index:
            raise RuntimeError(f"append: the cache is on {self.device}, keys on {new_k.device}, values on {new_v.device}")
        if slots is not None:
            if table is not None or lens is not None or cu is not None:
                raise RuntimeError("append: slots, or table, lens and cu")
            slots = ints(slots, shape[:1], "slots", self._index, torch.int64)
            (new_k, ks), (new_v, vs) = rows(new_k, code), rows(new_v, code)
            with on(self._index):
                check(lib().bq_kv4_append_slots(self._ref, new_k.data_ptr(), new_v.data_ptr(), code, shape[0], *ks, *vs,
                                                slots.data_ptr(), _stream(new_k)))
            return
        if table is None or lens is None or cu is None:
            raise RuntimeError("append: slots, or table, lens and cu")
        table, lens, B, width = self._table(table, lens, "append")
        cu = ints(cu, (B + 1,), "cu", self._index)
        (new_k, ks), (new_v, vs) = rows(new_k, code), rows(new_v, code)
        with on(self._index):
            check(lib().bq_kv4_append(self._ref, new_k.data_ptr(), new_v.data_ptr(), code, shape[0], *ks, *vs,
                                      table.data_ptr(), B, width, lens.data_ptr(), cu.data_ptr(), _stream(new_k)))

    def read(self, table: torch.Tensor, lens: torch.Tensor, most: int):
        """The keys and values held, f32 ``[sequences, heads, most, dim]`` each, zeros from
        ``lens[b]`` on."""
        require_device(self.device)
        table, lens, B, width = self._table(table, lens, "read")
        if most < 0:
            raise ValueError(f"read: {most} tokens")
        shape = (B, self.heads, most, self.dim)
        k = torch.empty(shape, dtype=torch.float32, device=self.device)
        v = torch.empty(shape, dtype=torch.float32, device=self.device)
        with on(self._index):
            check(lib().bq_kv4_read(self._ref, table.data_ptr(), B, width, lens.data_ptr(), most, k.data_ptr(), v.data_ptr(),
                                    _stream(k)))
        return k, v

    def attend(self, q: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, max_len: int | None = None,
               weights: torch.Tensor | None = None, scale: float | None = None) -> torch.Tensor:
        """Attention of each sequence's newest tokens over the cache: ``q [sequences, tokens, q_heads,
        dim]`` (f32, bf16 or f16), token ``t`` sees the first ``lens[b] - tokens + 1 + t`` cached
        tokens; where it sees none its output is 0. ``max_len``: no sequence is longer (default: what
        the table's pages hold; the work is planned for it, longer ones are cut). ``weights`` f32
        ``[sequences, heads, >= max_len]``: each cached token's softmax weights, summed over the
        queries of its key-value head, are added in place (rows that overlap, as an expanded view's, are
        refused). Returns ``[sequences, tokens, q_heads,
        dim]`` of q's type."""
        if weights is None:
            no_graph("attend", q)
        else:
            no_graph("attend", q, weights)
        require_device(self.device)
        code = type_of(q, "attend")
        shape = q.shape
        if len(shape) != 4 or shape[3] != self.dim or shape[2] % self.heads or shape[2] == 0:
            raise RuntimeError(f"attend: q {tuple(q.shape)} is [sequences, tokens, query heads, dim] over "
                               f"{self.heads} key-value heads of {self.dim}")
        if q.get_device() != self._index:
            raise RuntimeError(f"attend: the cache is on {self.device}, q on {q.device}")
        table, lens, B, width = self._table(table, lens, "attend")
        _, T, hq, dim = shape
        if shape[0] != B:
            raise RuntimeError(f"attend: {shape[0]} sequences of queries, {B} of pages")
        held = width * self.page
        max_len = held if max_len is None else max_len
        w, wb, wh = None, 0, 0
        if weights is not None:
            if weights.dtype is not torch.float32 or weights.get_device() != self._index:
                raise TypeError(f"attend: weights are float32 on {self.device}, got {weights.dtype} on {weights.device}")
            if weights.dim() != 3 or weights.shape[:2] != (B, self.heads) or weights.shape[2] < min(max_len, held):
                raise RuntimeError(f"attend: weights {tuple(weights.shape)} for {B} sequences, {self.heads} heads and "
                                   f"{min(max_len, held)} tokens")
            wb, wh, ws = weights.stride()
            if ws != 1 and weights.shape[2] > 1:
                raise RuntimeError("attend: weights of one head have to be contiguous")
            w = weights.data_ptr()
        out = torch.empty(shape, dtype=q.dtype, device=self.device)
        if B == 0 or T == 0:
            return out
        q, qs = rows(q, code)
        need = _attend_ws_bytes(B, self.heads, T * (hq // self.heads), dim, max_len, int(w is not None))
        ws = torch.empty(need, dtype=torch.uint8, device=self.device) if need else None
        with on(self._index):
            check(lib().bq_kv4_attend(self._ref, q.data_ptr(), code, T, hq, *qs, table.data_ptr(), B, width,
                                      lens.data_ptr(), max_len, dim ** -0.5 if scale is None else scale, out.data_ptr(),
                                      w, wb, wh, ws.data_ptr() if need else None, need, _stream(q)))
        return out

    def attend_chunk(self, q: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, cu: torch.Tensor,
                     max_len: int | None = None, scale: float | None = None) -> torch.Tensor:
        """Attention of chunks of new tokens over the cache, of another length for each sequence: ``q [n,
        q_heads, dim]`` (f32, bf16 or f16), sequence ``b``'s the rows ``cu[b] .. cu[b + 1]`` (``cu`` int32 on
        the device, ascending), the last ones of its ``lens[b]`` cached tokens, as ``append`` takes their
        keys and values before. Row ``i`` is token ``lens[b] - cu[b + 1] + i`` and sees the cached tokens up
        to itself; where it sees none its output is 0, and so are rows of no sequence. ``max_len``: no
        sequence is longer (default: what the table's pages hold; the work is planned for it, longer ones
        are cut). Returns ``[n, q_heads, dim]`` of q's type."""
        no_graph("attend_chunk", q)
        require_device(self.device)
        code = type_of(q, "attend_chunk")
        shape = q.shape
        if len(shape) != 3 or shape[2] != self.dim or shape[1] % self.heads or shape[1] == 0:
            raise RuntimeError(f"attend_chunk: q {tuple(q.shape)} is [tokens, query heads, dim] over {self.heads} "
                               f"key-value heads of {self.dim}")
        if q.get_device() != self._index:
            raise RuntimeError(f"attend_chunk: the cache is on {self.device}, q on {q.device}")
        table, lens, B, width = self._table(table, lens, "attend_chunk")
        cu = ints(cu, (B + 1,), "cu", self._index)
        n, hq, dim = shape
        if max_len is None:
            max_len = width * self.page
        out = torch.empty(shape, dtype=q.dtype, device=self.device)
        if n == 0:
            return out
        q, qs = rows(q, code)
        need = _chunk_ws_bytes(code, n, B, hq, self.heads, dim, max_len, self.pages * self.page)
        ws = torch.empty(need, dtype=torch.uint8, device=self.device) if need else None
        with on(self._index):
            check(lib().bq_kv4_attend_chunk(self._ref, q.data_ptr(), code, n, hq, *qs, table.data_ptr(), B, width,
                                            lens.data_ptr(), cu.data_ptr(), max_len, dim ** -0.5 if scale is None else scale,
                                            out.data_ptr(), ws.data_ptr() if need else None, need, _stream(q)))
        return out

    def evict(self, sums: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, new_table: torch.Tensor, keep: int,
              recent: int = 0):
        """Brings every (sequence, head) down to ``keep`` tokens: the ``recent`` last ones and, of the
        others, those of largest weight in ``sums`` f32 ``[sequences, heads, most]`` (what ``attend``
        added up; ties to the earlier token); a sequence of up to ``keep`` keeps all. They move in order
        to the pages of ``new_table [sequences, >= keep / page]``, none of which is in use (zeros for one whose
        entry is no page).
        Returns ``kept`` int32 ``[sequences, heads, keep]`` (their former places, -1 past the last),
        their ``weights`` (0 past the last) and ``left`` int32 ``[sequences]``, the new lengths."""
        no_graph("evict", sums)
        require_device(self.device)
        table, lens, B, width = self._table(table, lens, "evict")
        if new_table.dim() != 2 or new_table.shape[0] != B:
            raise RuntimeError(f"evict: new_table {tuple(new_table.shape)} for {B} sequences")
        new_table = ints(new_table, new_table.shape, "new_table", self._index)
        if sums.dtype is not torch.float32 or sums.get_device() != self._index:
            raise TypeError(f"evict: sums are float32 on {self.device}, got {sums.dtype} on {sums.device}")
        if sums.dim() != 3 or sums.shape[:2] != (B, self.heads):
            raise RuntimeError(f"evict: sums {tuple(sums.shape)} for {B} sequences and {self.heads} heads")
        if sums.stride(2) != 1 and sums.shape[2] > 1:
            sums = sums.contiguous()
        if keep < 1:
            raise ValueError(f"evict: keep {keep}")
        kept = torch.empty((B, self.heads, keep), dtype=torch.int32, device=self.device)
        weights = torch.empty((B, self.heads, keep), dtype=torch.float32, device=self.device)
        left = torch.empty(B, dtype=torch.int32, device=self.device)
        sb, sh, _ = sums.stride()
        need = lib().bq_kv4_evict_ws_bytes(B, self.heads, sums.shape[2], keep)
        ws = torch.empty(need, dtype=torch.uint8, device=self.device) if need else None
        with on(self._index):
            check(lib().bq_kv4_evict(self._ref, sums.data_ptr(), sb, sh, sums.shape[2], table.data_ptr(), B, width,
                                     lens.data_ptr(), new_table.data_ptr(), new_table.shape[1], keep, recent,
                                     kept.data_ptr(), weights.data_ptr(), left.data_ptr(), ws.data_ptr() if need else None,
                                     need, _stream(kept)))
        return kept, weights, left
