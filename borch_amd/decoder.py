"""A small decoder served with int8 Linears, prompt attention and a 4-bit key-value cache: the operators
of ``attention`` and ``kv4`` as a program uses them.

    model = Decoder(...).to("cuda").eval()
    quantize_for_int8(model)                      # the Linears, as in any other model
    state = DecoderState(model, sequences=2, tokens=4096)
    logits = model.prompt(state, ids, [700, 33], window=16)  # packed prompts: attention over them, caches filled
    state.evict(keep=512, recent=64)                         # the tokens that received least leave
    logits = model.step(state, logits.argmax(-1))            # one token a sequence over the cache

Or with the page tables on the GPU: texts read in pieces of any length, and a beam search, whose steps never
wait for the host.

    state = PagedState(model, sequences=8, pages=256, width=8)
    logits = model.read(state, ids, counts)              # the next pieces of up to 8 texts, packed
    tokens, scores = model.search(state, ids, [700], beams=8, steps=32, end=0)

Random weights and learned positions; the layers are pre-norm with GELU, the query heads grouped."""
from __future__ import annotations

import torch
import torch.nn as tnn

from . import nn
from .attention import prompt_attention
from .beams import beam_select
from .kv4 import Cache4
from .paging import Pages, copy_pages

__all__ = ["Decoder", "DecoderState", "PagedState"]


class DecoderLayer(tnn.Module):
    def __init__(self, d: int, heads: int, kv_heads: int, dim: int, mlp: int):
        super().__init__()
        self.heads, self.kv_heads, self.dim = heads, kv_heads, dim
        self.ln1 = tnn.LayerNorm(d)
        self.qkv = nn.Linear(d, (heads + 2 * kv_heads) * dim)
        self.proj = nn.Linear(heads * dim, d)
        self.ln2 = tnn.LayerNorm(d)
        self.fc1 = nn.Linear(d, mlp)
        self.fc2 = nn.Linear(mlp, d)

    def heads_of(self, x):
        """q [n, heads, dim], k and v [n, kv_heads, dim] of the tokens ``x [n, d]``: views of one output."""
        y = self.qkv(self.ln1(x)).view(x.shape[0], -1, self.dim)
        h, g = self.heads, self.kv_heads
        return y[:, :h], y[:, h:h + g], y[:, h + g:]

    def close(self, x, o):
        """The rest of the layer after the heads' outputs ``o [n, heads, dim]``."""
        x = x + self.proj(o.reshape(x.shape[0], -1))
        return x + self.fc2(tnn.functional.gelu(self.fc1(self.ln2(x))))


class Decoder(tnn.Module):
    def __init__(self, layers: int = 4, d: int = 512, heads: int = 8, kv_heads: int = 2, dim: int = 64, mlp: int = 2048,
                 vocab: int = 1024, context: int = 8192):
        super().__init__()
        self.embed, self.places = tnn.Embedding(vocab, d), tnn.Embedding(context, d)
        self.layers = tnn.ModuleList(DecoderLayer(d, heads, kv_heads, dim, mlp) for _ in range(layers))
        self.ln = tnn.LayerNorm(d)
        self.head = nn.Linear(d, vocab)
        self.kv_heads, self.dim, self.context = kv_heads, dim, context

    @torch.no_grad()
    def prompt(self, state: "DecoderState", ids: torch.Tensor, lens, window: int = 0) -> torch.Tensor:
        """Prompts packed one after another, ``ids [sum(lens)]``, into an empty ``state``; the logits of
        each one's last token ``[len(lens), vocab]``. What the cached tokens receive from the last ``window``
        tokens of each prompt is added to their sums, which an eviction goes by (0: none of it)."""
        if window < 0:
            raise ValueError(f"prompt: a window of {window} tokens")
        if ids.shape != (sum(lens),):
            raise RuntimeError(f"ids {tuple(ids.shape)} for prompts of {sum(lens)} tokens")
        cu = state.begin(lens)
        at = torch.cat([torch.arange(n, device=ids.device) for n in lens])
        window = min(window, state.longest)
        # of a prompt shorter than the window the first rows see nothing, whichever they are
        last = (cu[1:, None].long() - window + torch.arange(window, device=ids.device)).clamp_min(0)
        x = self.embed(ids) + self.places(at)
        for i, (layer, cache) in enumerate(zip(self.layers, state.caches)):
            q, k, v = layer.heads_of(x)
            cache.append(k, v, state.table, state.lens, cu)
            if window:
                cache.attend(q[last], state.table, state.lens, max_len=state.longest, weights=state.sums[i])
            x = layer.close(x, prompt_attention(q, k, v, cu))
        state.scored = window > 0
        return self.head(self.ln(x[cu[1:].long() - 1]))

    @torch.no_grad()
    def step(self, state: "DecoderState", ids: torch.Tensor) -> torch.Tensor:
        """One more token of each sequence, ``ids [sequences]``; its logits ``[sequences, vocab]``."""
        if ids.shape != (state.sequences,):
            raise RuntimeError(f"ids {tuple(ids.shape)} for {state.sequences} sequences")
        cu, at = state.grow()
        x = self.embed(ids) + self.places(at)
        for i, (layer, cache) in enumerate(zip(self.layers, state.caches)):
            q, k, v = layer.heads_of(x)
            cache.append(k, v, state.table, state.lens, cu)
            o = cache.attend(q[:, None], state.table, state.lens, max_len=state.longest, weights=state.sums[i])
            x = layer.close(x, o[:, 0])
        state.scored = True
        return self.head(self.ln(x))


    @torch.no_grad()
    def read(self, state: "PagedState", ids: torch.Tensor, counts: torch.Tensor) -> torch.Tensor:
        """The next ``counts`` int32 ``[sequences]`` tokens of each sequence, packed, ``ids [sum(counts)]`` (or
        more rows, past the last): a prompt's next piece, one token, or none. The logits of each one's last token
        ``[sequences, vocab]``; those of a sequence without new tokens say nothing, and where not all tokens find
        room (``state.ok`` 0) nothing changes and none do."""
        if ids.dim() != 1 or not len(ids) or ids.device != state.pages.device:
            raise RuntimeError(f"read: ids {tuple(ids.shape)} on {ids.device} are the tokens, one at least, on {state.pages.device}")
        got = state.pages.grow(counts, ids.shape[0])
        copy_pages(state.caches, got.moves)
        state.ok = got.ok
        x = self.embed(ids) + self.places(got.at.clamp_min(0))
        for layer, cache in zip(self.layers, state.caches):
            q, k, v = layer.heads_of(x)
            cache.append(k, v, slots=got.slots)
            x = layer.close(x, cache.attend_chunk(q, state.pages.table, state.pages.lens, got.cu))
        last = x[(got.cu[1:].long() - 1).clamp_min(0)]
        return self.head(self.ln(last))

    @torch.no_grad()
    def search(self, state: "PagedState", ids: torch.Tensor, lens, beams: int, steps: int, end: int = 0):
        """Beam search of ``steps`` tokens after each of the prompts ``ids [sum(lens)]``, packed, in a ``state`` of
        ``len(lens) * beams`` sequences; what they hold ends first. ``tokens`` int32 ``[prompts, beams, steps]``
        and ``scores`` f32 ``[prompts, beams]``, the best first; a beam that has ended goes on with ``end`` and
        gives its pages back."""
        B, S, dev = len(lens), len(lens) * beams, ids.device
        if state.pages.sequences != S or beams < 1 or steps < 1 or B < 1 or min(lens) < 1:
            raise RuntimeError(f"search: {B} prompts of at least one token, {beams} beams and {steps} steps, in a state of "
                               f"{state.pages.sequences} sequences")
        if ids.shape != (sum(lens),):
            raise RuntimeError(f"ids {tuple(ids.shape)} for prompts of {sum(lens)} tokens")
        if beams > 64 or not 0 <= end < self.embed.num_embeddings:
            raise RuntimeError(f"search: {beams} beams (64 at most), end token {end} of {self.embed.num_embeddings}")
        if max(lens) + steps - 1 > state.pages.width * state.pages.page:
            raise RuntimeError(f"search: {max(lens)} tokens and {steps - 1} more in a state of "
                               f"{state.pages.width * state.pages.page} a sequence")
        counts = torch.zeros(B, beams, dtype=torch.int32, device=dev)
        counts[:, 0] = torch.tensor(lens, dtype=torch.int32, device=dev)
        scores = torch.full((B, beams), -torch.inf, device=dev)
        scores[:, 0] = 0.0
        done = torch.zeros(B, beams, dtype=torch.bool, device=dev)
        tokens = torch.zeros(S, steps, dtype=torch.int32, device=dev)
        state.pages.cut(torch.zeros(S, dtype=torch.int32, device=dev))
        logits = self.read(state, ids, counts.view(-1))
        room, blank = state.ok, torch.zeros(S + 1, dtype=torch.int32, device=dev)
        one, none = torch.ones_like(blank[1:]), torch.full_like(blank[1:], -1)
        for t in range(steps):
            scores, parents, new, done = beam_select(logits, scores, done, end)
            tokens = tokens[parents.view(-1)]
            tokens[:, t] = new.view(-1)
            if t + 1 < steps:
                over = done.view(-1)
                state.pages.fork(torch.where(over, none, parents.view(-1)))
                live = over ^ one
                packed = blank.scatter(0, live.cumsum(0) * live, new.view(-1))  # those of ended beams at 0, left out
                logits = self.read(state, packed[1:], live)
                room = room * state.ok
        if not room.item():
            raise RuntimeError(f"search: the state's {state.pages.pages} pages are too few")
        return tokens.view(B, beams, steps), scores


class PagedState:
    """The caches of ``sequences`` sequences of up to ``width`` pages each out of ``pages``, whose tables are kept
    on the GPU (``paging.Pages``): ``pages.fork`` and ``pages.cut`` between the model's calls."""

    def __init__(self, model: Decoder, sequences: int, pages: int, width: int, page: int = 64):
        if width * page > model.context:
            raise RuntimeError(f"sequences of {width * page} tokens, the model has places for {model.context}")
        device = next(model.parameters()).device
        self.caches = [Cache4.zeros(pages, model.kv_heads, page, model.dim, device) for _ in model.layers]
        self.pages = Pages.zeros(sequences, width, pages, page, device)
        self.ok = torch.ones(1, dtype=torch.int32, device=device)


class DecoderState:
    """The caches of ``sequences`` sequences of up to ``tokens`` tokens, their page tables and lengths, and
    what each cached token received so far."""

    def __init__(self, model: Decoder, sequences: int, tokens: int, page: int = 64):
        p = next(model.parameters())
        width = -(-tokens // page)
        self.page, self.sequences, self.tokens, self.context = page, sequences, tokens, model.context
        # twice the pages: those in use, and those that an eviction fills
        self.caches = [Cache4.zeros(2 * sequences * width, model.kv_heads, page, model.dim, p.device) for _ in model.layers]
        self.free = list(range(2 * sequences * width))
        self.pages = [[] for _ in range(sequences)]  # of each sequence, on the host
        self.held, self.next = [0] * sequences, [0] * sequences  # cached tokens; the next token's place in the text
        self.table = torch.full((sequences, width), -1, dtype=torch.int32, device=p.device)
        self.lens = torch.zeros(sequences, dtype=torch.int32, device=p.device)
        self.sums = [torch.zeros(sequences, model.kv_heads, width * page, device=p.device) for _ in model.layers]
        self.scored = False  # whether the sums hold anything: steps add to them, prompts by their window

    @property
    def longest(self) -> int:
        return max(self.held)

    def _ints(self, values):
        return torch.tensor(values, dtype=torch.int32, device=self.table.device)

    def _room(self, lens):
        """Pages for `lens` tokens a sequence; the table and the lengths that say so."""
        if max(lens) > self.tokens:
            raise RuntimeError(f"{max(lens)} tokens in a cache of {self.tokens} a sequence")
        for pages, n in zip(self.pages, lens):
            while len(pages) * self.page < n:
                pages.append(self.free.pop())
        self.held = list(lens)
        width = self.table.shape[1]
        self.table.copy_(self._ints([p + [-1] * (width - len(p)) for p in self.pages]))
        self.lens.copy_(self._ints(self.held))

    def _in_context(self, places):
        """Refuses texts that go on past the model's learned places, before anything changes: evictions keep
        the caches short, not the texts."""
        if max(places) > self.context:
            raise RuntimeError(f"a text of {max(places)} tokens, the model has places for {self.context}")

    def begin(self, lens):
        """Room for the prompts; their first rows, packed, and the end."""
        if any(self.held):
            raise RuntimeError("the state holds tokens already")
        if len(lens) != self.sequences or min(lens) < 1:
            raise RuntimeError(f"{len(lens)} prompts of at least one token for {self.sequences} sequences")
        self._in_context(lens)
        self._room(lens)
        self.next = list(lens)
        return torch.cumsum(self._ints([0] + list(lens)), 0, dtype=torch.int32)

    def grow(self):
        """Room for one more token a sequence; their rows, and their places in the text."""
        self._in_context([n + 1 for n in self.next])
        self._room([n + 1 for n in self.held])
        at = torch.tensor(self.next, device=self.table.device)
        self.next = [n + 1 for n in self.next]
        return self._ints(list(range(self.sequences + 1))), at

    def evict(self, keep: int, recent: int = 0) -> None:
        """Every sequence down to ``keep`` tokens a head, in every layer (``Cache4.evict``)."""
        if keep < 1 or not 0 <= recent <= keep:
            raise ValueError(f"evict: keep {keep}, the {recent} latest of them")
        if keep >= self.longest:
            return
        if not self.scored and recent < keep:
            raise RuntimeError("evict: no cached token has received anything yet (prompt's window, or a step)")
        width = -(-keep // self.page)
        fresh = [[self.free.pop() for _ in range(width)] for _ in range(self.sequences)]
        table = self._ints(fresh)
        for cache, sums in zip(self.caches, self.sums):
            _, weights, left = cache.evict(sums, self.table, self.lens, table, keep, recent)
            sums.zero_()
            sums[:, :, :keep] = weights
        for pages in self.pages:
            self.free += pages
        lens = [min(n, keep) for n in self.held]
        self.pages = fresh
        for pages, n in zip(self.pages, lens):
            while len(pages) > -(-n // self.page):
                self.free.append(pages.pop())
        self._room(lens)
