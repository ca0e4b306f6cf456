"""A small decoder served with int8 Linears, prompt attention and a 4-bit key-value cache: the operators
of ``attention`` and ``kv4`` as a program uses them.

    model = Decoder(...).to("cuda").eval()
    quantize_for_int8(model)                      # the Linears, as in any other model
    state = DecoderState(model, sequences=2, tokens=4096)
    logits = model.prompt(state, ids, [700, 33], window=16)  # packed prompts: attention over them, caches filled
    state.evict(keep=512, recent=64)                         # the tokens that received least leave
    logits = model.step(state, logits.argmax(-1))            # one token a sequence over the cache

Random weights and learned positions; the layers are pre-norm with GELU, the query heads grouped."""
from __future__ import annotations

import torch
import torch.nn as tnn

from . import nn
from .attention import prompt_attention
from .kv4 import Cache4

__all__ = ["Decoder", "DecoderState"]


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
