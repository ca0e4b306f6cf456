"""A beam search's selection (``bq_beam_select``, ``include/bq.h``): of the beams of each request and the whole
vocabulary the best continuations, with what ``paging.Pages.fork`` needs to reorder the caches.

    best = beam_select(logits, scores, done, end)   # one step
    pages.fork(best.parents.view(-1))"""
from __future__ import annotations

from typing import NamedTuple

import torch

from ._lib import check, lib, require_device
from .attention import no_graph, on, type_of
from .int8 import _stream

__all__ = ["Selected", "beam_select"]


class Selected(NamedTuple):
    """``scores`` f32 ``[requests, beams]``, the best first; ``parents`` int32, the sequence ``request * beams +
    beam`` that each one continues; ``tokens`` int32; ``done`` bool: ended before, or now."""
    scores: torch.Tensor
    parents: torch.Tensor
    tokens: torch.Tensor
    done: torch.Tensor


def beam_select(logits: torch.Tensor, scores: torch.Tensor, done: torch.Tensor | None = None, end: int = -1) -> Selected:
    """The ``beams`` best continuations of each request: ``logits [requests * beams, vocab]`` (f32, bf16 or f16;
    rows may lie apart), ``scores`` f32 ``[requests, beams]`` what the beams have so far. A candidate's score is
    its beam's plus the token's log-probability, taken and compared in 64 bits; NaN counts as -infinity (and so
    does all of a beam with a NaN or +infinity among its logits, nothing above -infinity there, or an infinite
    score). A beam that is ``done`` (bool ``[requests, beams]``) has one candidate, the token ``end`` at the beam's
    own score; ``end``: the token that ends a beam (-1: none does). Equals go to the lower beam; within a beam the
    order is that of its logits, then of the tokens. A search starts from
    the scores ``[0, -inf, ...]``, where all beams are alike. At most 64 beams. No gradient is computed."""
    no_graph("beam_select", logits, scores)
    require_device(logits.device)
    code = type_of(logits, "beam_select")
    index, shape, size = logits.get_device(), scores.shape, logits.shape
    if len(shape) != 2 or len(size) != 2 or size[0] != shape[0] * shape[1] or not size[1] or not shape[1]:
        raise RuntimeError(f"beam_select: logits {tuple(logits.shape)} are [requests * beams, vocab], scores "
                           f"{tuple(scores.shape)} [requests, beams]")
    B, W = shape
    V = size[1]
    if scores.dtype is not torch.float32 or scores.get_device() != index:
        raise TypeError(f"beam_select: scores are float32 on {logits.device}, got {scores.dtype} on {scores.device}")
    if done is not None:
        if done.dtype is not torch.bool or done.get_device() != index or done.shape != shape:
            raise TypeError(f"beam_select: done is bool {tuple(shape)} on {logits.device}, got {done.dtype} "
                            f"{tuple(done.shape)} on {done.device}")
        if not 0 <= end < V:
            raise ValueError(f"beam_select: end token {end} of {V}, with beams that may be done")
        done = done.contiguous()
    pitch, step = logits.stride()
    if step != 1 and V > 1:
        logits, pitch = logits.contiguous(), V
    scores = scores.contiguous()
    parents = torch.empty_like(scores, dtype=torch.int32)
    out = Selected(torch.empty_like(scores), parents, torch.empty_like(parents), torch.empty_like(scores, dtype=torch.bool))
    if B == 0:
        return out
    need = lib().bq_beam_select_ws_bytes(code, B, W, V)
    ws = torch.empty(need, dtype=torch.uint8, device=scores.device)
    with on(index):
        check(lib().bq_beam_select(logits.data_ptr(), code, B, W, V, pitch, scores.data_ptr(),
                                   None if done is None else done.data_ptr(), end, out.scores.data_ptr(),
                                   out.parents.data_ptr(), out.tokens.data_ptr(), out.done.data_ptr(), ws.data_ptr(), need,
                                   _stream(logits)))
    return out
