"""Softmax attention over whole prompts (``bq_prompt_attention``, ``include/bq.h``): sequences of
different lengths packed one after another, grouped heads, causal or not, in f32, bf16 or f16.

It is the attention between a decoder's int8 projections when a prompt is read; ``kv4`` holds the
keys and values for the tokens that follow. Inference only: no gradient."""
from __future__ import annotations

import math

import torch

from ._lib import check, lib, require_device
from .int8 import _stream

__all__ = ["prompt_attention"]

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def type_of(t: torch.Tensor, what: str) -> int:
    code = TYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"{what}: takes float32, bfloat16 or float16, got {t.dtype}")
    return code


def rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` itself where its channels are contiguous and its rows 16-byte aligned, else a copy."""
    size = t.element_size()
    if t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(
            s * size % 16 == 0 for s, n in zip(t.stride()[:-1], t.shape) if n > 1):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def strides(t: torch.Tensor):
    """Strides of all axes but the last (0 for an axis of one)."""
    return [s if n > 1 else 0 for s, n in zip(t.stride()[:-1], t.shape)]


def ints(t: torch.Tensor, n, what: str, device) -> torch.Tensor:
    """An int32 index tensor of ``n`` entries on ``device``, contiguous."""
    if t.dtype != torch.int32:
        raise TypeError(f"{what}: expected int32, got {t.dtype}")
    if t.device != device:
        raise RuntimeError(f"{what}: on {t.device}, the operands are on {device}")
    if tuple(t.shape) != tuple(n):
        raise RuntimeError(f"{what}: expected the shape {tuple(n)}, got {tuple(t.shape)}")
    return t.contiguous()


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu: torch.Tensor, causal: bool = True,
                     scale: float | None = None) -> torch.Tensor:
    """``softmax(scale q k^T) v`` within each sequence: ``q [n, q_heads, dim]``, ``k``, ``v [n, heads,
    dim]`` (``heads`` divides ``q_heads``; ``dim`` 64 or 128) hold the sequences one after another,
    sequence ``b`` the rows ``cu[b] .. cu[b + 1]`` (``cu`` int32 on the device, ascending). Causal: a
    row sees the rows up to itself. ``scale`` defaults to ``dim ** -0.5``. Views of a fused
    projection's output are read in place. Returns ``[n, q_heads, dim]``; rows of no sequence are
    zeros."""
    require_device(q.device)
    code = type_of(q, "prompt_attention")
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise RuntimeError("prompt_attention: q, k and v are [tokens, heads, dim]")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"prompt_attention: q is {q.dtype}, k {k.dtype}, v {v.dtype}")
    if k.device != q.device or v.device != q.device:
        raise RuntimeError(f"prompt_attention: q is on {q.device}, k on {k.device}, v on {v.device}")
    n, hq, dim = q.shape
    h = k.shape[1]
    if k.shape != v.shape or k.shape[0] != n or k.shape[2] != dim:
        raise RuntimeError(f"prompt_attention: shapes q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}")
    if h == 0 or hq % h:
        raise RuntimeError(f"prompt_attention: {hq} query heads over {h} key-value heads")
    if cu.dim() != 1 or cu.shape[0] < 1:
        raise RuntimeError("prompt_attention: cu holds the sequences' first rows and the end")
    cu = ints(cu, cu.shape, "cu", q.device)
    out = torch.empty((n, hq, dim), dtype=q.dtype, device=q.device)
    if n == 0 or hq == 0:
        return out
    q, k, v = (x if max(strides(x)) <= 1 << 23 else x.contiguous() for x in (rows(q), rows(k), rows(v)))
    need = lib().bq_prompt_attention_ws_bytes(code, n, h, dim)
    ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    with torch.cuda.device(q.device):
        check(lib().bq_prompt_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), code, n, hq, h, dim, *strides(q),
                                        *strides(k), *strides(v), cu.data_ptr(), cu.shape[0] - 1, int(causal),
                                        1.0 / math.sqrt(dim) if scale is None else scale, out.data_ptr(),
                                        None if ws is None else ws.data_ptr(), need, _stream(q)))
    return out
