"""Softmax attention over whole prompts (``bq_prompt_attention``, ``include/bq.h``): sequences of
different lengths packed one after another, grouped heads, causal or not, in f32, bf16 or f16.

It is the attention between a decoder's int8 projections when a prompt is read; ``kv4`` holds the
keys and values for the tokens that follow. Inference only: operands that require a gradient are refused."""
from __future__ import annotations

from contextlib import nullcontext

import torch

from ._lib import check, lib, require_device
from .int8 import _stream

__all__ = ["prompt_attention"]

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
SIZES = (4, 2, 2)
_here = nullcontext()


def on(index: int):
    """The context in which a library call for device ``index`` runs (nothing to do on the current one)."""
    return _here if index == torch._C._cuda_getDevice() else torch.cuda.device(index)


def type_of(t: torch.Tensor, what: str) -> int:
    code = TYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"{what}: takes float32, bfloat16 or float16, got {t.dtype}")
    return code


def no_graph(what: str, *operands: torch.Tensor) -> None:
    """Refuses operands that autograd would record: the kernels keep no graph, and a result without one would
    drop their gradients in silence."""
    if torch.is_grad_enabled():
        for t in operands:
            if t.requires_grad:
                raise RuntimeError(f"{what}: no gradient is computed, and an operand requires one (torch.no_grad() or detach())")


def rows(t: torch.Tensor, code: int):
    """``t`` itself where its channels are contiguous and its rows 16-byte aligned, else a copy, and
    the strides of all axes but the last (those of an axis of one count for nothing)."""
    st = t.stride()
    if st[-1] == 1:
        every = t.data_ptr()
        for s in st[:-1]:
            every |= s * SIZES[code]
        if not every & 15:
            return t, st[:-1]
        st = [s if n > 1 else 0 for s, n in zip(st[:-1], t.shape)]
        if t.data_ptr() % 16 == 0 and not any(s * SIZES[code] % 16 for s in st):
            return t, st
    t = t.clone(memory_format=torch.contiguous_format)
    return t, t.stride()[:-1]


def ints(t: torch.Tensor, shape, what: str, index: int) -> torch.Tensor:
    """An int32 index tensor of ``shape`` on device ``index``, contiguous."""
    if t.dtype is not torch.int32:
        raise TypeError(f"{what}: expected int32, got {t.dtype}")
    if t.get_device() != index:
        raise RuntimeError(f"{what}: on {t.device}, the operands are on cuda:{index}")
    if t.shape != shape:
        raise RuntimeError(f"{what}: expected the shape {tuple(shape)}, got {tuple(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu: torch.Tensor, causal: bool = True,
                     scale: float | None = None) -> torch.Tensor:
    """``softmax(scale q k^T) v`` within each sequence: ``q [n, q_heads, dim]``, ``k``, ``v [n, heads,
    dim]`` (``heads`` divides ``q_heads``; ``dim`` 64 or 128) hold the sequences one after another,
    sequence ``b`` the rows ``cu[b] .. cu[b + 1]`` (``cu`` int32 on the device, ascending). Causal: a
    row sees the rows up to itself. ``scale`` defaults to ``dim ** -0.5``. Views of a fused
    projection's output are read in place. Returns ``[n, q_heads, dim]``; rows of no sequence are
    zeros."""
    no_graph("prompt_attention", q, k, v)
    require_device(q.device)
    code = type_of(q, "prompt_attention")
    shape = q.shape
    if len(shape) != 3 or k.dim() != 3:
        raise RuntimeError("prompt_attention: q, k and v are [tokens, heads, dim]")
    if k.dtype is not q.dtype or v.dtype is not q.dtype:
        raise TypeError(f"prompt_attention: q is {q.dtype}, k {k.dtype}, v {v.dtype}")
    index = q.get_device()
    if k.get_device() != index or v.get_device() != index:
        raise RuntimeError(f"prompt_attention: q is on {q.device}, k on {k.device}, v on {v.device}")
    n, hq, dim = shape
    kn, h, kd = k.shape
    if v.shape != k.shape or kn != n or kd != dim:
        raise RuntimeError(f"prompt_attention: shapes q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}")
    if h == 0 or hq % h:
        raise RuntimeError(f"prompt_attention: {hq} query heads over {h} key-value heads")
    B = cu.shape[0] - 1 if cu.dim() == 1 else -1
    if B < 0:
        raise RuntimeError("prompt_attention: cu holds the sequences' first rows and the end")
    cu = ints(cu, (B + 1,), "cu", index)
    out = torch.empty(shape, dtype=q.dtype, device=q.device)
    if n == 0 or hq == 0:
        return out
    (q, qs), (k, ks), (v, vs) = (rows(t, code) for t in (q, k, v))
    if code and max(ks[0], vs[0]) > 1 << 23:
        k, v = k.contiguous(), v.contiguous()
        ks, vs = k.stride()[:2], v.stride()[:2]
    need = lib().bq_prompt_attention_ws_bytes(code, n, h, dim) if code == 0 else 0
    ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    with on(index):
        check(lib().bq_prompt_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), code, n, hq, h, dim, *qs, *ks, *vs,
                                        cu.data_ptr(), B, int(causal), dim ** -0.5 if scale is None else scale,
                                        out.data_ptr(), ws.data_ptr() if need else None, need, _stream(q)))
    return out
