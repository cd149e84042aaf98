"""Embedding lookup with a scale, and its gradient by sorted tokens: rows of equal ids are
summed in a fixed order in fp32, without atomics, so that a training step repeats bit for bit.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd import forward_ad

from . import _lib
from .chunked_ssd import needs_grad, once
from .dropout import _rows


def _run(ids, weight, scale, padding=-1, order=None) -> torch.Tensor:
    out = weight.new_empty((*ids.shape, weight.shape[1]))
    if out.numel() == 0:
        return out
    if weight.shape[0] == 0:
        return out.zero_()
    _lib.embedding(ids, weight, scale, out, padding, order, checked=True)
    return out


class _EmbeddingFn(torch.autograd.Function):
    """The lookup makes the tokens' order by their ids too, which is all that the gradient needs
    of them."""

    @staticmethod
    def forward(ctx, weight, ids, scale, padding):
        V, C = ctx.table = weight.shape
        n = ids.numel()
        order = ctx.gradient = None
        if n and V and C:
            order = _lib.embedding_order(n, V, weight.device)
            ctx.gradient = _lib.embedding_gradient(n, V, C, weight.dtype, weight.device, scale)
        ctx.save_for_backward(order)
        return _run(ids, weight, scale, padding, order)

    @staticmethod
    def backward(ctx, dy):
        return once(_EmbeddingFn._grads)(ctx, dy)

    @staticmethod
    def _grads(ctx, dy):
        order, = ctx.saved_tensors
        if ctx.gradient is None:
            return dy.new_zeros(ctx.table), None, None, None
        dweight, pitch = dy.new_empty(ctx.table), ctx.table[1]
        if not dy.is_contiguous():
            dy = _rows(dy)
            pitch = dy.stride(0) if dy.shape[0] > 1 else pitch
        ctx.gradient(order, dy, pitch, dweight)
        return dweight, None, None, None


def embedding_lookup(ids: torch.Tensor, weight: torch.Tensor, scale: float = 1.0,
                     padding_idx: Optional[int] = None) -> torch.Tensor:
    """scale * weight[ids]: [*ids.shape, C] of weight's dtype, the product in fp32 and rounded
    once (a copy where scale is 1).

    ids: int64 or int32, any shape; weight: [V, C <= 2^20] fp32, bf16 or fp16 on the same
    device.  An id outside [0, V) gives a row of zeros and takes no gradient; padding_idx (from -V to
    V - 1) is looked up but takes none.

    Differentiable once in weight: a dense gradient [V, C], each row the sum over its tokens
    in a fixed order, in fp32, rounded once.  Forward and backward can be captured into a graph
    (the ids may change between replays)."""
    if weight.dim() != 2:
        raise ValueError(f"weight has shape {tuple(weight.shape)}, expected [V, C]")
    if ids.dtype is not torch.int64 and ids.dtype is not torch.int32:
        raise ValueError(f"ids are {ids.dtype}: int64 or int32 is needed")
    V, C = weight.shape
    _lib.check_columns(C)
    padding = -1
    if padding_idx is not None:
        if not -V <= padding_idx < V:
            raise ValueError(f"padding_idx={padding_idx} outside the table of {V}")
        padding = int(padding_idx) % V
    if weight.dtype not in _lib._DTYPES:
        raise RuntimeError(f"unsupported dtype {weight.dtype}")
    _lib._same_device(weight, ids)
    if not ids.is_contiguous():
        ids = ids.contiguous()
    if (C > 1 and weight.stride(1) != 1) or (V > 1 and weight.stride(0) < C):
        weight = weight.contiguous()
    if needs_grad(weight) or forward_ad._current_level >= 0:
        return _EmbeddingFn.apply(weight, ids, float(scale), padding)
    return _run(ids, weight, float(scale))
