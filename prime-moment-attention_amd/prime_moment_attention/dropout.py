"""Dropout with the residual add of a block's branch, from a counter-based generator:
the mask is computed where it is used, in the forward and again in the backward, and
never stored.

The random bits are Philox4x32-10 of (element, rng, call) alone, so a mask can be had
again from the two numbers in ``rng``, whatever the strides, the stream or the launch.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd import forward_ad

from . import _lib
from .chunked_ssd import needs_grad, once


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t as 2-D rows with contiguous columns: a view where the strides allow one."""
    cols = t.shape[-1] if t.dim() else 1
    if cols > 1 and t.stride(-1) != 1:
        t = t.contiguous()
    try:
        t = t.view(-1, cols)
    except RuntimeError:
        t = t.reshape(-1, cols)
    return t if t.shape[0] <= 1 or t.stride(0) >= cols else t.contiguous()


def _run(x, residual, p, rng, call) -> torch.Tensor:
    if x.is_contiguous() and (residual is None or residual.is_contiguous()):
        out = torch.empty_like(x)
        _lib.dropout_add(x, residual, out, p, rng, call)
        return out
    out = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    _lib.dropout_add(_rows(x), None if residual is None else _rows(residual), out.view(-1, x.shape[-1]), p, rng, call)
    return out


class _DropoutAddFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, rng, call):
        ctx.p, ctx.call = p, call
        ctx.save_for_backward(rng)  # an rng changed in place before the backward is refused
        return _run(x, residual, p, rng, call)

    @staticmethod
    def backward(ctx, dy):
        return once(_DropoutAddFn._grads)(ctx, dy)

    @staticmethod
    def _grads(ctx, dy):
        rng, = ctx.saved_tensors
        dx = _run(dy, None, ctx.p, rng, ctx.call) if ctx.needs_input_grad[0] else None
        return dx, (dy if ctx.needs_input_grad[1] else None), None, None, None


def dropout_rng(device, generator: Optional[torch.Generator] = None) -> torch.Tensor:
    """A fresh (seed, offset) for dropout_add, int64 [2] on the device, drawn from torch's
    generator (so torch.manual_seed repeats it, and a captured draw is new at each replay)."""
    return torch.randint(0, 1 << 62, (2,), device=device, generator=generator)


def dropout_add(x: torch.Tensor, residual: Optional[torch.Tensor], p: float, rng: torch.Tensor,
                call: int = 0) -> torch.Tensor:
    """residual + dropout(x) (residual None: dropout(x)): each element of x is kept with
    probability 1 - p and divided by it, in fp32, the sum rounded once; p counts in
    steps of 1/65536.

    x: fp32, bf16 or fp16 on the device, any shape; residual: the same shape and dtype.
    rng: int64 [2] on the device, (seed, offset), read when the kernel runs; ``call``
    tells apart the places of a model that share one rng.  Differentiable once; rng must
    keep its values until the backward has run."""
    if x.dim() == 0:
        raise ValueError("x must have at least one dimension")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"residual is {tuple(residual.shape)} {residual.dtype}, x {tuple(x.shape)} {x.dtype}")
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"p={p} outside [0, 1]")
    if not -(1 << 63) <= call < 1 << 63:
        raise ValueError(f"call={call} outside 64 bits")
    _lib._same_device(x, residual, rng)
    if x.numel() == 0:
        return x * 1 if residual is None else x + residual
    if needs_grad(x, residual) or forward_ad._current_level >= 0:
        return _DropoutAddFn.apply(x, residual, float(p), rng, int(call))
    return _run(x, residual, p, rng, call)
