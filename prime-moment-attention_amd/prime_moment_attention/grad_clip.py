"""The norm over many parameters' gradients, and clipping by it, in two launches for up to
192 tensors, without waiting for the device."""
from __future__ import annotations

from typing import Iterable, List, Tuple, Union

import torch

from . import _lib

Parameters = Union[torch.Tensor, Iterable[torch.Tensor]]
_grad_of, _is_contiguous = torch._C.TensorBase.grad.__get__, torch._C.TensorBase.is_contiguous


def _grads(parameters: Parameters) -> List[torch.Tensor]:
    if isinstance(parameters, torch.Tensor):
        parameters = (parameters,)
    return [g for g in map(_grad_of, parameters) if g is not None]


def _dense(g: torch.Tensor, written: bool) -> bool:
    """Whether g's elements fill a range of memory; ValueError where some share one and are to be
    written."""
    span, apart = 1, True
    for stride, size in sorted((st, sz) for sz, st in zip(g.shape, g.stride()) if sz != 1):
        apart = apart and stride >= span
        span += stride * (size - 1)
    if written and not apart:
        raise ValueError(f"a gradient of shape {tuple(g.shape)} and strides {g.stride()} overlaps itself")
    return apart and span == g.numel()


def _flat(grads: List[torch.Tensor], written: bool) -> Tuple[List[torch.Tensor], list]:
    """The gradients as ranges of memory, copies in place of those that are none, and
    (gradient, copy) of these."""
    if all(map(_is_contiguous, grads)):
        return grads, []
    copies = []
    for i, g in enumerate(grads):
        if g.layout is not torch.strided:
            raise ValueError(f"a gradient of layout {g.layout}: dense ones are needed")
        if not g.is_contiguous() and g.numel() and not _dense(g, written):
            grads[i] = g.detach().contiguous()
            copies.append((g.detach(), grads[i]))
    return grads, copies


def _norm_of(grads: List[torch.Tensor]) -> torch.Tensor:
    return torch.empty((), device=grads[0].device, dtype=torch.float32)


def grad_norm(parameters: Parameters) -> torch.Tensor:
    """The 2-norm over all gradients of the parameters (those without one are passed over) as
    one vector: an fp32 scalar on their device, its squares summed in 64 bits in a fixed order.
    Gradients: fp32, bf16 and fp16 as they come, on one device."""
    grads = _grads(parameters)
    if not grads:
        return torch.zeros(())
    grads, _ = _flat(grads, False)
    norm = _norm_of(grads)
    _lib.grad_norm(grads, norm)
    return norm


def clip_grad_norm_(parameters: Parameters, max_norm: float) -> torch.Tensor:
    """grad_norm, and every gradient times min(1, max_norm / (norm + 1e-6)) in place, in fp32,
    rounded once.  Returns the norm before clipping; the device is not waited for.

    Nothing is written where that factor is 1.  The factor is taken from the norm in 64 bits, so
    that finite gradients are clipped to max_norm also where the norm is beyond fp32 and returned
    as infinity.  An infinite element gives 0 (and NaN in its own place), a NaN NaN, as
    torch.nn.utils.clip_grad_norm_; an infinite max_norm clips nothing.  Gradients must not overlap each other."""
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm={max_norm} below 0")
    grads = _grads(parameters)
    if not grads:
        return torch.zeros(())
    written = list(grads)
    grads, copies = _flat(grads, True)
    norm = _norm_of(grads)
    _lib.grad_norm(grads, norm, max_norm)
    for g, copy in copies:
        g.copy_(copy)
    torch.autograd.graph.increment_version(written)
    return norm


def clip_grads_with_norm_(parameters: Parameters, max_norm: float, norm: torch.Tensor) -> None:
    """clip_grad_norm_ by a given norm (fp32 scalar on the gradients' device), as where it is
    taken over several processes' gradients: the root of the sum of their grad_norm squared.  An
    infinite norm gives 0."""
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm={max_norm} below 0")
    grads = _grads(parameters)
    if not grads:
        return
    written = list(grads)
    grads, copies = _flat(grads, True)
    _lib.grad_norm(grads, norm, max_norm, given=True)
    for g, copy in copies:
        g.copy_(copy)
    torch.autograd.graph.increment_version(written)
