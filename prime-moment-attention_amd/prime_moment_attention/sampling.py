"""Sampled tokens from given uniform numbers: temperature, top-k, top-p and min-p in
one kernel (the choice of generate, model.py:222-233, with two more cuts and exact
tie rules)."""
from __future__ import annotations

from typing import Optional, Union

import torch

from . import _lib

Param = Union[float, torch.Tensor]


def _per_row(v, dtype, device):
    """A per-row parameter in the kernel's type (a number as it is)."""
    if not torch.is_tensor(v):
        return v
    if dtype is torch.int32 and v.dtype is not dtype:
        v = v.to(torch.int64).clamp(0, (1 << 31) - 1)  # more than int32 holds: all
    return v.to(device=device, dtype=dtype).contiguous()


def sample_tokens(logits: torch.Tensor, uniforms: torch.Tensor, temperature: Param = 1.0,
                  top_k: Union[int, torch.Tensor] = 0, top_p: Param = 1.0, min_p: Param = 0.0,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One token per row of logits [n, vocab] (fp32, bf16 or fp16; vocab at most 2^20; one
    row expanded to n gives n draws of it): int64 [n], or written into ``out`` (int64 of n
    values).

    Tokens are ranked by logit, equal ones by index, and weigh exp((logit - largest) /
    temperature).  In this order: top_k keeps the first top_k (0: all); top_p of these
    the shortest prefix that holds at least top_p of their weight (1: all); min_p of
    these the ones with at least min_p times the largest weight.  The token is the first
    kept one by index whose running weight exceeds uniforms (fp32 [n], in [0, 1)) times
    the kept weight.  Every parameter is a number or a tensor of n values.

    temperature 0 takes the first of the largest logits.  NaN counts as -infinity and
    is never chosen; a row with nothing else is sampled as if all logits were equal.
    The same inputs give the same tokens whatever the batch, stream or launch."""
    if logits.dim() == 2 and logits.shape[1] > 1 and logits.stride(1) != 1:
        logits = logits.contiguous()
    dev = logits.device
    if out is None:
        out = torch.empty(logits.shape[0], device=dev, dtype=torch.int64)
    if logits.shape[0] == 0:
        return out
    _lib.sample(logits.detach(), uniforms, _per_row(temperature, torch.float32, dev),
                _per_row(top_k, torch.int32, dev), _per_row(top_p, torch.float32, dev),
                _per_row(min_p, torch.float32, dev), out)
    return out
