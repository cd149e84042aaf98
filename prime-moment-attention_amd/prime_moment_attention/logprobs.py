"""Log probabilities of given tokens, with the entropy and the likeliest alternatives, and
their gradient: one pass over the logits forward, one backward, nothing of their size kept
or made but the gradient itself."""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

from . import _lib
from .chunked_ssd import needs_grad, once

MAX_TOP = 64


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor
    entropy: Optional[torch.Tensor]
    top_logprobs: Optional[torch.Tensor]
    top_tokens: Optional[torch.Tensor]


def _rows(logits: torch.Tensor) -> torch.Tensor:
    """[n, vocab] with a contiguous vocabulary: a view where the strides allow one."""
    if logits.shape[-1] > 1 and logits.stride(-1) != 1:
        logits = logits.contiguous()
    return logits if logits.dim() == 2 else logits.reshape(-1, logits.shape[-1])


def _run(logits, tokens, top, entropy, ignore, stats):
    lead, dev, f32 = tokens.shape, logits.device, torch.float32
    lp = torch.empty(lead, device=dev, dtype=f32)
    ent = torch.empty(lead, device=dev, dtype=f32) if entropy else None
    top_lp = torch.empty((*lead, top), device=dev, dtype=f32) if top else None
    top_tokens = torch.empty((*lead, top), device=dev, dtype=torch.int64) if top else None
    if lp.numel():
        _lib.token_logprobs(_rows(logits), tokens, ignore, lp, ent, stats, top, top_lp, top_tokens, checked=True)
    return lp, ent, top_lp, top_tokens


class _TokenLogprobsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, top, entropy, ignore):
        stats = torch.empty((*tokens.shape, 2), device=logits.device, dtype=torch.float32)
        out = _run(logits, tokens, top, entropy, ignore, stats)
        ctx.gradient = _lib.token_logprobs_gradient(tokens.numel(), logits.shape[-1], logits.dtype, logits.device, ignore)
        ctx.save_for_backward(logits, tokens, stats, out[1])
        if top:
            ctx.mark_non_differentiable(out[2], out[3])
        ctx.set_materialize_grads(False)
        return out

    @staticmethod
    def backward(ctx, dlogprobs, dentropy, *_):
        return once(_TokenLogprobsFn._grads)(ctx, dlogprobs, dentropy)

    @staticmethod
    def _grads(ctx, dlogprobs, dentropy):
        if dlogprobs is None and dentropy is None:
            return None, None, None, None, None
        logits, tokens, stats, entropy = ctx.saved_tensors
        if dlogprobs is not None and not dlogprobs.is_contiguous():
            dlogprobs = dlogprobs.contiguous()
        if dentropy is not None and not dentropy.is_contiguous():
            dentropy = dentropy.contiguous()
        dlogits = logits.new_empty(logits.shape)
        if dlogits.numel():
            ctx.gradient(logits if logits.is_contiguous() else _rows(logits), tokens, stats, entropy, dlogprobs, dentropy, dlogits)
        return dlogits, None, None, None, None


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0, entropy: bool = False,
                   ignore_index: int = -100) -> TokenLogprobs:
    """With p = softmax(logits) over the last dimension, in fp32:

      logprobs [...]            log p[token]; 0 where the token is ignore_index, NaN for another
                                token outside the vocabulary
      entropy [...]             -sum p log p (None without ``entropy``)
      top_tokens [..., top]     the ``top`` (at most 64) largest logits' tokens, equal ones by
      top_logprobs [..., top]   index, NaN as -infinity, and their log probabilities
                                (None for top 0)

    logits: [..., vocab] fp32, bf16 or fp16, fewer than 2^31 rows of at most 2^24; tokens: [...]
    int64 or int32.  A logit of -infinity has probability 0 (a row of nothing else: log
    probabilities -infinity, entropy 0, no gradient); +infinity shares the probability with its
    equals; a NaN makes its row's results NaN.  The mean of -logprobs over the tokens that count is
    the cross entropy.

    Differentiable once in logits through logprobs and entropy, not through the top ones.
    Forward and backward can be captured into a graph."""
    if logits.dim() < 1 or logits.shape[:-1] != tokens.shape:
        raise ValueError(f"logits {tuple(logits.shape)} and tokens {tuple(tokens.shape)}: [..., vocab] and [...] are needed")
    if tokens.dtype is not torch.int64:
        if tokens.dtype is not torch.int32:
            raise ValueError(f"tokens are {tokens.dtype}: int64 or int32 is needed")
        tokens = tokens.to(torch.int64)
    if logits.dtype not in _lib._DTYPES:
        raise RuntimeError(f"unsupported dtype {logits.dtype}")
    if logits.shape[-1] == 0:
        raise ValueError("the vocabulary is empty")
    _lib.check_logits_size(tokens.numel(), logits.shape[-1])
    if not 0 <= top <= min(MAX_TOP, logits.shape[-1]):
        raise ValueError(f"top={top} outside 0 .. min({MAX_TOP}, vocab)")
    if not -(1 << 63) <= ignore_index < 1 << 63:
        raise ValueError(f"ignore_index={ignore_index} outside 64 bits")
    _lib._same_device(logits, tokens)
    tokens = tokens.contiguous()
    if needs_grad(logits) or forward_ad._current_level >= 0:
        return TokenLogprobs(*_TokenLogprobsFn.apply(logits, tokens, int(top), bool(entropy), int(ignore_index)))
    return TokenLogprobs(*_run(logits, tokens, int(top), entropy, int(ignore_index), None))
