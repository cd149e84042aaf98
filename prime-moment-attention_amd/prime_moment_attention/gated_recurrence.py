"""The gated linear recurrence: a layer with one fp32 state per channel, beside the
moment attentions.

``gated_recurrence`` is the operator.  Per sequence and channel,

    D_t = clamp(softplus(step_t), 1e-4, 50)      the selective module's step size
    a_t = exp(-D_t / tau)                        (selective.py:368, 385-386)
    h_t = a_t h_{t-1} + sqrt(1 - a_t^2) sigmoid(gate_t) x_t,    y_t = h_t

The factor sqrt(1 - a^2) keeps a state driven by independent inputs at their scale
whatever the decay.  Prompts, training (with gradients in x, step, gate, tau and the
state) and single tokens run prime_gated_scan.

``GatedLinearRecurrence`` is the layer, with the interface of the attention modules:
``forward(hidden_states, state=None, return_state=False) -> (out, next_state)``.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
import torch.nn as nn
from torch.autograd import forward_ad

from . import _lib
from .attention import project_out
from .chunked_ssd import needs_grad, once


def _channels(t: torch.Tensor) -> torch.Tensor:
    """t with contiguous channels (as it is where they are)."""
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def _thirds(proj: torch.Tensor):
    C = proj.shape[-1] // 3
    return proj[..., :C], proj[..., C:2 * C], proj[..., 2 * C:]


class _GatedScanFn(torch.autograd.Function):
    """prime_gated_scan with its backward.  x, step and gate, or (step and gate None) x
    holding all three as thirds of its columns, whose gradient is then one tensor."""

    @staticmethod
    def forward(ctx, x, step, gate, tau, state):
        ctx.stacked = step is None
        parts = _thirds(x) if ctx.stacked else (x, step, gate)
        B, L, C = parts[0].shape
        y = torch.empty(B, L, C, device=x.device, dtype=x.dtype)
        last = torch.empty(B, C, device=x.device, dtype=torch.float32)
        ckpt = torch.empty(B, -(-L // _lib.GATED_TILE), C, device=x.device, dtype=torch.float32)
        _lib.gated_scan(*parts, tau, state, y, last, ckpt, checked=True)
        ctx.save_for_backward(x, step, gate, tau, ckpt)
        ctx.has_state = state is not None
        ctx.set_materialize_grads(False)
        return y, last

    @staticmethod
    def backward(ctx, dy, dlast):
        return once(_GatedScanFn._grads)(ctx, dy, dlast)

    @staticmethod
    def _grads(ctx, dy, dlast):
        x, step, gate, tau, ckpt = ctx.saved_tensors
        parts = _thirds(x) if ctx.stacked else (x, step, gate)
        B, L, C = parts[0].shape
        dy = torch.zeros_like(parts[0]) if dy is None else _channels(dy.to(x.dtype))
        dlast = None if dlast is None else dlast.to(torch.float32).contiguous()
        new = torch.empty(B, L, 3 * C, device=x.device, dtype=x.dtype)
        if ctx.stacked:
            grads, out = _thirds(new), (new, None, None)
        else:
            grads = out = tuple(new.view(3, B, L, C))
        dtau = torch.empty(C, device=x.device, dtype=torch.float32)
        dstate = torch.empty(B, C, device=x.device, dtype=torch.float32) if ctx.has_state else None
        _lib.gated_scan_backward(*parts, tau, ckpt, dy, dlast, *grads, dtau, dstate, checked=True)
        return (*out, dtau, dstate)


def _scan(x, step, gate, tau, state, state_out):
    """(y, last state) of x, step, gate, or of x's thirds where step is None."""
    parts = (x, step, gate) if step is not None else _thirds(x)
    B, L, C = _lib.check_gated(*parts, tau, state, state_out)
    if not (L and B and C):
        h = parts[0].new_zeros((B, C), dtype=torch.float32) if state is None else state
        if state_out is not None:
            return torch.zeros_like(parts[0]), state_out.copy_(h)
        return (0 * (parts[0] + parts[1] + parts[2] + tau + h.unsqueeze(1))).to(x.dtype), h + 0
    leaves = x.requires_grad or tau.requires_grad or (step is not None and (step.requires_grad or gate.requires_grad)) or (
        state is not None and state.requires_grad)
    if (leaves and torch.is_grad_enabled()) or forward_ad._current_level >= 0:
        if state_out is not None:
            raise ValueError("state_out cannot be written while autograd records: take the returned state")
        return _GatedScanFn.apply(x, step, gate, tau, state)
    y = x.new_empty((B, L, C))
    if state_out is None:
        state_out = tau.new_empty((B, C)) if state is None else torch.empty_like(state)
    _lib.gated_scan(*parts, tau, state, y, state_out, checked=True)
    return y, state_out


def gated_recurrence(x: torch.Tensor, step: torch.Tensor, gate: torch.Tensor, tau: torch.Tensor,
                     state: Optional[torch.Tensor] = None, return_state: bool = False,
                     state_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """The recurrence over x, step, gate [B, L, C] (fp32, bf16 or fp16 alike; any batch
    and token strides) with tau fp32 [C], positive (below 1e-30 and above 1e33 it acts as
    these), and state fp32 [B, C] or None (zero): (y [B, L, C] of x's dtype, last state fp32 [B, C] or None without
    return_state).  Every token counts: the last state of a padded sequence has taken its
    padding in.

    Differentiable once in x, step, gate, tau and state.  The given state is left as it
    is; without autograd, ``state_out`` names the tensor that receives the last state
    (it may be ``state``: a decode step in place).  Forward and backward can be captured
    into a graph; as for any operator, no eager autograd graph of the same leaves may live
    meanwhile (torch would run a part of the captured backward on that graph's stream)."""
    if not x.stride(-1) == step.stride(-1) == gate.stride(-1) == 1:
        x, step, gate = _channels(x), _channels(step), _channels(gate)
    y, last = _scan(x, step, gate, tau, state, state_out)
    return y, (last if return_state else None)


class GatedLinearRecurrence(nn.Module):
    """in_proj (x, step and gate in one product) -> gated recurrence -> o_proj.  The
    state is fp32 [B, width].  log_tau [width] is learned; tau is held between min_tau
    and max_tau as the selective module's, and starts spread evenly over their
    logarithms, with a step size of 1."""

    def __init__(self, hidden_size: int, width: Optional[int] = None, min_tau: float = 2.0,
                 max_tau: float = 2000.0):
        super().__init__()
        self.hidden_size = hidden_size
        self.width = width or hidden_size
        self.min_tau = min_tau
        self.max_tau = max_tau
        self.inplace_state = False  # True: without autograd the incoming state tensor is updated in place
        self.in_proj = nn.Linear(hidden_size, 3 * self.width, bias=True)
        self.o_proj = nn.Linear(self.width, hidden_size, bias=False)
        self.log_tau = nn.Parameter(torch.zeros(self.width, dtype=torch.float32))
        self.init_gate_weights()

    def init_gate_weights(self):
        """Step size 1 and open-half gates at zero input, memories from min_tau to max_tau: a
        hundred thousandth inside, as fp32's log and exp end up to 4e-6 beyond for any range of
        floats, where get_tau's clamp gives log_tau no gradient."""
        W = self.width
        low, high = math.log(self.min_tau), math.log(self.max_tau)
        inside = min(1e-5, (high - low) / 4)
        with torch.no_grad():
            self.in_proj.bias.zero_()
            self.in_proj.bias[W:2 * W].fill_(math.log(math.exp(1.0) - 1.0))
            self.log_tau.copy_(torch.linspace(low + inside, high - inside, W))

    def get_tau(self, device: torch.device) -> torch.Tensor:
        return torch.clamp(torch.exp(self.log_tau.to(device).float()), min=self.min_tau, max=self.max_tau)

    def mix(self, hidden_states: torch.Tensor, state: Optional[torch.Tensor] = None, return_state: bool = False,
            in_place: bool = False):
        """The layer up to its output projection: (y [B, L, width], next state or None).
        in_place (or inplace_state): without autograd the given state tensor is updated."""
        proj = _channels(self.in_proj(hidden_states))
        state_out = None
        if state is not None:
            given, state = state, state.to(device=proj.device, dtype=torch.float32).contiguous()
            if ((in_place or self.inplace_state) and return_state and state is given
                    and not needs_grad(proj, state, self.log_tau)):
                state_out = state
        y, last = _scan(proj, None, None, self.get_tau(proj.device), state, state_out)
        return y.to(hidden_states.dtype), (last if return_state else None)

    def forward(self, hidden_states: torch.Tensor, state: Optional[torch.Tensor] = None, return_state: bool = False):
        y, next_state = self.mix(hidden_states, state, return_state)
        return project_out(self.o_proj, y), next_state
