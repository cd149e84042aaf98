"""Training with the gated recurrence off the plain path: sequences without tokens."""
import pytest
import torch

from prime_moment_attention import gated_recurrence

from gpu_util import dev

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,L,C", [(2, 0, 8), (0, 3, 8), (2, 3, 0)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("state", [False, True])
def test_nothing_to_do_has_gradients(B, L, C, dtype, state):
    """No token, no sequence or no channel: zeros for x, step, gate and tau, and the last state's
    gradient for the state, that it is."""
    leaves = [torch.zeros(B, L, C, device=dev(), dtype=dtype).requires_grad_() for _ in range(3)]
    leaves.append(torch.ones(C, device=dev()).requires_grad_())
    st = torch.ones(B, C, device=dev()).requires_grad_() if state else None
    y, last = gated_recurrence(*leaves, state=st, return_state=True)
    assert y.shape == (B, L, C) and y.dtype == dtype and last.shape == (B, C)
    grads = torch.autograd.grad(y.sum() + last.sum(), leaves + ([st] if state else []))
    assert all(g.shape == t.shape and not g.any() for g, t in zip(grads[:4], leaves))
    if state:
        assert torch.equal(last, st) and torch.equal(grads[4], torch.ones_like(st))
