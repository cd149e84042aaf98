"""Training with the gated recurrence and dropout off the plain path: sequences without tokens,
moment layers with dropout, autocast."""
import pytest
import torch

from gated_ref import keep_mask
from prime_moment_attention import dropout_rng, gated_recurrence, sample_tokens
from prime_moment_attention.model import PrimeBlock

from gpu_util import dev
from test_gpu_recurrent_model import loss64, model_of

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


def step(model, ids):
    torch.manual_seed(7)
    out = model(ids.to(dev()), labels=ids.to(dev()))
    out["loss"].backward()
    return out["loss"].item(), {n: p.grad.double().cpu() for n, p in model.named_parameters()}


@pytest.mark.parametrize("gated,selective", [((), False), ((), True), ((1,), False)])
def test_moment_layers_with_dropout(gated, selective, monkeypatch):
    """The training step of models with moment layers against the same model whose dropout is a
    product with the mask: a few roundings of 2^-24 apart in each of 4 branches, 2^-11 of a
    gradient's largest value with room for what the norms' and the readouts' cancellations make
    of them."""
    ids = torch.randint(0, 120, (3, 41), generator=torch.Generator().manual_seed(1))
    loss, grads = step(model_of(gated, 0.25, use_selective=selective).train(), ids)

    def drop(block, h, residual, rng, branch):
        keep, scale = keep_mask(h.numel(), 0.25, *rng.tolist(), 2 * block.layer + branch)
        return residual + h * torch.from_numpy(keep * scale).to(h.device, h.dtype).view(h.shape)
    monkeypatch.setattr(PrimeBlock, "_drop", drop)
    want, ref = step(model_of(gated, 0.25, use_selective=selective).train(), ids)
    assert abs(loss - want) < 1e-5
    for n, g in grads.items():
        assert (g - ref[n]).abs().max() <= 2.0 ** -11 * ref[n].abs().max(), n


def test_autocast():
    """bf16 branches into the fp32 residual stream, against float64: each of some 16 products and
    norms a way rounds by 2^-9, independently, and 4 sqrt(32) 2^-9 of the largest value is four
    times their sum's spread."""
    model = model_of((0, 1), 0.25).train()
    ids = torch.randint(0, 120, (3, 41), generator=torch.Generator().manual_seed(1))
    torch.manual_seed(7)
    rng = dropout_rng(dev())
    with torch.autocast("cuda", torch.bfloat16):
        loss, grads = step(model, ids)
    ref, w = loss64(model, ids, rng)
    ref.backward()
    assert abs(loss - ref.item()) < 4 * 32 ** 0.5 * 2.0 ** -9 * ref.item()
    for n, g in grads.items():
        assert (g - w[n].grad).abs().max() <= 4 * 32 ** 0.5 * 2.0 ** -9 * w[n].grad.abs().max(), n


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int16, torch.int64])
def test_top_k_of_other_types(dtype):
    g = torch.Generator(device=dev()).manual_seed(3)
    logits, u = torch.randn(6, 500, device=dev(), generator=g), torch.rand(6, device=dev(), generator=g)
    k = torch.tensor([0, 1, 5, 50, 100, 127], device=dev())
    assert torch.equal(sample_tokens(logits, u, top_k=k.to(dtype)), sample_tokens(logits, u, top_k=k.to(torch.int32)))
