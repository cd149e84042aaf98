"""CPU tests of the host side of gated layers, dropout and sampling: what layers begin with, the
warm start of a model that has some, blocks and configurations without dropout, types of top_k."""
import dataclasses
from types import SimpleNamespace

import pytest
import torch

from prime_moment_attention import GatedLinearRecurrence, PrimeConfig, PrimeForCausalLM
from prime_moment_attention.sampling import _per_row


@pytest.mark.parametrize("min_tau,max_tau,decay", [(1.0, 8000.0, 0.99), (2.0, 2000.0, 0.99), (3.0, 50.0, 0.995),
                                                   (200.0, 900.0, 0.9)])
@pytest.mark.parametrize("config_as_dict", [False, True])
def test_warm_start_keeps_the_gated_layers(tmp_path, min_tau, max_tau, decay, config_as_dict):
    """The same tau as the base's in every channel, those that training has moved past the ends
    too (off by the rounding of log and exp where the range had to be widened), and selective
    layers that begin with the base's decay though its tau lies outside that range."""
    cfg = PrimeConfig(vocab_size=96, hidden_size=128, num_layers=3, num_heads=2, head_dim=64, decay=decay,
                      min_tau=min_tau, max_tau=max_tau, gated_layers=(0, 2))
    torch.manual_seed(0)
    base = PrimeForCausalLM(cfg)
    with torch.no_grad():
        base.layers[2].self_attn.log_tau.add_(torch.randn(128))
    path = tmp_path / "base.pt"
    torch.save({"config": dataclasses.asdict(cfg) if config_as_dict else cfg,
                "model_state_dict": base.state_dict()}, path)
    sel = PrimeForCausalLM.from_pretrained_base_to_selective(str(path))
    cpu = torch.device("cpu")
    for i in (0, 2):
        a, b = base.layers[i].self_attn, sel.layers[i].self_attn
        assert torch.equal(a.in_proj.weight, b.in_proj.weight) and torch.equal(a.in_proj.bias, b.in_proj.bias)
        # log(2000) = 7.6 rounded to fp32: 2^-22 of tau
        assert torch.allclose(a.get_tau(cpu), b.get_tau(cpu), rtol=2.0 ** -21, atol=0)
        if min_tau < 10 and max_tau > 250:
            assert torch.equal(a.log_tau, b.log_tau) and (sel.config.min_tau, sel.config.max_tau) == (min_tau, max_tau)
    at = sel.layers[1].self_attn
    lam = torch.exp(-torch.nn.functional.softplus(at.delta_proj.bias) / at.get_tau(cpu))
    assert torch.allclose(lam, torch.full_like(lam, decay), rtol=1e-5)


@pytest.mark.parametrize("width", [1, 2, 64, 1000])
@pytest.mark.parametrize("min_tau,max_tau", [(2.0, 2000.0), (4.0, 1000.0), (2.0, 500.0), (3.0, 3000.0), (1.0, 4096.0),
                                             (0.3, 0.7), (1e-20, 1e30)])
def test_every_tau_begins_with_a_gradient(width, min_tau, max_tau):
    m = GatedLinearRecurrence(8, width=width, min_tau=min_tau, max_tau=max_tau)
    tau = m.get_tau(torch.device("cpu"))
    tau.sum().backward()
    assert torch.allclose(m.log_tau.grad, tau.detach(), rtol=1e-6) and (m.log_tau.grad > 0).all()
    assert tau[0] < min_tau * (1 + 2e-5) and (width == 1 or tau[-1] > max_tau * (1 - 2e-5))


def test_a_range_of_one_tau():
    tau = GatedLinearRecurrence(8, min_tau=5.0, max_tau=5.0).get_tau(torch.device("cpu"))
    assert torch.equal(tau, torch.full((8,), 5.0))


def test_a_block_without_rng_trains():
    """A block of the three-argument form in a model without dropout."""
    class Block(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.proj = torch.nn.Linear(16, 16)

        def forward(self, hidden_states, state=None, return_state=False):
            return hidden_states + self.proj(hidden_states), None
    model = PrimeForCausalLM(PrimeConfig(vocab_size=20, hidden_size=16, num_layers=2, num_heads=1, head_dim=16)).train()
    model.layers[1] = model.layers[0] = Block()
    ids = torch.arange(12).view(2, 6)
    model(ids, labels=ids)["loss"].backward()
    assert model.layers[0].proj.weight.grad.any()


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64, torch.uint16,
                                   torch.uint32, torch.float16, torch.float32])
def test_top_k_of_every_type(dtype):
    """As int32: none below 0, what int32 does not hold as its largest."""
    k = torch.tensor([0, 1, 50, 127]).to(dtype)
    got = _per_row(k, torch.int32, k.device)
    assert got.dtype == torch.int32 and got.tolist() == [0, 1, 50, 127]
    if dtype in (torch.int64, torch.uint32, torch.float32):
        assert _per_row(torch.tensor([4294967040]).to(dtype), torch.int32, k.device).tolist() == [(1 << 31) - 1]
    if dtype.is_signed:
        assert _per_row(torch.tensor([-3]).to(dtype), torch.int32, k.device).item() <= 0


def test_a_config_without_the_new_fields():
    """A configuration of another class, and a block pickled without its place and its dropout."""
    fields = dataclasses.asdict(PrimeConfig(vocab_size=20, hidden_size=16, num_layers=1, num_heads=1, head_dim=16))
    del fields["dropout"], fields["gated_layers"]
    model = PrimeForCausalLM(SimpleNamespace(**fields)).train()
    assert not model.drops_out
    block = model.layers[0]
    del block.layer, block.dropout
    block.self_attn.forward = lambda h, state=None, return_state=False: (h, None)
    ids = torch.arange(12).view(2, 6)
    model(ids, labels=ids)["loss"].backward()
    assert block.mlp.up_proj.weight.grad.any()
