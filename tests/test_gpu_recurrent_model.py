"""The gated recurrence, dropout and the sampler together, as a language model uses them:
a training step against a float64 composition of the same model, and decoding."""
import math

import pytest
import torch
import torch.nn.functional as F

from gated_ref import gated_forward, keep_mask, sample_row
from prime_moment_attention import (GatedLinearRecurrence, GreedyDecoder, PrimeConfig, PrimeForCausalLM,
                                    SamplingDecoder, dropout_rng)

from gpu_util import dev

pytestmark = pytest.mark.gpu


def model_of(gated, dropout=0.0, dtype=torch.float32, layers=2, seed=0, **kw):
    torch.manual_seed(seed)
    cfg = PrimeConfig(vocab_size=120, hidden_size=64, num_layers=layers, num_heads=2, head_dim=32, dropout=dropout,
                      gated_layers=gated, initializer_range=0.1, **kw)
    return PrimeForCausalLM(cfg).to(dev(), dtype)


def loss64(model, ids, rng):
    """The loss of a model of gated layers only, in float64 on the CPU, with the dropout
    masks of rng; and the parameters to differentiate in."""
    cfg = model.config
    w = {n: p.detach().double().cpu().requires_grad_() for n, p in model.named_parameters()}
    seed, offset = rng.tolist()
    rms = lambda t, n: t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + cfg.rms_norm_eps) * w[n]

    def drop(h, x, call):
        keep, scale = keep_mask(h.numel(), cfg.dropout, seed, offset, call)
        return x + h * torch.from_numpy(keep * scale).view(h.shape)
    x = w["embed_tokens.weight"][ids]
    for i in range(cfg.num_layers):
        p = f"layers.{i}."
        proj = rms(x, p + "input_layernorm.weight") @ w[p + "self_attn.in_proj.weight"].t() + w[p + "self_attn.in_proj.bias"]
        W = proj.shape[-1] // 3
        tau = w[p + "self_attn.log_tau"].exp().clamp(cfg.min_tau, cfg.max_tau)
        y, _ = gated_forward(proj[..., :W], proj[..., W:2 * W], proj[..., 2 * W:], tau)
        x = drop(y @ w[p + "self_attn.o_proj.weight"].t(), x, 2 * i)
        n = rms(x, p + "post_attention_layernorm.weight")
        m = F.silu(n @ w[p + "mlp.gate_proj.weight"].t()) * (n @ w[p + "mlp.up_proj.weight"].t())
        x = drop(m @ w[p + "mlp.down_proj.weight"].t(), x, 2 * i + 1)
    logits = rms(x, "norm.weight") @ w["embed_tokens.weight"].t()
    return F.cross_entropy(logits[:, :-1].reshape(-1, cfg.vocab_size), ids[:, 1:].reshape(-1)), w


@pytest.mark.parametrize("dropout", [0.0, 0.25])
def test_training_step(dropout):
    """Loss and every gradient.  fp32 products of at most 192 terms, 2 layers of 8 products
    and norms each way: 2^-24 a rounding, below 2^-24 (192 + 64) 8 of a gradient's largest
    value, with room for the norms' cancellations: 2^-11."""
    model = model_of((0, 1), dropout).train()
    ids = torch.randint(0, 120, (3, 41), generator=torch.Generator().manual_seed(1))
    torch.manual_seed(7)
    rng = dropout_rng(dev())
    torch.manual_seed(7)
    out = model(ids.to(dev()), labels=ids.to(dev()))
    out["loss"].backward()
    ref, w = loss64(model, ids, rng)
    ref.backward()
    assert abs(out["loss"].item() - ref.item()) < 1e-5
    for n, p in model.named_parameters():
        g, r = p.grad.double().cpu(), w[n].grad
        assert (g - r).abs().max() <= 2.0 ** -11 * r.abs().max(), n


def test_dropout_applies_in_training_only_and_repeats_with_the_seed():
    model = model_of((0,), 0.3).train()
    ids = torch.randint(0, 120, (2, 20), device=dev())
    def run():
        with torch.no_grad():
            return model(ids)["logits"]
    torch.manual_seed(3)
    a, b = run(), run()
    torch.manual_seed(3)
    assert torch.equal(a, run()) and not torch.equal(a, b)
    model.eval()
    assert torch.equal(run(), run())


def test_standalone_block_draws_its_own_mask():
    model = model_of((0,), 0.3).train()
    x = torch.randn(2, 9, 64, device=dev())
    torch.manual_seed(1)
    a, _ = model.layers[0](x)
    b, _ = model.layers[0](x)
    assert not torch.equal(a, b)


def test_refused_configurations():
    with pytest.raises(ValueError, match="dropout"):
        PrimeConfig(dropout=1.5)
    with pytest.raises(ValueError, match="gated_layers"):
        PrimeConfig(num_layers=2, gated_layers=(2,))


@pytest.mark.parametrize("gated", [(0, 1), (1,)])
@pytest.mark.parametrize("mlp", ["swiglu", "gelu"])
def test_steps_follow_the_prompt(gated, mlp):
    """Logits of a prompt at once and token by token, moment layers beside gated ones.
    (The moment layers' own paths agree to 1e-4 of the logits in fp32.)"""
    model = model_of(gated, mlp_type=mlp).eval()
    assert isinstance(model.layers[1].self_attn, GatedLinearRecurrence)
    ids = torch.randint(0, 120, (3, 12), device=dev())
    with torch.no_grad():
        whole = model(ids, return_states=True)
        states, steps = None, []
        for t in range(12):
            out = model(ids[:, t:t + 1], states=states, return_states=True)
            states = out["states"]
            steps.append(out["logits"])
    got = torch.cat(steps, 1)
    assert (got - whole["logits"]).abs().max() < 1e-3 * whole["logits"].abs().max()
    assert states[1].shape == (3, 64) and states[1].dtype == torch.float32


@pytest.mark.parametrize("gated", [(), (1,)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_greedy_decoder(gated, dtype):
    model = model_of(gated, dtype=dtype).eval()
    ids = torch.randint(0, 120, (4, 10), device=dev())
    with torch.no_grad():
        want = model.generate(ids, 8, temperature=0.0)
    for graph in (False, True):
        assert torch.equal(GreedyDecoder(model, use_graph=graph).generate(ids, 8), want)


def test_decoders_refuse_a_model_that_drops_out():
    """A decoder puts its model into eval mode; back in training it is refused."""
    model = model_of((1,), dropout=0.2)
    ids = torch.randint(0, 120, (2, 5), device=dev())
    for d in (GreedyDecoder(model), SamplingDecoder(model)):
        model.train()
        with pytest.raises(ValueError, match="eval"):
            d.generate(ids, 3)
    assert GreedyDecoder(model.eval()).generate(ids, 3).shape == (2, 8)


@pytest.mark.parametrize("gated", [(), (0, 1), (1,)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sampling_decoder(gated, dtype):
    """Eager, captured and generate give the same tokens from the same generator; each is
    the reference's choice for the logits it was drawn from."""
    model = model_of(gated, dtype=dtype, seed=2).eval()
    ids = torch.randint(0, 120, (4, 10), device=dev())
    gen = lambda: torch.Generator(device=dev()).manual_seed(11)
    runs = [SamplingDecoder(model, 0.9, 30, 0.95, 0.01, gen(), use_graph=g).generate(ids, 10) for g in (False, True)]
    assert torch.equal(runs[0], runs[1])
    with torch.no_grad():
        assert torch.equal(model.generate(ids, 10, 0.9, 30, top_p=0.95, min_p=0.01, generator=gen()), runs[0])
        logits = model(ids, logits_to_keep=1)["logits"][:, -1].double().cpu().numpy()
    u = torch.rand(4, device=dev(), generator=gen()).cpu()
    f = lambda v: torch.tensor(v, dtype=torch.float32).item()
    want = [sample_row(logits[i], u[i].item(), f(0.9), 30, f(0.95), f(0.01)) for i in range(4)]
    assert runs[0][:, 10].tolist() == want
    # longer runs: another generator, other tokens
    other = SamplingDecoder(model, 1.5, 0, 1.0, 0.0, torch.Generator(device=dev()).manual_seed(5)).generate(ids, 10)
    assert not torch.equal(other, runs[0])


def test_sampling_decoder_cuts_per_sequence():
    """One request greedy, one sampled, one with its own top_k: the greedy one equals the
    greedy decoder's."""
    model = model_of((1,), seed=3).eval()
    ids = torch.randint(0, 120, (3, 7), device=dev())
    d = SamplingDecoder(model, torch.tensor([0.0, 1.2, 1.0]), torch.tensor([0, 0, 1]),
                        generator=torch.Generator(device=dev()).manual_seed(1))
    got, greedy = d.generate(ids, 9), GreedyDecoder(model).generate(ids, 9)
    assert torch.equal(got[0], greedy[0]) and torch.equal(got[2], greedy[2]) and not torch.equal(got[1], greedy[1])


def test_generate_without_the_new_arguments_is_torch_multinomial():
    model = model_of(()).eval()
    ids = torch.randint(0, 120, (2, 5), device=dev())
    torch.manual_seed(4)
    got = model.generate(ids, 1, temperature=0.8, top_k=20)
    torch.manual_seed(4)
    with torch.no_grad():
        logits = model(ids, logits_to_keep=1)["logits"][:, -1] / 0.8
    v, _ = torch.topk(logits, 20)
    logits[logits < v[:, [-1]]] = -math.inf
    assert torch.equal(got[:, 5:], torch.multinomial(torch.softmax(logits, -1), 1))
