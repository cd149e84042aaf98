"""The embedding, the log probabilities and the clipping together, as a language model's
training step, its scoring and its decoding use them."""
import math

import pytest
import torch
import torch.nn.functional as F

import ends_ref as R
from gated_ref import gated_forward
from prime_moment_attention import (GreedyDecoder, PrimeConfig, PrimeForCausalLM, SamplingDecoder, clip_grad_norm_,
                                    token_logprobs)

from gpu_util import dev

pytestmark = pytest.mark.gpu


def model_of(dtype=torch.float32, seed=0, layers=2, gated=(0, 1), **kw):
    torch.manual_seed(seed)
    cfg = dict(vocab_size=130, hidden_size=64, num_layers=layers, num_heads=2, head_dim=32, gated_layers=gated,
               initializer_range=0.1)
    return PrimeForCausalLM(PrimeConfig(**{**cfg, **kw})).to(dev(), dtype)


def loss64(model, ids, labels):
    """The loss of a model of gated layers in float64 on the CPU, and its parameters."""
    cfg = model.config
    w = {n: p.detach().double().cpu().requires_grad_() for n, p in model.named_parameters()}
    rms = lambda t, n: t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + cfg.rms_norm_eps) * w[n]
    x = w["embed_tokens.weight"][ids] * cfg.embedding_scale
    for i in range(cfg.num_layers):
        p = f"layers.{i}."
        proj = rms(x, p + "input_layernorm.weight") @ w[p + "self_attn.in_proj.weight"].t() + w[p + "self_attn.in_proj.bias"]
        W = proj.shape[-1] // 3
        tau = w[p + "self_attn.log_tau"].exp().clamp(cfg.min_tau, cfg.max_tau)
        y, _ = gated_forward(proj[..., :W], proj[..., W:2 * W], proj[..., 2 * W:], tau)
        x = x + y @ w[p + "self_attn.o_proj.weight"].t()
        n = rms(x, p + "post_attention_layernorm.weight")
        x = x + (F.silu(n @ w[p + "mlp.gate_proj.weight"].t()) * (n @ w[p + "mlp.up_proj.weight"].t())) @ w[p + "mlp.down_proj.weight"].t()
    head = w.get("lm_head.weight", w["embed_tokens.weight"])
    logits = rms(x, "norm.weight") @ head.t()
    return F.cross_entropy(logits[:, :-1].reshape(-1, cfg.vocab_size), labels[:, 1:].reshape(-1)), w


@pytest.mark.parametrize("tied", [True, False])
@pytest.mark.parametrize("max_norm", [0.05, 100.0])
def test_training_step(tied, max_norm):
    """Loss, norm and every clipped gradient.  fp32 products of at most 192 terms, 2 layers of 8
    products and norms each way: 2^-24 a rounding, below 2^-24 (192 + 64) 8 of a gradient's largest
    value, with room for the norms' cancellations: 2^-11."""
    model = model_of(fused_training=True, embedding_scale=3.5, tie_word_embeddings=tied).train()
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(0, 130, (3, 41), generator=g)
    labels = torch.where(torch.rand(3, 41, generator=g) < 0.2, -100, ids)
    out = model(ids.to(dev()), labels=labels.to(dev()))
    loss, w = loss64(model, ids, labels)
    assert abs(float(out["loss"].detach()) - float(loss.detach())) <= 2.0 ** -16 * abs(float(loss.detach()))
    out["loss"].backward()
    loss.backward()
    want = math.sqrt(sum(float(t.grad.square().sum()) for t in w.values()))
    norm = model.clip_grad_norm_(max_norm)
    assert abs(float(norm) - want) <= 2.0 ** -11 * want
    c = min(1.0, max_norm / (want + 1e-6))
    for n, p in model.named_parameters():
        ref = w[n].grad * c
        assert (p.grad.double().cpu() - ref).abs().max() <= 2.0 ** -11 * ref.abs().max(), n


def test_fused_and_plain_losses_agree():
    """The two ways to a loss: one model, bf16 and fp32, moment attention too.  The logits are the
    same; the loss's sums of at most 2^8 values differ by their fp32 roundings."""
    for dtype, gated in ((torch.float32, ()), (torch.bfloat16, (1,))):
        plain = model_of(dtype, gated=gated, num_heads=1, head_dim=64)
        fused = model_of(dtype, gated=gated, num_heads=1, head_dim=64, fused_training=True)
        ids = torch.randint(0, 130, (2, 70), device=dev())
        for grad in (True, False):
            with torch.set_grad_enabled(grad):
                a, b = plain(ids, labels=ids), fused(ids, labels=ids)
            assert torch.equal(a["logits"], b["logits"])
            assert abs(float(a["loss"].detach()) - float(b["loss"].detach())) <= 2.0 ** -16 * float(a["loss"].detach())
        assert plain(ids, labels=torch.full_like(ids, -100))["loss"].isnan()
        assert fused(ids, labels=torch.full_like(ids, -100))["loss"].isnan()
        one = fused(ids[:, :1], labels=ids[:, :1])["loss"]
        assert one.isnan()
        with torch.no_grad():
            assert fused(ids[:, :1], labels=ids[:, :1])["loss"].isnan()


def test_embedding_scale_in_every_path():
    """Scaled by a power of two, a model is that with the table so scaled, bit for bit: the graph
    for training, the prefill, the functional step, the fused steps of both decoders."""
    kinds = [dict(dtype=torch.float32, gated=(1,), num_heads=1, head_dim=64),
             dict(dtype=torch.bfloat16, gated=(), hidden_size=256, num_heads=4, head_dim=64, mlp_type="gelu",
                  intermediate_size=512, vocab_size=160)]
    for kw in kinds:
        a = model_of(tie_word_embeddings=False, embedding_scale=4.0, **kw)
        b = model_of(tie_word_embeddings=False, **kw)
        with torch.no_grad():
            b.embed_tokens.weight.mul_(4.0)
        ids = torch.randint(0, 130, (3, 20), device=dev())
        assert torch.equal(a(ids)["logits"], b(ids)["logits"])
        with torch.no_grad():
            x, y = a(ids, return_states=True), b(ids, return_states=True)
            assert torch.equal(x["logits"], y["logits"])
            assert torch.equal(a(ids[:, :1], states=x["states"])["logits"], b(ids[:, :1], states=y["states"])["logits"])
        assert torch.equal(a.generate(ids, 5, temperature=0.0), b.generate(ids, 5, temperature=0.0))
        assert torch.equal(GreedyDecoder(a).generate(ids, 6), GreedyDecoder(b).generate(ids, 6))
        assert torch.equal(GreedyDecoder(a).generate(ids, 6), a.generate(ids, 6, temperature=0.0))


def test_modules_of_the_users_own_are_called():
    class Doubled(torch.nn.Embedding):
        def forward(self, ids):
            return 2 * super().forward(ids)
    model = model_of(fused_training=True, tie_word_embeddings=False, embedding_scale=0.5)
    ids = torch.randint(0, 130, (2, 9), device=dev())
    table = model.embed_tokens.weight
    assert torch.equal(model._embed(ids), table[ids] * 0.5)
    own = Doubled(130, 64).to(dev())
    with torch.no_grad():
        own.weight.copy_(table)
    model.set_input_embeddings(own)
    assert torch.equal(model._embed(ids), table[ids])
    model.set_input_embeddings(torch.nn.Embedding(130, 64, padding_idx=3).to(dev()))
    model(ids.clamp(min=3), labels=ids)["loss"].backward()
    assert (model.embed_tokens.weight.grad[3] == 0).all() and model.embed_tokens.weight.grad.abs().sum() > 0


def test_score():
    """Of every token after the ones before it: what the logits say of it."""
    for dtype in (torch.float32, torch.bfloat16):
        model = model_of(dtype)
        ids = torch.randint(0, 130, (3, 17), device=dev())
        r = model.score(ids, top=4, entropy=True)
        with torch.no_grad():
            logits = model(ids)["logits"][:, :-1].reshape(-1, 130)
        next_ids = ids[:, 1:].reshape(-1)
        lp, ent = R.logprobs(logits, next_ids)
        bound, bound_h = R.logprobs_bound(logits, next_ids)
        R.assert_within(r.logprobs.reshape(-1), lp, bound)
        R.assert_within(r.entropy.reshape(-1), ent, bound_h)
        assert r.top_tokens.shape == (3, 16, 4) and torch.equal(r.top_tokens.reshape(-1, 4), R.ranked(logits, 4))
        assert model.score(ids[:, :1]).logprobs.shape == (3, 0)
    model = model_of(dropout=0.1).train()
    with pytest.raises(ValueError, match="eval"):
        model.score(ids)


@pytest.mark.parametrize("use_graph", [False, True])
def test_decoder_with_log_probabilities(use_graph):
    """Each sampled token's log probability and alternatives are those of the logits it was drawn
    from, captured or not."""
    model = model_of()
    ids = torch.randint(0, 130, (3, 12), device=dev())
    decoder = SamplingDecoder(model, temperature=0.8, top_k=20, generator=torch.Generator(dev()).manual_seed(5),
                              use_graph=use_graph, logprobs=3)
    text, token = ids, decoder.prefill(ids)
    for _ in range(4):
        token = token.clone()
        with torch.no_grad():
            logits = model(text)["logits"][:, -1]
        lp, _ = R.logprobs(logits, token.view(-1))
        # the step's logits come from the recurrent form: fp32 sums in another order
        assert (decoder.logprobs.logprobs.double() - lp).abs().max() < 1e-4
        assert decoder.logprobs.top_tokens.shape == (3, 3)
        best, _ = R.logprobs(logits, decoder.logprobs.top_tokens[:, 0])
        assert (decoder.logprobs.top_logprobs[:, 0].double() - best).abs().max() < 1e-4
        assert (best - R.logprobs(logits, logits.argmax(1))[0]).abs().max() < 1e-4
        text = torch.cat([text, token], 1)
        token = decoder.step()
    plain = SamplingDecoder(model, temperature=0.8, top_k=20, generator=torch.Generator(dev()).manual_seed(5),
                            use_graph=use_graph)
    assert torch.equal(plain.generate(ids, 5)[:, :16], text) and plain.logprobs is None


def test_captured_training_step():
    """Forward, backward and clipping in one graph, replayed with new texts, eager work between."""
    model = model_of(fused_training=True, embedding_scale=2.0).train()
    ids = torch.randint(0, 130, (40, 50), device=dev())  # more tokens than one sum takes
    params = list(model.parameters())

    def step():
        loss = model(ids, labels=ids)["loss"]
        grads = torch.autograd.grad(loss, params)
        for p, g in zip(params, grads):
            p.grad = g
        return loss.detach(), model.clip_grad_norm_(0.1), grads

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, norm, grads = step()
    for _ in range(4):
        ids.random_(0, 130)
        graph.replay()
        torch.cuda.synchronize()
        got = [loss.clone(), norm.clone(), *[g.clone() for g in grads]]
        want_loss, want_norm, want = step()
        for a, b in zip(got, (want_loss, want_norm, *want)):
            # (the products' sums may be split otherwise while a graph is captured)
            assert (a - b).abs().max() <= 2.0 ** -16 * b.abs().max()


def test_steps_with_everything_on():
    """A few steps of plain descent run with everything on, and leave finite weights."""
    model = model_of(torch.bfloat16, gated=(0,), num_heads=1, head_dim=64, fused_training=True, dropout=0.1).train()
    ids = torch.randint(0, 130, (4, 33), device=dev())
    for _ in range(3):
        model.zero_grad()
        model(ids, labels=ids)["loss"].backward()
        norm = clip_grad_norm_(model.parameters(), 1.0)
        assert norm.isfinite() and norm > 0
        with torch.no_grad():
            for p in model.parameters():
                p.sub_(0.01 * p.grad)
    assert all(p.isfinite().all() for p in model.parameters())


def test_warm_start_keeps_the_fields(tmp_path):
    model = model_of(gated=(), num_heads=1, head_dim=64, embedding_scale=2.0, fused_training=True)
    path = str(tmp_path / "base.pt")
    torch.save({"config": model.config, "model_state_dict": model.state_dict()}, path)
    warm = PrimeForCausalLM.from_pretrained_base_to_selective(path, device=dev())
    assert warm.config.embedding_scale == 2.0 and warm.config.fused_training and warm.config.use_selective


def test_loss_of_rows_of_a_batch():
    """The mean of what token_logprobs gives is the loss, whatever the rows' views."""
    logits = torch.randn(3, 30, 200, device=dev())
    labels = torch.randint(0, 200, (3, 30), device=dev())
    lp = token_logprobs(logits[:, :-1], labels[:, 1:]).logprobs
    want = F.cross_entropy(logits[:, :-1].reshape(-1, 200).double(), labels[:, 1:].reshape(-1))
    assert abs(float(-lp.mean()) - float(want)) < 1e-5
