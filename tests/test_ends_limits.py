"""CPU checks of what the embedding, the log probabilities and the clipping refuse, and of what
the model leaves to modules of the user's own."""
import pytest
import torch

from prime_moment_attention import PrimeConfig, PrimeForCausalLM, _lib, embedding_lookup, token_logprobs

BIG = (1 << 32) + 5  # 5 in the 32 bits of a C int


def test_sizes_beyond_the_entry_points_are_refused():
    """By views that take no memory: none of them may be cut to 32 bits on the way."""
    one, ids = torch.zeros(1, 1), torch.zeros(3, dtype=torch.int64)
    for C in (BIG, (1 << 20) + 1):
        with pytest.raises(ValueError, match="columns"):
            embedding_lookup(ids, one.expand(2, C))
        with pytest.raises(ValueError, match="columns"):
            _lib.embedding(ids, one.expand(2, C), 1.0, one.expand(3, C))
        with pytest.raises(ValueError, match="columns"):
            _lib.embedding_backward(torch.zeros(0, dtype=torch.uint8), one.expand(3, C), 1.0, one.expand(2, C))
    for n, vocab in ((BIG, 1), (1 << 31, 1), (1, BIG), (1, (1 << 24) + 1)):
        x, t = one.expand(n, vocab), ids[:1].expand(n)
        with pytest.raises(ValueError, match="rows"):
            token_logprobs(x, t)
        with pytest.raises(ValueError, match="rows"):
            _lib.token_logprobs(x, t, -100, one, None, None, 0, None, None)
        with pytest.raises(ValueError, match="rows"):
            _lib.token_logprobs_backward(x, t, -100, one, None, one, None, x)
    with pytest.raises(RuntimeError, match="HIP device"):  # the largest sizes go on to the next check
        token_logprobs(one.expand(1, 1 << 24), ids[:1])
    with pytest.raises(RuntimeError, match="HIP device"):
        embedding_lookup(ids, one.expand(2, 1 << 20))


def test_embedding_refuses_a_padding_that_is_no_id():
    """-1 is none; 2^32 + 5 was id 5 to few tokens and none to many."""
    L, at = _lib.load(), [(i + 1) << 28 for i in range(4)]

    def call(padding, order=at[3], n=8, V=100, out=at[2]):
        return L.prime_embedding(at[0], 1, n, at[1], 64, V, 64, _lib.PRIME_BF16, 1.0, padding, out, order,
                                 L.prime_embedding_order_size(n, V), None)
    for n in (8, 40000):
        for padding in (-2, -100, 100, 1 << 31, (1 << 32) + 5, -(1 << 32) + 5):
            assert call(padding, n=n) == -1 and "padding" in _lib.last_error()
            assert call(padding, order=None, n=n) == -1
        for padding in (-1, 0, 99):  # these go on to the next check
            assert call(padding, n=n, out=at[1]) == -5


def _watch(module, name, calls):
    """Registers what the module's call is watched by under `name`; returns what takes it away."""
    seen = lambda *a: calls.append(name)
    if name.startswith("global"):
        return getattr(torch.nn.modules.module, "register_module_" + name[7:])(seen)
    if name == "forward":
        plain = module.forward
        module.forward = lambda ids: (seen(), plain(ids))[1]
        return None
    return getattr(module, "register_" + name)(seen)


@pytest.mark.parametrize("name", ["forward", "forward_hook", "forward_pre_hook", "full_backward_hook", "full_backward_pre_hook",
                                  "global forward_hook", "global forward_pre_hook", "global full_backward_hook",
                                  "global full_backward_pre_hook"])
@pytest.mark.parametrize("how", [dict(fused_training=True), dict(embedding_scale=2.0)])
def test_a_watched_embedding_is_called(name, how):
    model = PrimeForCausalLM(PrimeConfig(vocab_size=11, hidden_size=8, num_layers=1, num_heads=1, head_dim=8, **how))
    ids, calls = torch.tensor([[1, 10, 1]]), []
    handle = _watch(model.embed_tokens, name, calls)
    try:
        x = model._embed(ids)
        assert torch.equal(x, model.embed_tokens.weight[ids] * model.embedding_scale)
        x.sum().backward()
    finally:
        if handle is not None:
            handle.remove()
    assert name in calls


def test_a_replaced_class_forward_of_embeddings_is_called(monkeypatch):
    model = PrimeForCausalLM(PrimeConfig(vocab_size=11, hidden_size=8, num_layers=1, num_heads=1, head_dim=8,
                                         fused_training=True))
    monkeypatch.setattr(torch.nn.Embedding, "forward", lambda self, ids: 3 * self.weight[ids])
    ids = torch.tensor([[1, 10, 1]])
    assert torch.equal(model._embed(ids), 3 * model.embed_tokens.weight[ids])


def test_an_embedding_as_it_is_goes_to_the_kernel():
    model = PrimeForCausalLM(PrimeConfig(vocab_size=11, hidden_size=8, num_layers=1, num_heads=1, head_dim=8,
                                         fused_training=True))
    with pytest.raises(RuntimeError, match="HIP device"):
        model._embed(torch.tensor([[1, 10, 1]]))
