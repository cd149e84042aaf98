"""What the backward passes of the embedding and of the log probabilities keep: as saved tensors,
that hooks see, that are freed by the backward, and that come back as they were or are refused."""
import pytest
import torch
import torch.utils.checkpoint

from prime_moment_attention import _lib, embedding_lookup, token_logprobs

pytestmark = pytest.mark.gpu


def embedding_step(n=40000, V=900, C=24):
    w = torch.randn(V, C, device="cuda", requires_grad=True)
    ids = torch.randint(0, V, (n,), device="cuda")
    dy = torch.randn(n, C, device="cuda")
    return w, lambda: embedding_lookup(ids, w, 2.0), lambda y: torch.autograd.grad(y, w, dy)[0]


def logprobs_step(n=37, V=1003):
    x = torch.randn(n, V, device="cuda", requires_grad=True)
    t, g = torch.randint(0, V, (n,), device="cuda"), torch.randn(n, device="cuda")
    return x, lambda: token_logprobs(x, t, entropy=True), lambda r: torch.autograd.grad([r.logprobs, r.entropy], x, [g, g])[0]


STEPS = [embedding_step, logprobs_step]


@pytest.mark.parametrize("make", STEPS)
def test_a_second_backward_needs_a_retained_graph(make):
    _, forward, backward = make()
    out = forward()
    backward(out)
    with pytest.raises(RuntimeError, match="second time"):
        backward(out)


@pytest.mark.parametrize("make", STEPS)
def test_freed_by_the_backward_while_the_output_lives(make):
    sizes = dict(n=1 << 20, C=1) if make is embedding_step else dict(n=1 << 20, V=2)
    _, forward, backward = make(**sizes)
    backward(forward())
    before = torch.cuda.memory_allocated()
    out = forward()
    outputs = [out] if torch.is_tensor(out) else [t for t in out if t is not None]
    kept = sum(t.numel() * t.element_size() for t in outputs)
    grad = backward(out)
    del grad
    assert torch.cuda.memory_allocated() - before <= kept + (1 << 16)
    del out, outputs
    assert torch.cuda.memory_allocated() == before


@pytest.mark.parametrize("make, least", [(embedding_step, 8 * 40000), (logprobs_step, 37 * (1003 * 4 + 8 + 4 + 8))])
def test_hooks_see_all_of_it(make, least):
    _, forward, backward = make()
    want = backward(forward())
    sizes = []

    def pack(t):
        sizes.append(t.numel() * t.element_size())
        return t.cpu()

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t.cuda()):
        out = forward()
    assert sum(sizes) >= least
    full = [torch.full((s,), 255, dtype=torch.uint8, device="cuda") for s in sizes for _ in range(4)]
    del full
    assert torch.equal(backward(out), want)


OTHERS = {"on the host": lambda t: t.cpu(), "of another type": lambda t: t.to(torch.float16),
          "shorter": lambda t: t.flatten()[:-1].clone(), "with gaps": lambda t: t.repeat_interleave(2, -1)[..., ::2]}


@pytest.mark.parametrize("kind", OTHERS)
@pytest.mark.parametrize("make, count", [(embedding_step, 1), (logprobs_step, 4)])
def test_what_comes_back_otherwise_is_refused(make, count, kind):
    """Each saved tensor in turn.  (The logits may have gaps: their rows are found again.)"""
    _, forward, backward = make()
    want = backward(forward())
    for which in range(count):
        packed = []

        def pack(t):
            packed.append(None)
            return len(packed) - 1, t

        def unpack(held):
            at, t = held
            return OTHERS[kind](t) if at == which else t

        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            out = forward()
        assert len(packed) == count
        if count == 4 and which == 0 and kind == "with gaps":
            assert torch.equal(backward(out), want)
            continue
        with pytest.raises(RuntimeError, match="came back"):
            backward(out)


@pytest.mark.parametrize("reentrant", [True, False])
@pytest.mark.parametrize("make", STEPS)
def test_recomputed_by_a_checkpoint(make, reentrant):
    leaf, forward, backward = make()
    total = lambda out: out.square().sum() if torch.is_tensor(out) else out.logprobs.square().sum() + out.entropy.square().sum()
    want, = torch.autograd.grad(total(forward()), leaf)
    torch.utils.checkpoint.checkpoint(lambda _: total(forward()), leaf, use_reentrant=reentrant).backward()
    assert torch.equal(leaf.grad, want)


def test_an_order_with_room_for_more_tokens():
    """A buffer that is kept for the largest batch serves smaller ones."""
    V, C = 300, 20
    room = _lib.embedding_order(30000, V, "cuda")
    w = torch.randn(V, C, device="cuda", requires_grad=True)
    for n in (7, 3000, 30000):
        ids, dy = torch.randint(0, V, (n,), device="cuda"), torch.randn(n, C, device="cuda")
        _lib.embedding(ids, w.detach(), 1.0, torch.empty(n, C, device="cuda"), -1, room)
        got = torch.empty(V, C, device="cuda")
        _lib.embedding_backward(room, dy, 1.0, got)
        assert torch.equal(got, torch.autograd.grad(embedding_lookup(ids, w), w, dy)[0])
