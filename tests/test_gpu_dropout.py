"""GPU parity of dropout_add against its definition, Philox4x32-10 in Python integers
and the sum in float64.  x / (1 - p) is one fp32 product and one fp32 sum before the
rounding: 2 2^-24 of the magnitudes, and half a step of the type."""
import pytest
import torch

from gated_ref import keep_mask, philox_words
from prime_moment_attention import dropout_add, dropout_rng

from gpu_util import dev

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def rng_of(seed, offset):
    return torch.tensor([seed, offset], dtype=torch.int64, device=dev())


def reference(x, residual, p, seed, offset, call):
    keep, scale = keep_mask(x.numel(), p, seed, offset, call)
    y = torch.where(torch.from_numpy(keep).view(x.shape), x.double().cpu() * scale, 0.0)
    return y if residual is None else y + residual.double().cpu()


def check(got, ref, x, residual, scale=2.0):
    half = torch.finfo(got.dtype).eps / 2
    mag = x.double().cpu().abs() * scale + (0 if residual is None else residual.double().cpu().abs())
    bound = half * (ref.abs() + 4 * 2.0 ** -24 * mag + torch.finfo(got.dtype).smallest_normal) + 2 * 2.0 ** -24 * mag
    assert got.shape == ref.shape and ((got.double().cpu() - ref).abs() <= bound).all()


def test_known_answers():
    """The paper's known-answer vectors of Philox4x32-10."""
    assert philox_words(0, 0, 0) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones = (1 << 64) - 1
    assert philox_words(ones, ones, ones) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (3, 5), (2, 3, 64), (33, 501), (4, 9, 768)])
@pytest.mark.parametrize("p", [0.1, 0.5])
def test_values_and_gradients(shape, dtype, p):
    g = torch.Generator().manual_seed(len(shape))
    x, r, dy = (torch.randn(*shape, generator=g).to(dtype).to(dev()) for _ in range(3))
    seed, offset, call = -5, (1 << 63) - 2, 9  # the counter passes 2^63, the key is negative
    for res in (None, r):
        xg = x.clone().requires_grad_()
        rg = None if res is None else res.clone().requires_grad_()
        y = dropout_add(xg, rg, p, rng_of(seed, offset), call)
        check(y.detach(), reference(x, res, p, seed, offset, call), x, res)
        got = torch.autograd.grad(y, [xg] + ([] if res is None else [rg]), dy)
        check(got[0], reference(dy, None, p, seed, offset, call), dy, None)
        if res is not None:
            assert torch.equal(got[1], dy)
        with torch.no_grad():
            assert torch.equal(dropout_add(x, res, p, rng_of(seed, offset), call), y)


@pytest.mark.parametrize("p,what", [(0.0, "all"), (1.0, "none"), (1e-6, "all"), (1 - 1e-6, "none")])
def test_ends_of_p(p, what):
    x, r = torch.randn(40, 100, device=dev()), torch.randn(40, 100, device=dev())
    y = dropout_add(x, r, p, rng_of(1, 2))
    assert torch.equal(y, x + r if what == "all" else r)


def test_dropped_infinity_leaves_zero():
    x = torch.full((4096,), float("inf"), device=dev())
    y = dropout_add(x, None, 0.5, rng_of(3, 4))
    keep = torch.from_numpy(keep_mask(4096, 0.5, 3, 4, 0)[0])
    assert torch.equal(y.cpu(), torch.where(keep, float("inf"), 0.0))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_do_not_change_the_mask(dtype):
    x, r = (torch.randn(6, 40, 64, device=dev()).to(dtype) for _ in range(2))
    y = dropout_add(x, r, 0.3, rng_of(5, 6))
    wide = torch.zeros(6, 40, 203, device=dev(), dtype=dtype)
    wide[..., 67:131] = x
    assert torch.equal(dropout_add(wide[..., 67:131], r, 0.3, rng_of(5, 6)), y)
    assert torch.equal(dropout_add(x, wide[..., 67:131], 0.3, rng_of(5, 6)), dropout_add(x, x, 0.3, rng_of(5, 6)))
    t = x.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(dropout_add(t, r, 0.3, rng_of(5, 6)), y)
    e = x[:1].expand(6, -1, -1)
    assert torch.equal(dropout_add(e, r, 0.3, rng_of(5, 6)), dropout_add(e.contiguous(), r, 0.3, rng_of(5, 6)))
    f = x.transpose(1, 2)
    assert torch.equal(dropout_add(f, None, 0.3, rng_of(5, 6)), dropout_add(f.contiguous(), None, 0.3, rng_of(5, 6)))


def test_calls_and_offsets_differ_and_shares_are_p():
    x = torch.ones(1 << 20, device=dev())
    a, b, c = (dropout_add(x, None, 0.25, rng_of(7, o), k) for o, k in ((0, 0), (0, 1), (1, 0)))
    assert torch.equal(b, c) and not torch.equal(a, b)
    for t in (a, b):  # 2^20 coins: five standard deviations are 5 sqrt(0.1875 / 2^20) = 0.0021
        assert abs((t == 0).double().mean().item() - 0.25) < 0.0022
    both = ((a == 0) & (b == 0)).double().mean().item()
    assert abs(both - 0.0625) < 5 * (0.0625 / 2 ** 20) ** 0.5


def test_rng_changed_before_the_backward_is_refused():
    x = torch.randn(100, device=dev(), requires_grad=True)
    rng = rng_of(1, 1)
    y = dropout_add(x, None, 0.5, rng)
    rng += 1
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


def test_captured_step_draws_anew():
    x = torch.randn(500, 96, device=dev(), requires_grad=True)
    rng = rng_of(11, 0)

    def work():
        y = dropout_add(x, None, 0.4, rng.clone(), 3)
        return y.detach(), torch.autograd.grad(y, x, torch.ones_like(y))[0]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        work()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = work()
    seen = []
    for i in range(4):
        rng.copy_(torch.tensor([11, i]))
        g.replay()
        torch.cuda.synchronize()
        seen.append(outs[0].clone())
        for a, b in zip([t.clone() for t in outs], work()):
            assert torch.equal(a, b)
    assert not torch.equal(seen[0], seen[1])


def test_rng_repeats_with_the_seed():
    torch.manual_seed(4)
    a = dropout_rng(dev())
    torch.manual_seed(4)
    assert torch.equal(a, dropout_rng(dev())) and a.dtype == torch.int64 and a.shape == (2,)


def test_refusals():
    x = torch.zeros(4, 8, device=dev())
    with pytest.raises(ValueError, match="outside"):
        dropout_add(x, None, 1.5, rng_of(0, 0))
    with pytest.raises(ValueError, match="residual"):
        dropout_add(x, x[:2], 0.1, rng_of(0, 0))
    with pytest.raises(ValueError, match="rng"):
        dropout_add(x, None, 0.1, torch.zeros(2, device=dev()))
    assert dropout_add(x[:0], None, 0.1, rng_of(0, 0)).shape == (0, 8)


def test_more_than_32_bits_of_elements():
    """The elements behind 2^31 have their own bits, and so do the last ones of a ragged end."""
    n = (1 << 31) + 8 * 1000 + 5
    x = torch.ones(n, dtype=BF16, device=dev())
    y = dropout_add(x, None, 0.5, rng_of(21, 22))
    del x
    for block in (0, (1 << 28) - 1, 1 << 28, (1 << 28) + 999, (1 << 28) + 1000):
        words = philox_words(block, 22, 21)
        bits = [h for w in words for h in (w & 0xFFFF, w >> 16)]
        got = y[8 * block:8 * block + 8].cpu()
        assert got.tolist() == [2.0 if b >= 32768 else 0.0 for b in bits[:got.numel()]]


def test_expanded_gradient_and_same_tensor_twice():
    x = torch.randn(12, 40, device=dev(), requires_grad=True)
    y = dropout_add(x, x, 0.3, rng_of(1, 9))
    g, = torch.autograd.grad(y.sum(), x)  # the upstream gradient is one number, expanded
    keep, scale = keep_mask(480, 0.3, 1, 9, 0)
    want = 1 + torch.from_numpy(keep * scale).view(12, 40)
    assert (g.double().cpu() - want).abs().max() <= 4 * 2.0 ** -24 * 3


def test_create_graph_once():
    """First gradients with create_graph are had; a second derivative is refused."""
    x = torch.randn(100, device=dev(), requires_grad=True)
    g, = torch.autograd.grad(dropout_add(x, None, 0.3, rng_of(1, 9)).sum(), x, create_graph=True)
    assert torch.isfinite(g).all()
    with pytest.raises(RuntimeError):
        g.sum().backward()
