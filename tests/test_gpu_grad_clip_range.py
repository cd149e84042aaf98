"""Clipping by a norm beyond fp32, whatever the number of tensors."""
import math

import pytest
import torch

import ends_ref as R
from prime_moment_attention import clip_grad_norm_, clip_grads_with_norm_, grad_norm
from test_gpu_grad_clip import params

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("count", [1, 2, 192, 193, 400, 700])
def test_the_factor_does_not_depend_on_the_number_of_tensors(count):
    """The same 8400 numbers in one tensor or in many: their squares beyond fp32, or below it, or
    the norm itself beyond it."""
    g = torch.Generator(device="cuda").manual_seed(count)
    for size, max_norm in ((1e30, 1.0), (1.0, 0.3), (1e-30, 1e-31), (3e38, 1e38), (3e38, 1e4)):
        flat = size * (0.5 + 0.5 * torch.rand(8400, generator=g, device="cuda"))
        grads = list(flat.clone().split(8400 // count))
        norm, want, bounds = R.clipped([flat], max_norm)
        got = clip_grad_norm_(params(grads), max_norm)
        if norm > torch.finfo(torch.float32).max:
            assert got == math.inf
        else:
            assert abs(float(got) - norm) <= 2 * R.U32 * norm
        R.assert_within(torch.cat(grads), want[0], bounds[0], f"{size}")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_factors_below_fp32s_normal_numbers(dtype):
    """A norm above 2^126 times the limit: as a single fp32 number the factor would have lost bits."""
    for count, size, max_norm in ((9000, 3e38, 1.0), (9000, 3e38, 1e-3), (10, 3e38, 1e-4), (9000, 1e38, 1e-6), (4099, 2e38, 30.0),
                                  (9000, 1e-3, 1e-33), (300, 3e38, 1e9)):
        g = (size * (0.5 + 0.5 * torch.rand(count, device="cuda"))).to(dtype)
        g[::7] = 0.0
        g[1::7] = 1.0
        for parts in (1, 250):
            mine = g.clone()
            norm, want, bounds = R.clipped([g], max_norm)
            clip_grad_norm_(params(list(mine.split(-(-count // parts)))), max_norm)
            R.assert_within(mine, want[0], bounds[0], f"{count} of {size}")


def test_not_finite_in_many_tensors():
    for bad in (math.inf, math.nan):
        grads = [torch.ones(3, device="cuda") for _ in range(200)]
        grads[7][1] = bad
        norm = clip_grad_norm_(params(grads), 1.0)
        assert norm == math.inf or (bad != bad and norm.isnan())
        want = 0.0 if bad == math.inf else math.nan
        for k, x in enumerate(grads):
            w = torch.full((3,), want, device="cuda")
            if k == 7:
                w[1] = math.nan
            assert torch.equal(x.nan_to_num(7.0), w.nan_to_num(7.0)), k


def test_a_given_norm_is_fp32():
    """An infinite one gives 0, as its caller has nothing better."""
    grads = [torch.full((1000,), 3e38, device="cuda")]
    norm = grad_norm(params(grads))
    assert norm == math.inf
    clip_grads_with_norm_(params(grads), 1.0, norm)
    assert (grads[0] == 0).all()


def test_captured_with_many_tensors():
    grads = [torch.randn(5, device="cuda") for _ in range(200)]
    ps = params(grads)
    clip_grad_norm_(ps, 1.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip_grad_norm_(ps, 1.0)
    for k in range(4):
        for x in grads:
            x.normal_().mul_(10.0 ** (12 * k))
        twins = [x.clone() for x in grads]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, clip_grad_norm_(params(twins), 1.0))
        assert all(torch.equal(a, b) for a, b in zip(grads, twins))
