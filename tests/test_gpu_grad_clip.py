"""The gradient norm over many tensors and clipping by it, against their plain forms in 64 bits."""
import math

import pytest
import torch

import ends_ref as R
from prime_moment_attention import clip_grad_norm_, clip_grads_with_norm_, grad_norm

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def params(grads):
    """Parameters with these gradients, as they are."""
    out = []
    for g in grads:
        p = torch.nn.Parameter(torch.empty(g.shape, device="cuda", dtype=g.dtype))
        p.grad = g
        out.append(p)
    return out


def check(grads, max_norm):
    before = [g.clone() for g in grads]
    ps = params(grads)
    norm, want, bounds = R.clipped(before, max_norm)
    assert abs(float(grad_norm(ps)) - norm) <= 2 * R.U32 * norm
    got = clip_grad_norm_(ps, max_norm)
    assert got.dtype is F32 and got.shape == () and abs(float(got) - norm) <= 2 * R.U32 * norm
    for k, (g, w, b, g0) in enumerate(zip(grads, want, bounds, before)):
        if max_norm >= norm + 1e-6:
            assert torch.equal(g, g0), k
        R.assert_within(g, w, b, f"gradient {k}")
    return got


SHAPES = [[(1,)], [(7,)], [(8,)], [(9,), (1,), (0,), (3, 5)], [(2048,)], [(2049,), (4095,)], [(1000, 33)],
          [(64,)] * 40 + [(128, 128)] * 9, [(700, 1001), (13,), (1 << 20,)], [(17,)] * 191, [(17,)] * 192,
          [(33,)] * 193, [(5, 29)] * 500, [(0,), (0, 4)]]


@pytest.mark.parametrize("dtype", [F32, BF16, F16, "mixed"])
@pytest.mark.parametrize("shapes", SHAPES, ids=lambda s: f"{len(s)}x{'x'.join(map(str, s[0]))}")
def test_sizes(dtype, shapes):
    g = gen(len(shapes))
    kinds = [dtype if dtype != "mixed" else (BF16, F32, F16)[i % 3] for i in range(len(shapes))]
    make = lambda: [torch.randn(s, generator=g, device="cuda").to(k) for s, k in zip(shapes, kinds)]
    check(make(), 0.37)
    check(make(), 1e6)
    check(make(), 0.0)


def test_buckets():
    """Gradients that lie one after the other in one buffer, starting anywhere."""
    for dtype in (F32, BF16, F16):
        sizes = [1, 2, 3, 63, 64, 65, 1000, 4097, 1, 12345, 7]
        buf = torch.randn(sum(sizes) + 9, generator=gen(1), device="cuda").to(dtype)
        guard = buf.clone()
        grads = list(buf[5:-4].split(sizes))
        check(grads, 1.0)
        assert torch.equal(buf[:5], guard[:5]) and torch.equal(buf[-4:], guard[-4:])
        grads = list(buf[5:-4].split(sizes))[::-1]  # from the last to the first
        check(grads, 0.5)


def test_strides():
    """Transposed, permuted and channels-last gradients, columns of a buffer, every other one."""
    base = lambda *s: torch.randn(*s, device="cuda")
    wide = base(40, 90)
    rest = wide.clone()
    check([base(30, 50).t(), base(4, 5, 6).permute(2, 0, 1), base(2, 3, 4, 5).to(memory_format=torch.channels_last),
           wide[:, 10:20], wide[:, 30:45], base(64)[::2], base(9)], 0.7)
    keep = [*range(10), *range(20, 30), *range(45, 90)]
    assert torch.equal(wide[:, keep], rest[:, keep]) and not torch.equal(wide[:, 10:20], rest[:, 10:20])


def test_far_from_one():
    """Squares that fp32 could not hold, or would lose."""
    for size in (1e30, 1e-30, 1e-38):
        check([size * torch.randn(3000, device="cuda"), size * torch.randn(77, device="cuda").bfloat16().float()], size)
    g = torch.full((1000,), 3e38, device="cuda")
    norm = clip_grad_norm_(params([g]), 1.0)  # the norm itself is beyond fp32; the factor is in 64 bits
    assert norm == math.inf and torch.allclose(g, torch.full_like(g, 1000 ** -0.5))
    check([torch.zeros(50, device="cuda")], 1.0)


def test_not_finite():
    for bad in (math.inf, -math.inf, math.nan):
        g = [torch.randn(500, device="cuda"), torch.randn(3, 70, device="cuda").bfloat16()]
        g[1][1, 5] = bad
        twin = [x.clone() for x in g]
        norm = clip_grad_norm_(params(g), 1.0)
        want = torch.nn.utils.clip_grad_norm_(params(twin), 1.0)
        assert norm.isnan() if bad != bad else norm == math.inf
        assert norm.isnan() == want.isnan()
        for a, b in zip(g, twin):
            assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))
    g = torch.tensor([math.inf, 1.0], device="cuda")
    assert clip_grad_norm_(params([g]), math.inf) == math.inf and g[0] == math.inf and g[1] == 1.0


def test_given_norm():
    g = [torch.randn(700, device="cuda"), torch.randn(40, 30, device="cuda").t()]
    before = [x.clone() for x in g]
    norm = grad_norm(params(g))
    all_norm = (norm.square() + 100.0).sqrt()
    clip_grads_with_norm_(params(g), 2.0, all_norm)
    _, want, bounds = R.clipped(before, 2.0, float(all_norm))
    for a, w, b in zip(g, want, bounds):
        R.assert_within(a, w, b)
    clip_grads_with_norm_(params(g), 2.0, torch.ones((), device="cuda"))  # below: nothing happens
    for a, w, b in zip(g, want, bounds):
        R.assert_within(a, w, b)


def test_same_as_torch_on_a_module():
    torch.manual_seed(0)
    m = torch.nn.Sequential(torch.nn.Linear(30, 40), torch.nn.Tanh(), torch.nn.Linear(40, 5)).cuda()
    m(torch.randn(16, 30, device="cuda")).square().sum().backward()
    m[0].bias.grad = None  # passed over
    mine = [None if p.grad is None else p.grad.clone() for p in m.parameters()]
    want = torch.nn.utils.clip_grad_norm_(m.parameters(), 0.5)
    theirs = [p.grad for p in m.parameters()]
    for p, g in zip(m.parameters(), mine):
        p.grad = g
    got = clip_grad_norm_(m.parameters(), 0.5)
    assert torch.allclose(got, want, rtol=1e-6)
    for p, g in zip(m.parameters(), theirs):
        assert (p.grad is None) == (g is None) and (g is None or torch.allclose(p.grad, g, rtol=1e-6))


def test_refusals_on_the_device():
    a = torch.randn(100, device="cuda")
    p = params([a[:60], a[59:]])
    with pytest.raises(RuntimeError, match="overlap"):
        clip_grad_norm_(p, 1.0)
    p = params([a, a])
    with pytest.raises(RuntimeError, match="overlap"):
        clip_grad_norm_(p, 1.0)
    twice = math.sqrt(2) * float(a.double().norm())  # which has a norm all the same
    assert abs(float(grad_norm(p)) - twice) <= 2 * R.U32 * twice
    p = params([a[:1].expand(4, 1)])
    p[0].grad = a[:1].expand(4)[:, None]
    with pytest.raises(ValueError, match="overlaps itself"):
        clip_grad_norm_(p, 1.0)
    twice = 2 * abs(float(a[0]))
    assert abs(float(grad_norm(p)) - twice) <= 2 * R.U32 * twice
    with pytest.raises(RuntimeError, match="dtype"):
        clip_grad_norm_(params([a.double()]), 1.0)
    with pytest.raises(ValueError, match="fp32"):
        clip_grads_with_norm_(params([a]), 1.0, torch.ones((), device="cuda", dtype=torch.float64))
    with pytest.raises(RuntimeError, match="HIP device"):
        clip_grads_with_norm_(params([a]), 1.0, torch.ones(()))


def test_version_of_the_gradients():
    """A graph that saved a gradient notices that clipping changed it."""
    w = torch.randn(20, device="cuda", requires_grad=True)
    g = torch.randn(20, device="cuda")
    p = params([g])
    y = (w * p[0].grad).sum()
    clip_grad_norm_(p, 0.1)
    with pytest.raises(RuntimeError, match="modified"):
        y.backward()


def test_same_bits_every_time_and_streams():
    sets = [[torch.randn(300, 501, device="cuda").bfloat16(), torch.randn(77777, device="cuda")] for _ in range(3)]
    twins = [[g.clone() for g in s] for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    norms = []
    for st, s in zip(streams, sets):
        with torch.cuda.stream(st):
            norms.append(clip_grad_norm_(params(s), 1.0))
    torch.cuda.synchronize()
    for n, s, t in zip(norms, sets, twins):
        assert torch.equal(n, clip_grad_norm_(params(t), 1.0))
        assert all(torch.equal(a, b) for a, b in zip(s, t))


def test_captured_and_replayed():
    g = gen(3)
    grads = [torch.randn(s, generator=g, device="cuda").to(d) for s, d in (((5000,), F32), ((40, 41), BF16), ((3,), F32))]
    ps = params(grads)
    clip_grad_norm_(ps, 1.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip_grad_norm_(ps, 1.0)
    for k in range(4):
        for x in grads:
            x.normal_(generator=g).mul_(10.0 ** (k - 2))
        twins = [x.clone() for x in grads]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, clip_grad_norm_(params(twins), 1.0))
        assert all(torch.equal(a, b) for a, b in zip(grads, twins))


def test_tensor_beyond_32_bits():
    n = (1 << 32) + 12345
    g = torch.ones(n, device="cuda", dtype=BF16)
    g[-1] = 3.0
    p = params([g])
    norm = clip_grad_norm_(p, 2.0 ** 15)
    want = math.sqrt(n - 1 + 9)
    assert abs(float(norm) - want) <= 2 * R.U32 * want
    c = torch.tensor([1.0, 3.0]).double() * (2.0 ** 15 / (want + 1e-6))
    R.assert_within(torch.stack([g[0], g[-1]]), c, c * (2.0 ** -8 + 3 * R.U32))
    assert (g[:-1] == g[0]).all()
