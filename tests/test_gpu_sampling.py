"""GPU parity of sample_tokens against the definition in float64, row by row
(tests/gated_ref.py): whole numbers, so every token has to be equal."""
import numpy as np
import pytest
import torch

from gated_ref import sample_row
from prime_moment_attention import sample_tokens

from gpu_util import dev

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
INF = float("inf")


def check(logits, u, **kw):
    """Every row against the reference; numbers or per-row lists as parameters."""
    n = logits.shape[0]
    types = {"temperature": F32, "top_k": torch.int32, "top_p": F32, "min_p": F32}
    on_dev = {k: torch.tensor(v, dtype=types[k], device=dev()) if isinstance(v, (list, np.ndarray)) else v
              for k, v in kw.items()}
    u = torch.as_tensor(u, dtype=F32)
    got = sample_tokens(logits.to(dev()), u.to(dev()), **on_dev).cpu().tolist()
    rows = logits.double().numpy()
    ref = []
    for i in range(n):
        # the parameters as the kernel sees them, rounded to fp32
        at = {k: (float(np.float32(v[i] if isinstance(v, (list, np.ndarray)) else v))) for k, v in kw.items()}
        if "temperature" in at:
            at["T"] = at.pop("temperature")
        if "top_k" in at:
            at["top_k"] = int(at["top_k"])
        ref.append(sample_row(rows[i], float(u[i]), **at))
    assert got == ref
    return got


def make(n, V, dtype, seed, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, V, generator=g) * scale).to(dtype), torch.rand(n, generator=g)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("V", [1, 2, 63, 1024, 1025, 5003, 50304])
def test_cuts(V, dtype):
    logits, u = make(12, V, dtype, V)
    check(logits, u)
    check(logits, u, temperature=0.7, top_k=50)
    check(logits, u, temperature=1.3, top_p=0.9)
    check(logits, u, min_p=0.05)
    check(logits, u, temperature=0.9, top_k=40, top_p=0.8, min_p=0.02)
    rng = np.random.default_rng(V)
    check(logits, u, temperature=rng.uniform(0.2, 2.0, 12), top_k=rng.integers(0, 2 * V + 1, 12),
          top_p=rng.uniform(0.0, 1.1, 12), min_p=rng.uniform(0.0, 0.5, 12))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_equal_logits(dtype):
    """Ties everywhere: the lower index counts as the higher rank."""
    logits = torch.zeros(9, 2000, dtype=dtype)
    u = torch.linspace(0, 0.999, 9)
    check(logits, u)
    check(logits, u, top_k=7)
    check(logits, u, top_p=0.5)
    check(logits, u, top_k=100, top_p=0.25, min_p=1.0)
    few = torch.tensor([0.0, 1.0, 2.0])[torch.randint(0, 3, (9, 2000), generator=torch.Generator().manual_seed(1))]
    for kw in (dict(top_k=900), dict(top_k=1500, top_p=0.7), dict(top_p=0.95), dict(min_p=0.2)):
        check(few.to(dtype), u, **kw)


def test_greedy_and_top_one():
    logits, u = make(6, 3000, BF16, 5)
    logits[:, 100] = logits[:, 2000] = 20.0
    for kw in (dict(temperature=0.0), dict(top_k=1), dict(top_p=0.0), dict(top_p=-1.0), dict(temperature=-1.0)):
        assert check(logits, u, **kw) == [100] * 6
    # min_p of 1 keeps both
    assert set(check(logits, torch.tensor([0.0, 0.2, 0.49, 0.51, 0.7, 0.99]), min_p=1.0)) == {100, 2000}
    assert sample_tokens(logits.to(dev()), u.to(dev()), min_p=2.0).cpu().tolist() == check(logits, u, min_p=1.0)


def test_masked_infinite_and_nan_logits():
    logits, u = make(8, 777, F32, 6)
    logits[0, :] = -INF
    logits[1, :] = float("nan")
    logits[2, :-1] = -INF
    logits[3, ::2] = float("nan")
    logits[4, [5, 600]] = INF
    logits[5, :] = torch.finfo(F32).min
    logits[6, 1:] = torch.finfo(F32).min
    logits[7, :] = torch.finfo(F32).max
    for kw in ({}, dict(top_k=3), dict(top_p=0.5), dict(min_p=0.1), dict(top_k=200, top_p=0.9, min_p=0.01),
               dict(temperature=0.0), dict(temperature=1e-30), dict(temperature=1e30)):
        got = check(logits, u, **kw)
        assert got[2] == 776 and got[3] % 2 == 1 and got[4] in (5, 600) and got[6] == 0


def test_signed_zeros_are_equal():
    logits = torch.full((1, 10), -0.0)
    logits[0, 4] = 0.0
    assert check(logits, [0.5], top_k=1) == [0]


def test_ends_of_the_uniforms():
    """0 takes the first kept token with weight; numbers of 1 and more, which no generator
    gives, the last one; below 0 and NaN count as 0."""
    logits, _ = make(5, 400, F32, 7)
    logits[:, :3] = -INF
    got = sample_tokens(logits.to(dev()), torch.tensor([0.0, 1.0, 2.0, -1.0, float("nan")], device=dev())).tolist()
    assert got == [3, 399, 399, 3, 3]
    check(logits, [0.0, 1 - 2.0 ** -24, 0.5, 2.0 ** -24, 2.0 ** -30], top_k=30)


def test_flat_border_hits():
    """Uniforms that fall exactly on the borders between equal weights."""
    logits = torch.zeros(64, 1024)
    u = torch.arange(64) / 64.0
    assert check(logits, u) == [16 * i for i in range(64)]
    check(logits, u, top_k=512)
    check(logits, u, top_p=0.125)


def test_frequencies_follow_the_softmax():
    logits = torch.tensor([[0.0, 1.0, 2.0, -1.0, 0.5]])
    n = 1 << 16
    u = ((torch.arange(n) + 0.5) / n).to(F32)  # every quantile once: counts are exact to one token a border
    got = sample_tokens(logits.expand(n, 5).to(dev()), u.to(dev()), temperature=0.8).cpu()
    p = torch.softmax(logits[0].double() / 0.8, 0)
    assert ((torch.bincount(got, minlength=5) / n - p).abs() <= 2.0 / n).all()


def test_rows_apart_and_other_columns():
    """Row strides, a view off the vector's boundary, the last token of a sequence's logits."""
    for dtype in (F32, BF16):
        logits, u = make(7, 1003, dtype, 8)
        wide = torch.full((7, 3, 1020), 99.0, dtype=dtype)
        wide[:, -1, 5:1008] = logits
        ref = check(logits, u, top_p=0.9)
        assert sample_tokens(wide.to(dev())[:, -1, 5:1008], u.to(dev()), top_p=0.9).tolist() == ref
        assert sample_tokens(logits.t().contiguous().to(dev()).t(), u.to(dev()), top_p=0.9).tolist() == ref


def test_batch_does_not_change_a_row():
    logits, u = make(300, 2048, BF16, 9)
    a = sample_tokens(logits.to(dev()), u.to(dev()), top_p=0.95, temperature=1.5)
    b = torch.cat([sample_tokens(logits[i:i + 1].to(dev()), u[i:i + 1].to(dev()), top_p=0.95, temperature=1.5)
                   for i in range(0, 300, 37)])
    assert torch.equal(a[::37], b)


@pytest.mark.parametrize("V", [131072, 151936, 1 << 20])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_large_vocabularies(V, dtype):
    logits, u = make(3, V, dtype, 10)
    check(logits, u)
    check(logits, u, top_k=1000, top_p=0.9)
    check(logits, u, top_p=0.97, min_p=1e-4)


def test_out_stream_and_graph():
    logits, u = (t.to(dev()) for t in make(16, 3001, BF16, 11))
    out = torch.zeros(16, 1, dtype=torch.int64, device=dev())
    assert sample_tokens(logits, u, top_k=20, out=out.view(-1)).data_ptr() == out.data_ptr()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = sample_tokens(logits, u, top_k=20)
    s.synchronize()
    assert torch.equal(again, out.view(-1))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        sample_tokens(logits, u, top_k=20, out=out.view(-1))
    for i in range(4):
        a, b = make(16, 3001, BF16, 30 + i)
        logits.copy_(a)
        u.copy_(b)
        g.replay()
        torch.cuda.synchronize()
        got = out.view(-1).clone()
        assert torch.equal(got, sample_tokens(logits, u, top_k=20))


def test_refusals():
    logits, u = (t.to(dev()) for t in make(4, 100, F32, 12))
    with pytest.raises(ValueError, match="uniforms"):
        sample_tokens(logits, u[:2])
    with pytest.raises(ValueError, match="top_p"):
        sample_tokens(logits, u, top_p=torch.ones(3, device=dev()))
    with pytest.raises(ValueError, match="logits"):
        sample_tokens(logits[0], u[:1])
    with pytest.raises(RuntimeError, match="vocab"):
        sample_tokens(torch.zeros(1, (1 << 20) + 1, device=dev()), u[:1])
    assert sample_tokens(logits[:0], u[:0]).shape == (0,)


def test_draws_of_one_row():
    """One row expanded to many, and a top_k beyond 32 bits: all."""
    logits, u = make(1, 5003, BF16, 21)
    u = torch.rand(300, generator=torch.Generator().manual_seed(3))
    got = sample_tokens(logits.to(dev()).expand(300, -1), u.to(dev()), 0.8, top_k=200).tolist()
    assert got == check(logits.expand(300, -1).contiguous(), u, temperature=0.8, top_k=200)
    each = sample_tokens(logits.to(dev()).expand(300, -1), u.to(dev()), 0.8).tolist()
    many = torch.full((300,), (1 << 32) + 5, device=dev())
    for k in ((1 << 32) + 5, -(1 << 32) + 5, many):
        assert sample_tokens(logits.to(dev()).expand(300, -1), u.to(dev()), 0.8, top_k=k).tolist() == each


def test_offsets_past_32_bits():
    V = 5000
    big = torch.zeros((1 << 31) + 2 * V, dtype=BF16, device=dev())
    logits, u = make(2, V, BF16, 13)
    view = big.as_strided((2, V), ((1 << 31) + 100, 1), 7)
    view.copy_(logits)
    assert sample_tokens(view, u.to(dev()), top_p=0.9).tolist() == check(logits, u, top_p=0.9)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("scale", [0.01, 0.5, 1.0, 2.0, 4.0, 30.0])
def test_flat_to_peaked(scale, dtype):
    """From one bucket full of tokens to a handful of them that weigh anything: every way
    through the cuts."""
    logits, u = make(10, 20011, dtype, 14, scale)
    check(logits, u)
    for p in (0.05, 0.5, 0.9, 0.99, 0.9999):
        check(logits, u, top_p=p)
        check(logits, u, top_p=p, min_p=0.01)
    for k in (1, 2, 100, 1000, 1024, 1025, 5000, 20010, 20011):
        check(logits, u, top_k=k)
        check(logits, u, top_k=k, top_p=0.8, temperature=1.7)
    for m in (1e-6, 1e-3, 0.3, 0.999):
        check(logits, u, min_p=m)


@pytest.mark.parametrize("n", [255, 257, 700])
def test_more_rows_than_compute_units(n):
    logits, u = make(n, 4500, BF16, 15)
    rng = np.random.default_rng(n)
    check(logits, u, temperature=rng.uniform(0.3, 2.0, n), top_k=rng.choice([0, 1, 50, 1000, 3000], n),
          top_p=rng.choice([1.0, 0.9, 0.5], n), min_p=rng.choice([0.0, 0.05], n))


def test_ties_through_the_top_k_border():
    """A thousand tokens of one value at the border of every cut."""
    logits = torch.full((6, 3000), -1.0)
    logits[:, 500:520] = 2.0
    logits[:, 1000:2400] = 1.0
    u = torch.tensor([0.0, 0.1, 0.5, 0.9, 0.99, 1 - 2.0 ** -24])
    for kw in (dict(top_k=700), dict(top_k=1400), dict(top_k=21, top_p=0.99), dict(top_p=0.6), dict(top_p=0.9),
               dict(top_k=1420, min_p=0.2), dict(top_k=1421)):
        check(logits, u, **kw)
        check(logits.to(BF16), u, **kw)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V,ks", [(50304, (1000, 1010, 1023, 1024, 1025, 3000)), (4000, (240, 250, 255, 256, 257, 900))])
def test_top_k_near_the_threads(V, ks, dtype):
    """As many kept tokens as a workgroup has threads, and ties that reach past them."""
    logits, u = make(24, V, dtype, V + 2)
    if dtype is F32:
        logits = (logits * 32).round() / 32
    for kw in ({}, {"top_p": 0.93, "min_p": 0.001}):
        check(logits, u, temperature=0.9, top_k=np.array(ks * 4), **kw)


@pytest.mark.parametrize("V", [900, 4000, 40000])
def test_mass_estimates_that_are_off(V):
    """top_p where the heavier tokens lie at the upper ends of equal steps of the logit and
    the lighter ones at the lower ends: what counts alone tell of the masses is off."""
    n = 64
    step = torch.arange(V) * 2000 // V
    for edge in (40, 150, 400):
        x = -(step + torch.where(step < edge, 0.03, 0.97)) * (30.5 / 4094)
        perm = torch.randperm(V, generator=torch.Generator().manual_seed(edge))
        logits = x[perm].expand(n, V).contiguous()
        u = torch.rand(n, generator=torch.Generator().manual_seed(V))
        check(logits, u, top_p=np.linspace(0.02, 0.9999, n))
        check(logits, u, top_p=np.linspace(0.02, 0.9999, n), min_p=0.01)


@pytest.mark.parametrize("T", [1e-38, 1e-6, 1e6, 3e38, INF])
@pytest.mark.parametrize("V", [300, 5003, 50304])
def test_ends_of_the_temperature(V, T):
    logits, u = make(8, V, F32, 5)
    logits[1, ::3] = -INF
    logits[2, ::5] = float("nan")
    logits[3] *= 1e37
    for kw in ({}, {"top_k": 40}, {"top_k": 2000}, {"top_p": 0.7}, {"min_p": 0.5}, {"min_p": 1.0},
               {"top_k": 100, "top_p": 0.9, "min_p": 0.1}):
        check(logits, u, temperature=T, **kw)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("kw", [{}, {"top_k": 60}, {"top_k": 700, "top_p": 0.9}, {"top_p": 0.97}, {"min_p": 0.02}])
def test_a_row_alone_and_among_many(kw, dtype):
    """The launches for few and for many rows of a long vocabulary give the same tokens."""
    logits, u = (t.to(dev()) for t in make(300, 20000, dtype, 31, scale=2.0))
    a = sample_tokens(logits, u, 1.1, **kw)
    for i in range(0, 300, 23):
        assert torch.equal(sample_tokens(logits[i:i + 1], u[i:i + 1], 1.1, **kw), a[i:i + 1])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [16, 272])
def test_top_k_near_the_lanes(n, dtype):
    """As many kept tokens as a wave has lanes, ties around that number among them."""
    logits, u = make(n, 9000, dtype, 33)
    if dtype is F32:
        logits = (logits * 8).round() / 8
    ks = np.resize([1, 2, 60, 62, 63, 64, 65, 66], n)
    check(logits, u, top_k=ks)
    check(logits, u, temperature=1.7, top_k=ks, top_p=0.8)
    check(logits, u, temperature=1.7, top_k=ks, min_p=0.05)


def test_two_streams_at_once():
    logits, u = make(8, 50304, BF16, 16)
    logits, u = logits.to(dev()), u.to(dev())
    want = sample_tokens(logits, u, top_p=0.9)
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(sample_tokens(logits, u, top_p=0.9))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
