"""GPU parity of the gated linear recurrence (gated_recurrence, GatedLinearRecurrence)
against its token-by-token float64 form (tests/gated_ref.py), values and gradients.

Tolerances.  The kernels compute in fp32 from the same inputs.  A gate is off by a few
roundings of 2^-24 and by the exponent's (|s| 2^-24), together below 32 2^-24 for the
inputs here, which moves a state by at most twice that of its largest value; every token
adds one rounding of the state, independent of the others: 2 sqrt(L) of them cover the
sum with a margin of four over its standard deviation.  So F(L) = (64 + 2 sqrt(L)) 2^-24
of the tensor's largest value, plus the result's own rounding, half a step of its type.
A gradient composes two such recurrences: 2 F(L).  dtau sums over tokens: 2 F(L) of the
sum of its terms' magnitudes."""
import math

import pytest
import torch

from gated_ref import gated_forward
from prime_moment_attention import GatedLinearRecurrence, _lib, gated_recurrence

from gpu_util import dev

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def f_tol(L):
    return (64 + 2 * math.sqrt(L)) * 2.0 ** -24


def close(got, ref, tol, scale=None, what=""):
    got, ref = got.detach().double().cpu(), ref.detach().double()
    assert got.shape == ref.shape, what
    assert torch.isfinite(got).all(), what
    return within(got, ref, tol, scale, torch.float64, what)


def within(got, ref, tol, scale, dtype, what):
    half = torch.finfo(dtype).eps / 2
    scale = ref.abs().max() if scale is None else scale
    err = (got - ref).abs() - half * ref.abs() - half * torch.finfo(dtype).smallest_normal
    worst = (err - tol * scale).max()
    assert worst <= 0, f"{what}: {worst:.3e} over (largest error {(got - ref).abs().max():.3e}, scale {scale})"


def check(got, ref, dtype, tol, what, scale=None):
    assert got.dtype == dtype, what
    g = got.detach().double().cpu()
    assert g.shape == ref.shape and torch.isfinite(g).all(), what
    within(g, ref.detach(), tol, scale, dtype, what)


def inputs(B, L, C, dtype, seed, state=True):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    x, step, gate, dy = r(B, L, C), r(B, L, C) * 2 + 0.5, r(B, L, C) * 2, r(B, L, C)
    tau = 2.0 * 1000.0 ** torch.rand(C, generator=g)
    x, step, gate, dy = (t.to(dtype) for t in (x, step, gate, dy))
    return x, step, gate, tau, (r(B, C) if state else None), dy, r(B, C)


def reference(x, step, gate, tau, state, dy, dlast):
    """y, last, gradients, and the sum of magnitudes of dtau's terms."""
    L = [t.double().requires_grad_() for t in (x, step, gate)]
    taus = tau.double().expand(x.shape).clone().requires_grad_()  # one tau per element
    st = state.double().requires_grad_() if state is not None else None
    y, last = gated_forward(*L, taus, st)
    grads = torch.autograd.grad([y, last], [*L, taus] + ([st] if st is not None else []),
                                [dy.double(), dlast.double()])
    return y, last, grads


def run_case(B, L, C, dtype, seed, state, place=lambda t: t):
    x, step, gate, tau, st, dy, dlast = inputs(B, L, C, dtype, seed, state)
    leaves = [place(t.to(dev())).requires_grad_() for t in (x, step, gate)]
    tau_d = tau.to(dev()).requires_grad_()
    st_d = st.to(dev()).requires_grad_() if st is not None else None
    y, last = gated_recurrence(*leaves, tau_d, state=st_d, return_state=True)
    got = torch.autograd.grad([y, last], leaves + [tau_d] + ([st_d] if st is not None else []),
                              [place(dy.to(dev())), dlast.to(dev())])
    with torch.no_grad():
        y0, last0 = gated_recurrence(*leaves, tau_d, state=st_d, return_state=True)
    assert torch.equal(y0, y) and torch.equal(last0, last)
    ry, rlast, rg = reference(x, step, gate, tau, st, dy, dlast)
    t = f_tol(L)
    check(y, ry, dtype, t, "y")
    check(last, rlast, F32, t, "last state")
    for g, r, n in zip(got[:3], rg[:3], ("dx", "dstep", "dgate")):
        check(g, r, dtype, 2 * t, n)
    check(got[3], rg[3].sum((0, 1)), F32, 2 * t, "dtau", scale=rg[3].abs().sum((0, 1)))
    if st is not None:
        check(got[4], rg[4], F32, 2 * t, "dstate")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("B,L,C", [(1, 1, 1), (3, 1, 5), (2, 2, 64), (1, 15, 6), (2, 16, 130), (1, 17, 501),
                                   (5, 100, 33), (2, 333, 256), (1, 1025, 96)])
def test_values_and_gradients(B, L, C, dtype):
    """From one token and one channel to lengths off the 16-token tile and widths off
    every vector, with and without a state."""
    run_case(B, L, C, dtype, 100 + L + C, state=L % 2 == 0 or L == 1)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,L,C", [(1, 5000, 64), (3, 2047, 200), (70, 40, 64)])
def test_split_over_time(B, L, C, dtype):
    """Few long sequences (many segments), and many short ones (one segment)."""
    run_case(B, L, C, dtype, 200 + L, state=True)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("L", [4, 8, 9, 16, 17, 20, 32, 33])
@pytest.mark.parametrize("B", [2, 520])
def test_short_prompts(B, L, dtype):
    """Few tokens of few and of many sequences: walked, or split over a span's waves."""
    run_case(B, L, 250, dtype, L, True)


@pytest.mark.parametrize("B", [1, 5000])
def test_long_memory_keeps_its_value(B):
    """One token of input, then 6,000 with almost no decay: z = 1e-4 / 2000 = 5e-8 lies
    below half a rounding of a = 1, so a form that rounds a would not decay at all, and
    moves h by less than its spacing, so a state without its dropped bits would decay by
    the spacing.  One sequence (segments), and many (one segment each)."""
    L, C = 6000, 64
    x = torch.zeros(1, L, C)
    x[:, 0] = 1.0
    step, gate = torch.full((1, L, C), -20.0), torch.zeros(1, L, C)
    tau, state = torch.full((C,), 2000.0), torch.full((1, C), 3.0)
    if B > 1:
        wide = lambda t: t.to(dev()).expand(B, -1, -1)
        y, last = gated_recurrence(wide(x), wide(step), wide(gate), tau.to(dev()),
                                   state.to(dev()).expand(B, -1).contiguous(), True)
        assert torch.equal(y[0], y[-1]) and torch.equal(last[0], last[-1])
        _, rl = gated_forward(*(t.double() for t in (x, step, gate, tau, state)))
        assert ((3.0 - last[:1].double().cpu()) - (3.0 - rl)).abs().max() < 1e-2 * (3.0 - rl).abs().max()
        return
    y, last = gated_recurrence(*(t.to(dev()) for t in (x, step, gate, tau)), state=state.to(dev()), return_state=True)
    ry, rl = gated_forward(*(t.double() for t in (x, step, gate, tau, state)))
    check(y, ry, F32, f_tol(L), "y")
    # the decay over the whole length, 3 (1 - exp(-3e-4)) = 9e-4, to a part in a hundred
    assert abs((3.0 - last.double().cpu()) - (3.0 - rl)).max() < 1e-2 * (3.0 - rl).abs().max()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("how", ["columns", "odd columns", "transposed", "odd rows"])
def test_strides(how, dtype):
    """Column ranges of one projection, ranges off the vector's boundary, [L, B, C]
    storage, and rows of odd length."""
    def place(t):
        B, L, C = t.shape
        if how == "transposed":
            return t.transpose(0, 1).contiguous().transpose(0, 1)
        wide = t.new_zeros(B, L, 3 * C + 5 if how == "odd rows" else 3 * C + 6)
        o = {"columns": C, "odd columns": C + 1, "odd rows": 1}[how]
        wide[..., o:o + C] = t
        return wide[..., o:o + C]
    run_case(2, 77, 128, dtype, 300, True, lambda t: place(t.detach()))


def test_channels_apart_are_gathered():
    x, step, gate, tau, st, _, _ = inputs(2, 9, 16, F32, 1)
    flip = lambda t: t.to(dev()).transpose(1, 2).contiguous().transpose(1, 2)
    a = gated_recurrence(flip(x), flip(step), flip(gate), tau.to(dev()), st.to(dev()), True)
    b = gated_recurrence(*(t.to(dev()) for t in (x, step, gate, tau, st)), True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_batch_and_upstream_broadcasts():
    """Inputs expanded over the batch (stride 0) and an expanded upstream gradient."""
    x, step, gate, tau, st, dy, _ = inputs(1, 50, 48, F32, 2)
    leaves = [t.to(dev()).requires_grad_() for t in (x, step, gate)]
    tau_d = tau.to(dev()).requires_grad_()
    y, _ = gated_recurrence(*(t.expand(4, -1, -1) for t in leaves), tau_d)
    got = torch.autograd.grad(y.sum(), leaves + [tau_d])
    ones = torch.ones_like(dy)
    _, _, rg = reference(x, step, gate, tau, None, ones, torch.zeros(1, 48))
    for g, r in zip(got[:3], rg[:3]):  # four equal gradients, summed by torch: two more roundings
        check(g, 4 * r, F32, 2 * f_tol(50) + 2 ** -22, "expanded")
    check(got[3], 4 * rg[3].sum((0, 1)), F32, 2 * f_tol(50), "dtau", scale=4 * rg[3].abs().sum((0, 1)))


@pytest.mark.parametrize("only", ["y", "state"])
def test_one_output_used(only):
    x, step, gate, tau, st, dy, dlast = inputs(2, 40, 32, F32, 3)
    leaves = [t.to(dev()).requires_grad_() for t in (x, step, gate, tau, st)]
    y, last = gated_recurrence(*leaves, True)
    got = torch.autograd.grad(y if only == "y" else last, leaves, (dy if only == "y" else dlast).to(dev()))
    zero = torch.zeros_like
    _, _, rg = reference(x, step, gate, tau, st, dy if only == "y" else zero(dy), zero(dlast) if only == "y" else dlast)
    for i in (0, 1, 2, 4):
        check(got[i], rg[i], F32, 2 * f_tol(40), str(i))


def test_clamped_steps_have_no_step_gradient():
    x, step, gate, tau, st, dy, dlast = inputs(1, 32, 16, F32, 4)
    step[..., :8], step[..., 8:] = -30.0, 60.0
    leaves = [t.to(dev()).requires_grad_() for t in (x, step, gate, tau, st)]
    y, last = gated_recurrence(*leaves, True)
    got = torch.autograd.grad([y, last], leaves, [dy.to(dev()), dlast.to(dev())])
    assert not got[1].any()
    ry, _, rg = reference(x, step, gate, tau, st, dy, dlast)
    check(y, ry, F32, f_tol(32), "y")
    check(got[0], rg[0], F32, 2 * f_tol(32), "dx")


@pytest.mark.parametrize("value", [float("inf"), float("nan")])
@pytest.mark.parametrize("where", ["x", "step", "gate"])
def test_non_finite_input_stays_in_its_channel(value, where):
    """What comes before it and the other channels keep their values.  (A step or gate
    of +infinity is a finite gate: clamped, or 1.)"""
    x, step, gate, tau, st, _, _ = inputs(2, 300, 32, F32, 5)
    call = lambda: gated_recurrence(*(t.to(dev()) for t in (x, step, gate, tau, st)), True)
    y0, l0 = call()
    {"x": x, "step": step, "gate": gate}[where][1, 100, 7] = value
    y1, l1 = call()
    same = torch.ones(2, 300, 32, dtype=torch.bool)
    same[1, 100:, 7] = False
    assert torch.equal(y1.cpu()[same], y0.cpu()[same])
    finite = math.isinf(value) and where != "x"
    assert torch.isfinite(y1[1, 100:, 7]).all() == finite and not (torch.isfinite(y1[1, 100:, 7]).any() and not finite)
    assert torch.isfinite(l1[1, 7]).item() == finite


def test_steps_follow_the_prompt():
    """A prompt of 37 tokens at once, and token by token with the state in place.  Within a
    call the state keeps what its roundings drop; between calls it is fp32: at most 37
    roundings of half a step more."""
    x, step, gate, tau, st, _, _ = (t.to(dev()) for t in inputs(3, 37, 96, F32, 6))
    y, last = gated_recurrence(x, step, gate, tau, st, True)
    h = st.clone()
    for t in range(37):
        yt, out = gated_recurrence(x[:, t:t + 1], step[:, t:t + 1], gate[:, t:t + 1], tau, h, True, state_out=h)
        assert out is h and (yt[:, 0] - y[:, t]).abs().max() <= 37 * 2.0 ** -24 * y.abs().max()
    assert (h - last).abs().max() <= 37 * 2.0 ** -24 * y.abs().max()


def test_split_state_in_place():
    x, step, gate, tau, st, _, _ = (t.to(dev()) for t in inputs(1, 4000, 64, F32, 7))
    y, last = gated_recurrence(x, step, gate, tau, st, True)
    h = st.clone()
    y2, _ = gated_recurrence(x, step, gate, tau, h, True, state_out=h)
    assert torch.equal(h, last) and torch.equal(y, y2)


def test_gradient_against_differences():
    """<grad, v> against central differences of the kernel's own forward along v, summed
    in float64: truncation eps^2 / 6 of a third derivative of order one, rounding
    F(L) / eps of the sum's terms; eps = 2^-7 leaves both below 1e-3 of the magnitudes."""
    x, step, gate, tau, st, dy, _ = (t.to(dev()) for t in inputs(2, 60, 32, F32, 8))
    f = lambda *a: (gated_recurrence(*a)[0].double() * dy.double()).sum().item()
    args = [x, step, gate, tau, st]
    leaves = [t.clone().requires_grad_() for t in args]
    grads = torch.autograd.grad(gated_recurrence(*leaves)[0], leaves, dy)
    eps = 2.0 ** -7
    for i, g in enumerate(grads):
        v = torch.sign(g)
        at = lambda s: f(*(t + s * eps * v if j == i else t for j, t in enumerate(args)))
        slope, grad = (at(1) - at(-1)) / (2 * eps), (g.double() * v.double()).sum().item()
        assert abs(slope - grad) < 2e-3 * g.abs().sum().item(), (i, slope, grad)


def test_second_derivative_refused():
    leaves = [t.to(dev()).requires_grad_() for t in inputs(1, 4, 8, F32, 9)[:4]]
    y, _ = gated_recurrence(*leaves)
    g, = torch.autograd.grad(y.sum(), leaves[0], create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_empty():
    z = torch.zeros(2, 0, 8, device=dev())
    y, last = gated_recurrence(z, z, z, torch.ones(8, device=dev()), torch.ones(2, 8, device=dev()), True)
    assert y.shape == (2, 0, 8) and torch.equal(last, torch.ones(2, 8, device=dev()))


def test_another_stream():
    args = [t.to(dev()) for t in inputs(2, 700, 64, BF16, 10)[:5]]
    y, last = gated_recurrence(*args, True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y2, last2 = gated_recurrence(*args, True)
    s.synchronize()
    assert torch.equal(y, y2) and torch.equal(last, last2)


def test_captured_training_step():
    """Forward and backward captured once, replayed on changing inputs with eager work
    between, against the eager gradients."""
    args = [t.to(dev()) for t in inputs(2, 600, 64, F32, 11)]
    x, step, gate, tau, st, dy, dlast = args

    def work():
        leaves = [t.detach().requires_grad_() for t in (x, step, gate, tau, st)]
        y, last = gated_recurrence(*leaves, True)
        return (y.detach(), last.detach(), *torch.autograd.grad([y, last], leaves, [dy, dlast]))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        work()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = work()
    for i in range(4):
        new = inputs(2, 600, 64, F32, 20 + i)
        for t, n in zip(args, new):
            t.copy_(n)
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        for a, b in zip(got, work()):
            assert torch.equal(a, b)


def test_module_matches_its_composition():
    torch.manual_seed(0)
    m = GatedLinearRecurrence(48, width=40).to(dev())
    h = torch.randn(2, 21, 48, device=dev(), requires_grad=True)
    st = torch.randn(2, 40, device=dev(), requires_grad=True)
    out, last = m(h, st, return_state=True)
    grads = torch.autograd.grad([out.sum(), last.sum()], [h, st, *m.parameters()])
    m64 = GatedLinearRecurrence(48, width=40).double()
    m64.load_state_dict({k: v.double().cpu() for k, v in m.state_dict().items()})
    m64.log_tau.data = m.log_tau.data.double().cpu()
    h64, st64 = h.detach().double().cpu().requires_grad_(), st.detach().double().cpu().requires_grad_()
    p = m64.in_proj(h64)
    tau = m64.log_tau.exp().clamp(m64.min_tau, m64.max_tau)
    y, l64 = gated_forward(p[..., :40], p[..., 40:80], p[..., 80:], tau, st64)
    ref = torch.autograd.grad([m64.o_proj(y).sum(), l64.sum()], [h64, st64, *m64.parameters()])
    # two fp32 products of 48 and 40 terms around the recurrence: 2^-24 per term of the
    # magnitudes, at most 100 of them, on top of the recurrence's own
    for g, r, n in zip(grads, ref, ["h", "state"] + [n for n, _ in m.named_parameters()]):
        within(g.double().cpu(), r, 4 * f_tol(21) + 200 * 2.0 ** -24, max(r.abs().max(), 1.0), F32, n)
    with torch.no_grad():
        out2, last2 = m(h, st, return_state=True)
        assert torch.allclose(out2, out, rtol=0, atol=1e-5) and torch.equal(last2, last)
        kept = st.clone()
        m.inplace_state = True
        _, last3 = m(h, kept, return_state=True)
        assert last3 is kept and torch.equal(kept, last)


def test_module_tau_follows_its_parameter():
    """However the parameter is written, behind autograd's back too."""
    m = GatedLinearRecurrence(16).to(dev())
    h = torch.randn(1, 5, 16, device=dev())
    with torch.no_grad():
        a = m(h)[0]
        m.log_tau.add_(0.5)
        b = m(h)[0]
        m.log_tau.data.fill_(3.0)
        c = m(h)[0]
        m.log_tau.data.copy_(GatedLinearRecurrence(16).log_tau)
        d = m(h)[0]
    assert not torch.equal(a, b) and not torch.equal(b, c) and torch.equal(a, d)


def test_infinite_steps_and_gates_act_as_their_limits():
    """step +-infinity as +-1e5 (clamped both), gate +-infinity as +-1e4 (1 and 0): the same
    values, and finite gradients that are 0 there."""
    x, step, gate, tau, st, dy, dlast = inputs(2, 200, 48, F32, 6)
    at = torch.zeros(2, 200, 48, dtype=torch.int64)
    at[0, 3, 5], at[1, 130, 7], at[0, 60, 0], at[1, 199, 47] = 1, 2, 3, 4
    runs = []
    for s, g in ((math.inf, math.inf), (1e5, 1e4)):
        step[at == 1], step[at == 2], gate[at == 3], gate[at == 4] = s, -s, g, -g
        leaves = [t.to(dev()).clone().requires_grad_() for t in (x, step, gate, tau, st)]
        y, last = gated_recurrence(*leaves, True)
        runs.append([y, last, *torch.autograd.grad([y, last], leaves, [dy.to(dev()), dlast.to(dev())])])
    for a, b in zip(*runs):
        assert torch.isfinite(a).all() and torch.equal(a, b)
    dstep, dgate = runs[0][3].cpu(), runs[0][4].cpu()
    assert not dstep[(at == 1) | (at == 2)].any() and not dgate[at > 2].any()


def test_offsets_past_32_bits():
    """Sequences further apart than 2^31 elements, and tokens further apart than 2^27."""
    big = torch.zeros((1 << 31) + (1 << 20), dtype=BF16, device=dev())
    x, step, gate, tau, st, dy, dlast = inputs(2, 10, 64, BF16, 12)

    def apart(t, offset, sb, sl):
        v = big.as_strided(t.shape, (sb, sl, 1), offset)
        return v.copy_(t)
    views = [apart(t, 4096 * i, (1 << 31) + 32768, 256) for i, t in enumerate((x, step, gate))]
    tau_d, st_d = tau.to(dev()), st.to(dev())
    ref = gated_recurrence(*(t.to(dev()) for t in (x, step, gate)), tau_d, st_d, True)
    got = gated_recurrence(*views, tau_d, st_d, True)
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    big.zero_()
    views = [apart(t, 4096 * i, 128, (1 << 27) + 64) for i, t in enumerate((x, step, gate))]
    leaves = [v.detach().requires_grad_() for v in views]
    flat = [t.to(dev()).requires_grad_() for t in (x, step, gate)]
    g = [torch.autograd.grad(gated_recurrence(*l, tau_d, st_d)[0], l, dy.to(dev())) for l in (leaves, flat)]
    assert all(torch.equal(a, b) for a, b in zip(*g))


def test_two_streams_at_once():
    """Split calls that run beside each other, each with its own chain."""
    args = [[t.to(dev()) for t in inputs(1, 9000, 200, F32, 40 + i)[:5]] for i in range(4)]
    want = [gated_recurrence(*a, True) for a in args]
    streams = [torch.cuda.Stream() for _ in args]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for a, s in zip(args, streams):
            with torch.cuda.stream(s):
                got.append(gated_recurrence(*a, True))
    torch.cuda.synchronize()
    for i, (y, last) in enumerate(got):
        assert torch.equal(y, want[i % 4][0]) and torch.equal(last, want[i % 4][1])


def test_same_result_every_time():
    """Many spans in flight: which of them is first does not show."""
    args = [t.to(dev()) for t in inputs(2, 20000, 320, BF16, 50)]
    leaves = [t.detach().requires_grad_() for t in args[:5]]

    def run():
        y, last = gated_recurrence(*leaves, True)
        return (y.detach(), last.detach(), *torch.autograd.grad([y, last], leaves, args[5:]))
    first = run()
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(run(), first))


def test_a_length_of_many_chains():
    """Spans of several chain heads against one segment's reference, state and gradient through all of them."""
    run_case(1, 128 * 35 + 3, 64, F32, 60, True)


def test_retained_graph_backward_twice():
    args = [t.to(dev()) for t in inputs(1, 700, 64, F32, 13)]
    leaves = [t.detach().requires_grad_() for t in args[:5]]
    y, last = gated_recurrence(*leaves, True)
    a = torch.autograd.grad([y, last], leaves, args[5:], retain_graph=True)
    b = torch.autograd.grad([y, last], leaves, args[5:])
    assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_the_same_tensor_in_every_place():
    """x, step and gate one tensor: its gradient is the sum of the three."""
    x, _, _, tau, st, dy, dlast = inputs(2, 50, 64, F32, 14)
    one = x.to(dev()).requires_grad_()
    got, = torch.autograd.grad(gated_recurrence(one, one, one, tau.to(dev()))[0], one, dy.to(dev()))
    _, _, rg = reference(x, x, x, tau, None, dy, torch.zeros_like(dlast))
    check(got, rg[0] + rg[1] + rg[2], F32, 2 * f_tol(50) * 3 + 2 ** -23, "sum")
