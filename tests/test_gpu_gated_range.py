"""The gated recurrence over the whole range of its numbers, element by element: what a state
keeps after something far larger has been forgotten.

Tolerances, u = 2^-24 a rounding.  A token's a = 2^-z is off by the roundings of z (softplus 4,
log2(e) / tau 2, their product 1, exp2 2), below 9 u (1 + z) of a, its b by 16 u of b; a sum of z
over a tile, a span and a chain of spans has at most 15 + 7 + 15 roundings, each below u of the
sum.  So a term that has come through tokens with decays a is off by at most K u (1 + z) a token,
K = 48, of what is left of it, and a sum of terms by that of their magnitudes: with m_t = a m_{t-1}
+ |b| and m's own error E_t = a (E_{t-1} + K u (1 + z) m_{t-1}) + 16 u |b|, nothing is taken of
the largest value.  The result's own rounding adds u of it.  Decays below 2^-126 may come to 0."""
import pytest
import torch

from gated_ref import STEP_MAX, STEP_MIN, gated_forward
from prime_moment_attention import gated_recurrence

from gpu_util import dev

pytestmark = pytest.mark.gpu

U, K = 2.0 ** -24, 48.0


def magnitudes(a, z, b, start):
    """m_t and E_t as above; start: the magnitude before the first token."""
    m, e, ms, es = start, torch.zeros_like(start), [], []
    for at, zt, bt in zip(a.unbind(1), z.unbind(1), b.abs().unbind(1)):
        e = at * (e + K * U * (1 + zt) * m) + 16 * U * bt
        m = at * m + bt
        ms.append(m), es.append(e)
    return torch.stack(ms, 1), torch.stack(es, 1)


def within(got, ref, bound, what):
    err = (got.detach().double().cpu() - ref.detach()).abs()
    over = err - bound - U * ref.detach().abs() - 1e-30
    at = over.argmax()
    assert torch.isfinite(err).all() and over.max() <= 0, f"{what}: {err.view(-1)[at]:.3e} against {bound.view(-1)[at]:.3e}"


def forgetting(kind, L, C=70):
    """x, step, gate, tau, state, dy, dlast: something large, then quick forgetting."""
    g = torch.Generator().manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=g)
    x, gate, dy = r(2, L, C), r(2, L, C), r(2, L, C)
    tau = torch.where(torch.arange(C) % 2 == 0, 2.0, 7.0)
    step = 1.0 + 0.1 * r(2, L, C)
    state, dlast = r(2, C), r(2, C)
    big = 10.0 ** (3 + 4 * torch.rand(2, C, generator=g))
    if kind == "state":      # a large state, the first token nearly drops it
        state, step[:, 0] = big, 50.0
        dlast, step[:, -1] = big, 50.0
    elif kind == "token":    # large tokens, each dropped at once or by the next ones' steps
        at = range(3, L, 50)
        for t in at:
            x[:, t], dy[:, t] = big, big
            step[:, t + 1 if t + 1 < L else t] = 20.0 + 30.0 * torch.rand(2, C, generator=g)
    elif kind == "steps":    # ordinary steps, over which a whole tile or span forgets
        state, dlast = big, big
        x[:, L // 2], dy[:, L // 2] = big, big
    return x, step, gate, tau, state, dy, dlast


@pytest.mark.parametrize("L", [1, 5, 16, 40, 128, 300, 128 * 20 + 9])
@pytest.mark.parametrize("kind", ["state", "token", "steps"])
def test_what_comes_after_is_kept(kind, L):
    """One token, walked tokens, one tile, part of a span, a span, three spans, and spans past
    a chain head: values, last state and every gradient."""
    args = forgetting(kind, L)
    leaves = [t.to(dev()).requires_grad_() for t in args[:5]]
    y, last = gated_recurrence(*leaves, return_state=True)
    got = torch.autograd.grad([y, last], leaves, [t.to(dev()) for t in args[5:]])
    x, step, gate, tau, state, dy, dlast = (t.double() for t in args)
    ref = [t.clone().requires_grad_() for t in (x, step, gate, tau.expand(x.shape), state)]
    ry, rlast = gated_forward(*ref)
    rg = torch.autograd.grad([ry, rlast], ref, [dy, dlast])

    soft = torch.logaddexp(step, torch.zeros_like(step)).clamp(STEP_MIN, STEP_MAX)
    z = soft / tau / 0.693147
    a, n, s = torch.exp(-soft / tau), (-torch.expm1(-2 * soft / tau)).sqrt(), torch.sigmoid(gate)
    h, eh = magnitudes(a, z, n * s * x, state.abs())
    within(y, ry, eh, "y")
    within(last, rlast, eh[:, -1], "last state")
    # the whole gradient of h_t, and what reaches the state: the same recurrence backwards
    ahead = lambda t: torch.cat([t[:, 1:], torch.zeros_like(t[:, :1])], 1)
    terms = dy.abs()
    terms[:, -1] += dlast.abs()
    G, eG = (t.flip(1) for t in magnitudes(ahead(a).flip(1), ahead(z).flip(1), terms.flip(1), torch.zeros_like(state)))
    within(got[0], rg[0], n * s * (eG + 16 * U * G), "dx")
    within(got[2], rg[2], n * s * (1 - s) * x.abs() * (eG + 16 * U * (1 + gate.abs()) * G), "dgate")
    before = torch.cat([state.abs().unsqueeze(1), h[:, :-1]], 1)
    e_before = torch.cat([torch.zeros_like(state).unsqueeze(1), eh[:, :-1]], 1)
    w, ew = a * (a / n * s * x.abs() + before), a * e_before
    bound = (eG * w + G * (ew + K * U * (1 + z) * w)) / tau
    within(got[1], rg[1], bound, "dstep")
    within(got[3], rg[3].sum((0, 1)), (bound * soft / tau + U * L * rg[3].abs()).sum((0, 1)), "dtau")
    within(got[4], rg[4], a[:, 0] * (eG[:, 0] + K * U * (1 + z[:, 0]) * G[:, 0]), "dstate")


def test_open_gates_keep_their_gradient():
    """dgate = G n x s (1 - s) where 1 - s is far below a rounding of s.  x and dy of one sign,
    so that G has no cancellation.  1 - s = e s with e = exp(-gate): 2 u |gate| of it from the
    exponent; G as a state of 40 tokens.  (Float64's own sigmoid loses 1 - s too: the reference is
    dx x sigmoid(-gate).)"""
    g = torch.Generator().manual_seed(6)
    r = lambda *s: torch.rand(*s, generator=g)
    x, dy, step, tau = 0.5 + r(2, 40, 64), 0.5 + r(2, 40, 64), 4 * r(2, 40, 64) - 2, 2.0 * 1000.0 ** r(64)
    gate = 8.0 + 12.0 * r(2, 40, 64)
    gate[0, ::7], gate[1, ::7] = 60.0, -60.0
    leaves = [t.to(dev()).requires_grad_() for t in (x, step, gate, tau)]
    got = torch.autograd.grad(gated_recurrence(*leaves)[0], leaves[2], dy.to(dev()))[0]
    ref = [t.double().requires_grad_() for t in (x, step, gate, tau)]
    dx, = torch.autograd.grad(gated_forward(*ref)[0], ref[0], dy.double())
    want = (dx * ref[0] * torch.sigmoid(-ref[2])).detach()
    off = ((got.double().cpu() - want) / want).abs()
    assert (off <= U * (64 + 2 * 40 ** 0.5 + 2 * gate.abs())).all(), off.max()


@pytest.mark.parametrize("L", [1, 5, 200])
def test_the_ends_of_tau(L):
    """tau below 1e-30 forgets everything at once (no gradient but in x and gate), tau above
    1e30 nothing, and takes in next to nothing: no infinity comes of either, and no NaN."""
    g = torch.Generator().manual_seed(7)
    r = lambda *s: torch.randn(*s, generator=g)
    tau = torch.tensor([1e-45, 1e-39, 1.2e-38, 1e-31, 1e-29, 1e-20, 1e20, 1e29, 1e33, 1e36, 1e38, 3.4e38])
    C = tau.numel()
    x, step, gate, dy, state, dlast = r(2, L, C), r(2, L, C), r(2, L, C), r(2, L, C), r(2, C), r(2, C)
    step[:, ::3] = -20.0
    leaves = [t.to(dev()).requires_grad_() for t in (x, step, gate, tau, state)]
    y, last = gated_recurrence(*leaves, return_state=True)
    got = [t.double().cpu() for t in torch.autograd.grad([y, last], leaves, [dy.to(dev()), dlast.to(dev())])]
    ref = [t.double().requires_grad_() for t in (x, step, gate, tau, state)]
    ry, rlast = gated_forward(*ref)
    want = torch.autograd.grad([ry, rlast], ref, [dy.double(), dlast.double()])
    for a, b, n in zip([y, last, *got], [ry, rlast, *want], ["y", "last", "dx", "dstep", "dgate", "dtau", "dstate"]):
        a, b = a.detach().double().cpu(), b.detach()
        assert torch.isfinite(a).all(), n
        # n = sqrt(2 D / tau) is below 1e-14 for the large ones: within that of the reference, and of
        # a first-order bound elsewhere
        assert (a - b).abs().max() <= 1e-13 + (64 + 2 * L ** 0.5) * 2 * U * b.abs().max(), n
