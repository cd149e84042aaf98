"""Plain forms in 64 bits of the embedding, the log probabilities of tokens and the gradient
clipping, and the bounds that their roundings give (not collected: no test_ prefix)."""
import math

import torch

U32 = 2.0 ** -24  # half a step of fp32, relative


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def least(dtype) -> float:
    """Half the distance of the smallest numbers (fp32: below it exp2's results vanish)."""
    return {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126, torch.float32: 2.0 ** -126}[dtype]


def assert_within(got, want, bound, what=""):
    """got against want in 64 bits: equal where want is not finite, else within bound."""
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    bound = torch.as_tensor(bound, dtype=torch.float64).cpu().expand(want.shape)
    assert got.shape == want.shape, f"{what}: shape {tuple(got.shape)}, expected {tuple(want.shape)}"
    fine = torch.isfinite(want)
    odd = ~fine & ~((got == want) | (torch.isnan(got) & torch.isnan(want)))
    assert not odd.any(), f"{what}: {got[odd][:3]} for {want[odd][:3]}"
    over = fine & ~((got - want).abs() <= bound)
    if over.any():
        i = (torch.where(over, (got - want).abs() / bound.clamp(min=1e-300), 0.0)).argmax()
        raise AssertionError(f"{what}: {int(over.sum())} of {want.numel()} off, the worst at {int(i)}: {float(got.flatten()[i])!r} "
                             f"for {float(want.flatten()[i])!r}, bound {float(bound.flatten()[i]):.3g}")


# ---------------------------------------------------------------- embedding

def lookup(ids, weight, scale=1.0):
    """(rows in 64 bits, bound): the product in fp32, then one rounding."""
    w, ids = weight.detach().double().cpu(), ids.long().cpu()
    inside = (ids >= 0) & (ids < w.shape[0])
    out = torch.zeros(*ids.shape, w.shape[1], dtype=torch.float64)
    s = float(torch.tensor(scale, dtype=torch.float32))
    out[inside] = w[ids[inside]] * s
    return out, out.abs() * (half_step(weight.dtype) * (1 + U32) + U32) * (scale != 1.0) + (least(weight.dtype) if scale != 1.0 else 0.0)


def lookup_grad(ids, dy, V, scale=1.0, padding=None):
    """(dweight in 64 bits, bound).  A sum of m terms in fp32, in any order and by parts, is off
    by at most (m - 1) u times the sum of their sizes (to first order; 1.01 covers the rest)."""
    C = dy.shape[-1]
    ids, dy = ids.long().cpu().flatten(), dy.detach().double().cpu().reshape(-1, C)
    takes = (ids >= 0) & (ids < V)
    if padding is not None:
        takes &= ids != padding % V
    at, rows = ids[takes], dy[takes]
    s = float(torch.tensor(scale, dtype=torch.float32))
    grad = torch.zeros(V, C, dtype=torch.float64).index_add_(0, at, rows)
    size = torch.zeros(V, C, dtype=torch.float64).index_add_(0, at, rows.abs())
    m = torch.bincount(at, minlength=V).double().unsqueeze(1)
    return grad * s, lambda dtype: (1.01 * (m + 1) * U32 * size * abs(s) * (1 + half_step(dtype))
                                    + half_step(dtype) * (grad * s).abs() + least(dtype))


# ---------------------------------------------------------------- log probabilities

def row_probs(x):
    """(log p, p) of rows [n, V] in 64 bits, with the operator's rules for rows without a finite
    largest value."""
    x = x.detach().double()
    top = x.amax(1, keepdim=True)
    logp = (x - top) - torch.log(torch.exp(x - top).sum(1, keepdim=True))  # (64 bits lose a log S next to 1e38)
    inf = torch.isinf(x) & (x > 0)
    count = inf.sum(1, keepdim=True).double()
    shared = torch.where(inf, -torch.log(count.clamp(min=1)), -math.inf)
    logp = torch.where(count > 0, shared, logp)
    logp = torch.where(top == -math.inf, -math.inf, logp)
    logp = torch.where(torch.isnan(x).any(1, keepdim=True), math.nan, logp)
    return logp, logp.exp()


def logprobs(x, tokens, ignore=-100):
    """(log probabilities, entropy) [n] of rows [n, V] in 64 bits."""
    logp, p = row_probs(x)
    inside = (tokens >= 0) & (tokens < x.shape[1])
    lp = torch.where(inside, logp.gather(1, torch.where(inside, tokens, 0).unsqueeze(1)).squeeze(1), math.nan)
    lp = torch.where(tokens == ignore, 0.0, lp)
    lp = torch.where(lp < -torch.finfo(torch.float32).max, -math.inf, lp)  # beyond the result's type
    return lp, -torch.where(p == 0, 0.0, p * logp).sum(1)


def ranked(x, top):
    """The `top` first tokens by logit, equal ones by index, NaN as -infinity."""
    x = x.detach().double()
    return torch.where(torch.isnan(x), -math.inf, x).sort(dim=1, descending=True, stable=True).indices[:, :top]


def logprobs_grad(x, tokens, g, h, ignore=-100):
    """d(sum g logprobs + h entropy) / dx in 64 bits (g or h may be None)."""
    logp, p = row_probs(x)
    _, entropy = logprobs(x, tokens, ignore)
    dx = torch.zeros_like(p)
    nothing = (logp == -math.inf).all(1, keepdim=True)
    if g is not None:
        g = torch.where(tokens == ignore, 0.0, g.double())
        inside = (tokens >= 0) & (tokens < x.shape[1])
        g = torch.where(inside | (tokens == ignore), g, math.nan).unsqueeze(1)
        dx = dx - g * p
        dx.scatter_add_(1, torch.where(inside, tokens, 0).unsqueeze(1), torch.where(inside.unsqueeze(1), g, 0.0))
    if h is not None:
        dx = dx - h.double().unsqueeze(1) * torch.where(p == 0, 0.0, p * (logp + entropy.unsqueeze(1)))
    return torch.where(nothing, 0.0, dx)


def row_bounds(x):
    """What the roundings in a row's statistics come to, in units of u = 2^-24.  With d_j the
    distance to the largest logit in powers of 2:
      2^d_j is off by |d_j| ln 2 (d's rounding and that of log2(e)) and 2 (the instruction);
      a sum of V terms by the additions that one term goes through: V / 256 + 32 in a lane (V / 64
        for up to 4096), 16 for rescalings and joins;
      so L = log2 S by  e_L = 1.45 (sum p (2 |d| + 2) + adds) + 4 |L| + 2,
      entropy by        e_H = e_L + 1.45 (sum p |d| (3 |d| + 6 + 2 adds)) + 4 (|L| + sum p |d|) + 4."""
    logp, p = row_probs(x)
    x = x.detach().double()
    V = x.shape[1]
    d = ((x - x.amax(1, keepdim=True)) * math.log2(math.e)).abs()
    d = torch.where(torch.isfinite(d), d, 0.0)
    adds = (V / 64 if V <= 4096 else V / 256) + 48
    mean, square = (p * d).nan_to_num().sum(1), (p * d * d).nan_to_num().sum(1)
    L = -(logp.amax(1) / math.log(2)).nan_to_num(neginf=0.0)
    e_l = 1.45 * (2 * mean + 2 + adds) + 4 * L.abs() + 2
    e_h = e_l + 1.45 * (3 * square + (6 + 2 * adds) * mean) + 4 * (L.abs() + mean) + 4
    return d, e_l, e_h


def logprobs_bound(x, tokens):
    """Bounds of (logprobs, entropy): d_t is off by 2 |d_t|, the difference and the factor by 2
    of the result."""
    d, e_l, e_h = row_bounds(x)
    inside = (tokens >= 0) & (tokens < x.shape[1])
    dt = d.gather(1, torch.where(inside, tokens, 0).unsqueeze(1)).squeeze(1)
    lp, h = (t.nan_to_num(neginf=0.0).abs() for t in logprobs(x, tokens))
    return U32 * (e_l + 2 * dt + 3 * lp + 1), U32 * (e_h + 3 * h + 1)


def grad_bound(x, tokens, g, h, dx, ignore=-100):
    """p is off by (2 |d| + e_L + 4) u, the factors by 4 u each and the entropy in them by e_H."""
    d, e_l, e_h = row_bounds(x)
    logp, p = (t.nan_to_num(neginf=0.0) for t in row_probs(x))
    _, H = (t.nan_to_num() for t in logprobs(x, tokens, ignore))
    zero = torch.zeros(x.shape[0], dtype=torch.float64, device=x.device)
    g = (zero if g is None else torch.where(tokens == ignore, 0.0, g.double())).abs().unsqueeze(1)
    h = (zero if h is None else h.double()).abs().unsqueeze(1)
    size = p * (g + h * (logp.abs() + H.unsqueeze(1)))
    rel = 2 * d + e_l.unsqueeze(1) + 16
    bound = U32 * (size * rel + p * h * (e_h + 2 * e_l).unsqueeze(1) + 4 * g * (p > 0) + 4 * dx.abs().nan_to_num())
    return bound * 1.01 + half_step(x.dtype) * dx.abs().nan_to_num() + least(x.dtype) * (1 + 4 * (g + h))


# ---------------------------------------------------------------- clipping

def clipped(grads, max_norm, norm=None):
    """(norm, the gradients in 64 bits, their bounds): the factor and the product are rounded to
    fp32, then once to the type."""
    if norm is None:
        norm = math.sqrt(sum(float(g.detach().double().square().sum()) for g in grads))
    c = min(1.0, max_norm / (norm + 1e-6))
    want = [g.detach().double() * c for g in grads]
    return norm, want, [w.abs() * (half_step(w0.dtype) + 2.02 * U32) + least(w0.dtype) for w, w0 in zip(want, grads)]
