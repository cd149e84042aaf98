"""Log probabilities of tokens, entropy, alternatives and gradients, against their plain forms
in 64 bits."""
import contextlib
import math

import pytest
import torch

import ends_ref as R
from prime_moment_attention import _lib, token_logprobs

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
INF, NAN = math.inf, math.nan


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def check(x, tokens, top=0, entropy=True, g=None, h=None, ignore=-100):
    """Forward with everything asked for and with nothing but the log probabilities, and the
    gradients for g and h."""
    n, V = x.shape
    r = token_logprobs(x, tokens, top=top, entropy=entropy, ignore_index=ignore)
    want, want_h = R.logprobs(x, tokens, ignore)
    bound, bound_h = R.logprobs_bound(x, tokens)
    R.assert_within(r.logprobs, want, bound, "logprobs")
    R.assert_within(token_logprobs(x, tokens, ignore_index=ignore).logprobs, want, bound, "logprobs alone")
    if entropy:
        R.assert_within(r.entropy, want_h, bound_h, "entropy")
    if top:
        order = R.ranked(x, top)
        assert torch.equal(r.top_tokens, order), "top tokens"
        for k in range(top):
            lp, _ = R.logprobs(x, order[:, k], -1)  # (no token is -1)
            R.assert_within(r.top_logprobs[:, k], lp, R.logprobs_bound(x, order[:, k])[0], f"top {k}")
    else:
        assert r.top_tokens is None and r.top_logprobs is None
    if g is None and h is None:
        return r
    leaf = x.detach().requires_grad_()
    r = token_logprobs(leaf, tokens, top=top, entropy=h is not None, ignore_index=ignore)
    R.assert_within(r.logprobs, want, bound, "logprobs in training")
    outs, grads = zip(*[(o, d) for o, d in ((r.logprobs, g), (r.entropy, h)) if d is not None])
    dx, = torch.autograd.grad(outs, leaf, grads)
    want = R.logprobs_grad(x, tokens, g, h, ignore)
    assert dx.dtype is x.dtype
    R.assert_within(dx, want, R.grad_bound(x, tokens, g, h, want, ignore), "gradient")
    return r


SIZES = [(1, 1, 1), (1, 2, 2), (3, 7, 7), (5, 8, 8), (4, 9, 1), (4, 63, 20), (2, 257, 64), (9, 1025, 5), (7, 2048, 10),
         (3, 2049, 20), (2, 4099, 64), (513, 2100, 3), (1, 50304, 20), (2, 50257, 5), (1, 160001, 10), (520, 5001, 0)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n, V, top", SIZES)
def test_sizes(dtype, n, V, top):
    g = gen(n + V)
    x = (torch.randn(n, V, generator=g, device="cuda") * (1 + 3 * torch.rand(n, 1, generator=g, device="cuda"))).to(dtype)
    tokens = torch.randint(0, V, (n,), generator=g, device="cuda")
    tokens[::3] = x[::3].float().argmax(1)
    a, b = torch.randn(2, n, generator=g, device="cuda")
    check(x, tokens, top, True, a, b)
    check(x, tokens, 0, False, a)
    check(x, tokens, 0, True, None, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [5, 100, 2048, 3001, 20000])
def test_rows_out_of_the_ordinary(dtype, V):
    """Banned tokens, rows of nothing but -infinity, the type's lowest value as a mask, rows of
    it alone, its largest, infinities, NaN, equal logits, one token far above the rest."""
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    x = torch.randn(20, V, generator=gen(V), device="cuda").to(dtype)
    x[0, 1:] = -INF
    x[1] = -INF
    x[2, :-1] = low
    x[3] = low
    x[4, : V // 2] = -INF
    x[5, 2] = INF
    x[6, 1:4] = INF
    x[7, 3] = NAN
    x[8] = 2.5
    x[9] = 0.0
    x[9, 1::2] = -0.0
    x[10] = high
    x[11, 2], x[11, 3] = high, low
    x[12] = -INF
    x[12, 4] = low
    x[13] = -INF
    x[13, 1], x[13, 2] = NAN, INF
    x[14, 3] += 60.0
    x[15] = -INF
    x[15, 0] = INF
    x[16] *= 1e3
    x[17] = torch.arange(V, device="cuda").to(dtype) * (-1 if V < 3000 else 1)
    x[18] = -INF
    x[18, 2], x[18, 4] = NAN, 1.0
    x[19, 1:] = low / 2
    g = torch.randn(20, device="cuda")
    for tokens in (torch.full((20,), 3, device="cuda"), torch.full((20,), 0, device="cuda"),
                   torch.arange(20, device="cuda") % 5):
        check(x, tokens, min(V, 20), True, g, 0.3 * g + 1)
        check(x, tokens, 1, True, g)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [600, 2048, 3000, 16385, 50304])
def test_alternatives_where_they_are_hard_to_tell(dtype, V):
    """Sorted rows, neighbours that are the largest, coarse and equal logits, ties that reach over
    the last place, few tokens that are not banned."""
    g = gen(V)
    rows = []
    x = torch.randn(V, generator=g, device="cuda")
    rows += [x.sort().values, x.sort(descending=True).values, torch.round(x), torch.round(4 * x), x.clamp(max=1.0)]
    y = x.clone()
    y[V // 3:V // 3 + 70] = 9.0 + torch.rand(70, generator=g, device="cuda")
    rows.append(y)
    y = x.clone()
    y[::8] += 20.0  # one element of each vector
    rows.append(y)
    y = x.clone()
    y[V - 300:] += 20.0
    rows.append(y)
    for count in (1, 3, 19, 63, 64, 200):
        y = torch.full((V,), -INF, device="cuda")
        at = torch.randperm(V, generator=g, device="cuda")[:count]
        y[at] = x[at]
        rows.append(y)
    y = torch.zeros(V, device="cuda")
    y[torch.randperm(V, generator=g, device="cuda")[:10]] = 1.0
    rows += [y, -y, torch.full((V,), -0.0, device="cuda")]
    for step in (7, 64, 1024):  # the largest all in the same lanes
        y = x.clone()
        y[5::step] = 30.0 + x[5::step]
        rows.append(y)
    x = torch.stack(rows).to(dtype)
    tokens = torch.zeros(len(rows), dtype=torch.int64, device="cuda")
    for top in (1, 5, 20, 64):
        r = token_logprobs(x, tokens, top=top)
        assert torch.equal(r.top_tokens, R.ranked(x, top)), top
        many = x.repeat(30, 1)
        assert torch.equal(token_logprobs(many, tokens.repeat(30), top=top).top_tokens, r.top_tokens.repeat(30, 1))


def test_tokens_that_do_not_count():
    x = torch.randn(6, 3000, device="cuda")
    tokens = torch.tensor([3, -100, 2999, 3000, -1, -100], device="cuda")
    g, h = torch.randn(2, 6, device="cuda")
    check(x, tokens, 2, True, g, h)
    check(x, tokens, 0, False, g)
    check(x[:3], tokens[:3] * 0 - 7, 0, True, g[:3], None, ignore=-7)
    r = check(x, torch.full((6,), -100, device="cuda"), 0, True, g, h)
    assert (r.logprobs == 0).all()
    check(x, torch.full((6,), 5, device="cuda"), 0, True, g, h, ignore=5)  # a token of the vocabulary
    y = x.clone()
    y[1], y[5] = NAN, -INF  # rows that do not count give no gradient whatever is in them
    y.requires_grad_()
    dx, = torch.autograd.grad(token_logprobs(y, tokens).logprobs, y, g)
    assert (dx[[1, 5]] == 0).all() and dx[3:5].isnan().all() and dx[[0, 2]].isfinite().all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [70, 2501])
def test_views(dtype, V):
    """Rows that start anywhere, wide and zero strides, a vocabulary that is not contiguous,
    batches of more dimensions, int32 tokens, broadcast gradients."""
    gg = gen(V)
    wide = torch.randn(4, 6, V + 9, generator=gg, device="cuda").to(dtype)
    tokens = torch.randint(0, V, (4, 6), generator=gg, device="cuda")
    flat = lambda t: t.reshape(-1, V)
    for at in (0, 1, 3, 9):
        x = wide[..., at:at + V]
        r = token_logprobs(x, tokens, top=3, entropy=True)
        s = token_logprobs(flat(x).contiguous(), tokens.flatten(), top=3, entropy=True)
        assert r.logprobs.shape == (4, 6) and r.entropy.shape == (4, 6) and r.top_tokens.shape == (4, 6, 3)
        for a, b in zip(r, s):
            assert torch.equal(a.flatten(), b.flatten())
        g = torch.randn(24, generator=gg, device="cuda")
        check(x[1], tokens[1], 2, True, g[:6], g[6:12])
        check(x[:, 2], tokens[:, 2], 2, True, g[:4], g[4:8])
    x = wide[..., :V]
    assert torch.equal(token_logprobs(x, tokens.int()).logprobs, token_logprobs(x, tokens).logprobs)
    turned = torch.randn(V, 5, generator=gg, device="cuda").to(dtype).t()
    check(turned, tokens.flatten()[:5], 4, True, g[:5], g[5:10])
    check(x[0, :1].expand(6, V), tokens[0], 3, True)
    one = x[0, 0]
    assert token_logprobs(one, tokens[0, 0], top=2).top_tokens.shape == (2,)
    leaf = x[:, :-1].detach().requires_grad_()  # the shifted logits of a loss: rows of two strides
    lp = token_logprobs(leaf, tokens[:, 1:]).logprobs
    dx, = torch.autograd.grad(lp.sum(), leaf)
    want = R.logprobs_grad(flat(x[:, :-1]), tokens[:, 1:].flatten(), torch.ones(20, device="cuda"), None)
    ones = torch.ones(20, device="cuda")
    R.assert_within(flat(dx), want, R.grad_bound(flat(x[:, :-1]), tokens[:, 1:].flatten(), ones, None, want))
    row = x[0, :1].detach().clone().requires_grad_()  # the gradient of a broadcast row is their sum
    dx, = torch.autograd.grad(token_logprobs(row.expand(6, V), tokens[0]).logprobs.sum(), row)
    each = R.logprobs_grad(row.expand(6, V), tokens[0], ones[:6], None)
    bound = R.grad_bound(row.expand(6, V), tokens[0], ones[:6], None, each)
    bound = bound.sum(0) + 8 * R.half_step(dtype) * each.abs().sum(0)  # torch adds six rows of dtype
    R.assert_within(dx[0], each.sum(0), bound)


def test_nothing_to_do():
    x = torch.randn(0, 9, device="cuda").requires_grad_()
    r = token_logprobs(x, torch.zeros(0, dtype=torch.int64, device="cuda"), top=2, entropy=True)
    assert r.logprobs.shape == (0,) and r.entropy.shape == (0,) and r.top_tokens.shape == (0, 2)
    dx, = torch.autograd.grad(r.logprobs.sum() + r.entropy.sum(), x)
    assert dx.shape == (0, 9)


def test_gradient_against_differences():
    """Of the plain form in 64 bits: (f(x + e) - f(x - e)) / 2 e, off by e^2 f''' / 6 (below
    1e-9 here) and the rounding of f over e (1e-10)."""
    g = gen(9)
    x = torch.randn(2, 40, generator=g, device="cuda").double()
    tokens = torch.tensor([4, 39], device="cuda")
    a, b = torch.randn(2, 2, generator=g, device="cuda")
    x = x.float()
    leaf = x.clone().requires_grad_()
    r = token_logprobs(leaf, tokens, entropy=True)
    dx, = torch.autograd.grad([r.logprobs, r.entropy], leaf, [a, b])
    e = 1e-5
    for i in range(2):
        for j in range(40):
            f = []
            for s in (e, -e):
                y = x.double()
                y[i, j] += s
                lp, h = R.logprobs(y, tokens)
                f.append(float((a.double() * lp + b.double() * h).sum()))
            bound = R.grad_bound(x, tokens, a, b, dx.double())[i, j]
            assert abs((f[0] - f[1]) / (2 * e) - float(dx[i, j])) <= 2e-9 + float(bound)


def test_cross_entropy_of_a_loss():
    x = torch.randn(50, 4000, device="cuda").requires_grad_()
    t = torch.randint(0, 4000, (50,), device="cuda")
    t[::7] = -100
    loss = -token_logprobs(x, t).logprobs.sum() / (t != -100).sum()
    want = torch.nn.functional.cross_entropy(x.double(), t)
    assert abs(float(loss.detach()) - float(want.detach())) < 1e-5 * float(want.detach())
    ours, theirs = torch.autograd.grad(loss, x)[0], torch.autograd.grad(want, x)[0]
    assert (ours - theirs).abs().max() < 1e-6


def test_row_alone_and_among_many():
    """A row's results do not depend on the batch it is in (within one size rule they are the
    same bits)."""
    x = torch.randn(600, 3001, device="cuda")
    t = torch.randint(0, 3001, (600,), device="cuda")
    whole = token_logprobs(x, t, top=4, entropy=True)
    again = token_logprobs(x, t, top=4, entropy=True)
    part = token_logprobs(x[7:527], t[7:527], top=4, entropy=True)
    for a, b, c in zip(whole, again, part):
        assert torch.equal(a, b) and torch.equal(a[7:527], c)


def test_saved_and_once():
    x = torch.randn(3, 50, device="cuda", requires_grad=True)
    t = torch.tensor([1, 2, 3], device="cuda")
    r = token_logprobs(x, t, top=2, entropy=True)
    assert not r.top_logprobs.requires_grad and not r.top_tokens.requires_grad
    first, = torch.autograd.grad(r.logprobs.square().sum(), x, retain_graph=True)
    again, = torch.autograd.grad(r.logprobs.square().sum(), x, retain_graph=True, create_graph=True)
    assert torch.equal(first, again)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        (again * again).sum().backward(retain_graph=True)
    with torch.no_grad():
        x.add_(1.0)
    with pytest.raises(RuntimeError, match="modified"):
        r.logprobs.sum().backward()


def test_saved_on_the_host_and_memory_used_in_between():
    """What the backward needs outlives the forward: saved tensors that come back as others (in
    rows without the view's gaps), and everything free in memory written over."""
    buf, t = torch.randn(37, 1010, device="cuda"), torch.randint(0, 1003, (37,), device="cuda")
    g = torch.randn(37, device="cuda")

    def grad(hooks, dirty):
        x = buf[:, 4:1007].detach().requires_grad_()
        with hooks:
            r = token_logprobs(x, t, entropy=True)
        if dirty:
            full = [torch.full((size,), NAN, device="cuda") for size in (37, 74, 37 * 1003) for _ in range(8)]
            del full
        return torch.autograd.grad([r.logprobs, r.entropy], x, [g, g])[0]

    want = grad(contextlib.nullcontext(), False)
    assert torch.equal(grad(contextlib.nullcontext(), True), want)
    assert torch.equal(grad(torch.autograd.graph.save_on_cpu(), True), want)


def test_streams_side_by_side():
    streams = [torch.cuda.Stream() for _ in range(3)]
    data = [(torch.randn(300, 30000, device="cuda"), torch.randint(0, 30000, (300,), device="cuda")) for _ in streams]
    torch.cuda.synchronize()
    out = []
    for s, (x, t) in zip(streams, data):
        with torch.cuda.stream(s):
            out.append(token_logprobs(x, t, top=5, entropy=True))
    torch.cuda.synchronize()
    for r, (x, t) in zip(out, data):
        for a, b in zip(r, token_logprobs(x, t, top=5, entropy=True)):
            assert torch.equal(a, b)


def test_captured_and_replayed():
    g = gen(6)
    x = torch.randn(40, 9001, generator=g, device="cuda").requires_grad_()
    t = torch.randint(0, 9001, (40,), generator=g, device="cuda")
    d = torch.randn(2, 40, generator=g, device="cuda")

    def step(v):
        r = token_logprobs(v, t, top=3, entropy=True)
        return (*r, torch.autograd.grad([r.logprobs, r.entropy], v, [d[0], d[1]])[0])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x)
    for k in range(4):
        with torch.no_grad():
            x.normal_(generator=g).mul_(k + 1)
        t.random_(0, 9001, generator=g)
        if k == 2:
            with torch.no_grad():
                x[3] = -INF
            t[4] = -100
        graph.replay()
        torch.cuda.synchronize()
        want = step(x.detach().clone().requires_grad_())
        for a, b in zip(out, want):
            assert torch.equal(a.detach(), b.detach())


def test_more_rows_than_a_grid_and_offsets_beyond_32_bits():
    n, V = 70000, 33000  # 4.6 GB
    x = torch.empty(n, V, device="cuda", dtype=torch.bfloat16).normal_(generator=gen(1)).requires_grad_()
    t = torch.randint(0, V, (n,), generator=gen(2), device="cuda")
    g, h = torch.randn(2, n, generator=gen(3), device="cuda")
    r = token_logprobs(x, t, top=2, entropy=True)
    dx, = torch.autograd.grad([r.logprobs, r.entropy], x, [g, h])
    rows = torch.tensor([0, 1, 65534, 65535, 65536, n - 2, n - 1], device="cuda")
    y = x.detach()[rows]
    lp, ent = R.logprobs(y, t[rows])
    bound, bound_h = R.logprobs_bound(y, t[rows])
    R.assert_within(r.logprobs[rows], lp, bound)
    R.assert_within(r.entropy[rows], ent, bound_h)
    assert torch.equal(r.top_tokens[rows], R.ranked(y, 2))
    want = R.logprobs_grad(y, t[rows], g[rows], h[rows])
    R.assert_within(dx[rows], want, R.grad_bound(y, t[rows], g[rows], h[rows], want))


def test_entry_point_leaves_what_is_not_its_own():
    x, t = torch.randn(5, 1003, device="cuda"), torch.tensor([0, 1, 2, 3, 1002], device="cuda")
    lp, ent, stats = (torch.full((k + 16,), 7.0, device="cuda") for k in (5, 5, 10))
    tl, tt = torch.full((31,), 7.0, device="cuda"), torch.full((31,), 7, device="cuda")
    mid = lambda b: b[8:-8]
    _lib.token_logprobs(x, t, -100, mid(lp), mid(ent), mid(stats), 3, mid(tl), mid(tt))
    dx = torch.full((5, 1010), 7.0, device="cuda")
    one = torch.ones(5, device="cuda")
    _lib.token_logprobs_backward(x, t, -100, mid(stats), mid(ent), one, one, dx[:, 3:1006])
    for b in (lp, ent, stats, tl, tt):
        assert (b[:8] == 7).all() and (b[-8:] == 7).all()
    assert (dx[:, :3] == 7).all() and (dx[:, 1006:] == 7).all()
    want = R.logprobs_grad(x, t, one, one)
    R.assert_within(dx[:, 3:1006], want, R.grad_bound(x, t, one, one, want))
    with pytest.raises(ValueError):
        _lib.token_logprobs(x, t, -100, lp, ent, stats, 0, None, None)
