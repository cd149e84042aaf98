"""CPU checks of the embedding's, the log probabilities' and the clipping's entry points: they
refuse bad arguments before any device work, at the C ABI and in the Python layer, and the
tests' own references agree with torch's."""
import array
import math

import pytest
import torch

import ends_ref as R
from prime_moment_attention import (_lib, clip_grad_norm_, clip_grads_with_norm_, embedding_lookup, grad_norm,
                                    token_logprobs)

BF, F32 = _lib.PRIME_BF16, _lib.PRIME_F32
AT = [(i + 1) << 28 for i in range(12)]  # addresses far apart; never dereferenced


def test_embedding_refuses_before_device_work():
    need = _lib.load().prime_embedding_order_size(8, 100)

    def call(ids=AT[0], i64=1, n=8, w=AT[1], ld=64, V=100, C=64, dt=BF, out=AT[2], order=AT[3], no=need):
        return _lib.load().prime_embedding(ids, i64, n, w, ld, V, C, dt, 1.0, -1, out, order, no, None)
    assert need > 0 and call(ids=None) == -1 and call(w=None) == -1 and call(out=None) == -1
    assert call(n=0) == -1 and call(V=0) == -1 and call(C=0) == -1 and call(n=(1 << 30) + 1) == -1
    assert call(V=1 << 31) == -1 and call(C=(1 << 20) + 1, ld=1 << 21) == -1
    assert call(ld=63) == -1 and "stride" in _lib.last_error()
    assert call(dt=5) == -3
    assert call(ids=AT[0] + 4) == -4 and call(ids=AT[0] + 2, i64=0) == -4
    assert call(w=AT[1] + 1) == -4 and call(out=AT[2] + 1) == -4 and call(out=AT[2] + 2, dt=F32) == -4
    assert call(out=AT[1] + 64) == -5 and call(out=AT[0]) == -5 and call(out=AT[1] + 2 * (99 * 64 + 63)) == -5
    assert call(no=need - 1) == -1 and "order" in _lib.last_error() and call(order=AT[3] + 8) == -1
    assert call(order=AT[0]) == -5 and call(order=AT[1] + 16) == -5 and call(order=AT[2] + 16) == -5
    # more threads than a launch has
    assert call(n=1 << 30, C=1 << 13, ld=1 << 13, order=None) == -1 and "grid" in _lib.last_error()


def test_embedding_backward_refuses_before_device_work():
    L = _lib.load()
    size, osize = L.prime_embedding_backward_workspace_size, L.prime_embedding_order_size
    need, norder = size(8, 64), osize(8, 100)

    def call(order=AT[0], no=norder, n=8, dy=AT[1], ld=64, V=100, C=64, dt=BF, dw=AT[2], ws=AT[3], nw=need):
        return L.prime_embedding_backward(order, no, n, dy, ld, V, C, dt, 1.0, dw, ws, nw, None)
    assert need > 0 and size(0, 64) == 0 and size(8, 0) == 0 and osize(0, 100) == 0 and osize(8, 0) == 0
    assert call(order=None) == -1 and call(dy=None) == -1 and call(dw=None) == -1 and call(ws=None) == -1
    assert call(nw=need - 1) == -1 and "workspace" in _lib.last_error() and call(ws=AT[3] + 8) == -1
    assert call(no=norder - 1) == -1 and "order" in _lib.last_error() and call(order=AT[0] + 8) == -1
    assert call(ld=63) == -1 and call(dt=4) == -3 and call(dw=AT[2] + 1) == -4
    assert call(dw=AT[1] + 128) == -5 and call(dw=AT[0]) == -5 and call(ws=AT[2] + 16) == -5
    assert call(ws=AT[1]) == -5 and call(ws=AT[0]) == -5


def test_logprobs_refuse_before_device_work():
    def call(x=AT[0], dt=BF, n=4, V=100, st=100, tok=AT[1], lp=AT[2], ent=AT[3], stats=AT[4], top=5, tl=AT[5], tt=AT[6]):
        return _lib.load().prime_token_logprobs(x, dt, n, V, st, tok, -100, lp, ent, stats, top, tl, tt, None)
    assert call(x=None) == -1 and call(tok=None) == -1 and call(lp=None) == -1
    assert call(tl=None) == -1 and call(tt=None) == -1
    assert call(n=0) == -1 and call(V=0) == -1 and call(V=(1 << 24) + 1) == -1 and call(st=-1) == -1
    assert call(top=-1) == -1 and call(top=65) == -1 and call(V=4, top=5) == -1 and "top" in _lib.last_error()
    assert call(dt=3) == -3
    assert call(x=AT[0] + 1) == -4 and call(tok=AT[1] + 4) == -4 and call(lp=AT[2] + 2) == -4 and call(tt=AT[6] + 4) == -4
    assert call(lp=AT[0] + 4) == -5 and call(ent=AT[1]) == -5 and call(stats=AT[2] + 4) == -5 and call(tt=AT[5] + 8) == -5


def test_logprobs_backward_refuses_before_device_work():
    def call(x=AT[0], dt=BF, n=4, V=100, st=100, tok=AT[1], stats=AT[2], ent=AT[3], g=AT[4], h=AT[5], dx=AT[6], sd=100):
        return _lib.load().prime_token_logprobs_backward(x, dt, n, V, st, tok, -100, stats, ent, g, h, dx, sd, None)
    assert call(x=None) == -1 and call(stats=None) == -1 and call(dx=None) == -1 and call(ent=None) == -1
    assert call(sd=99) == -1 and call(n=-1) == -1 and call(dt=8) == -3
    assert call(dx=AT[6] + 1) == -4 and call(g=AT[4] + 1) == -4 and call(stats=AT[2] + 3) == -4
    assert call(dx=AT[0]) == -5 and call(dx=AT[0] + 200) == -5 and call(dx=AT[2] + 8) == -5 and call(dx=AT[5]) == -5


def test_clipping_refuses_before_device_work():
    L = _lib.load()

    def call(data=(AT[0], AT[1]), sizes=(100, 50), dts=(BF, F32), norm=AT[4], ws=AT[5], n=1 << 20, max_norm=1.0, given=0, both=True):
        a = [array.array(t, v) for t, v in (("Q", data), ("q", sizes), ("i", dts))]
        p = [x.buffer_info()[0] for x in a]
        if both:
            assert L.prime_grad_norm(*p, len(data), norm, ws, n, None) == L.prime_grad_clip(*p, len(data), max_norm, norm, given, ws, n, None)
        return L.prime_grad_clip(*p, len(data), max_norm, norm, given, ws, n, None)
    assert call(norm=None) == -1 and call(ws=None) == -1 and call(n=7) == -1 and "workspace" in _lib.last_error()
    assert call(sizes=(100, -1)) == -1 and call(data=(AT[0], 0)) == -1 and call(sizes=(1 << 35, 1)) == -1
    assert call(sizes=((1 << 35) - 8, (1 << 35) - 8)) == -1
    assert call(dts=(BF, 7)) == -3
    assert call(data=(AT[0] + 1, AT[1])) == -4 and call(data=(AT[0], AT[1] + 2)) == -4 and call(norm=AT[4] + 2) == -4
    assert call(norm=AT[0] + 8) == -5 and call(ws=AT[1]) == -5 and call(norm=AT[5] + 4) == -5
    # tensors that overlap each other have a norm, but are not clipped
    assert call(data=(AT[0], AT[0] + 196), both=False) == -5 and "overlap" in _lib.last_error()
    assert call(data=(AT[1] + 4, AT[1]), both=False) == -5 and call(data=(AT[0], AT[0]), both=False) == -5
    assert call(max_norm=-1.0, both=False) == -1 and call(max_norm=math.nan, both=False) == -1
    assert L.prime_grad_norm_workspace_size(None, 3) == 0


def test_python_layer_refuses_host_tensors_and_bad_arguments():
    w, ids = torch.zeros(9, 4), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="HIP device"):
        embedding_lookup(ids, w)
    with pytest.raises(ValueError, match="ids"):
        embedding_lookup(ids.float(), w)
    with pytest.raises(ValueError, match="weight"):
        embedding_lookup(ids, w[0])
    for pad in (9, -10):
        with pytest.raises(ValueError, match="padding_idx"):
            embedding_lookup(ids, w, padding_idx=pad)
    with pytest.raises(RuntimeError, match="dtype"):
        embedding_lookup(ids, w.double())
    x, t = torch.zeros(3, 9), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="HIP device"):
        token_logprobs(x, t)
    with pytest.raises(ValueError, match="tokens"):
        token_logprobs(x, t[:2])
    with pytest.raises(ValueError, match="tokens"):
        token_logprobs(x, t.float())
    with pytest.raises(RuntimeError, match="dtype"):
        token_logprobs(x.double(), t)
    with pytest.raises(ValueError, match="empty"):
        token_logprobs(x[:, :0], t)
    for top in (-1, 10):
        with pytest.raises(ValueError, match="top"):
            token_logprobs(x, t, top=top)
    with pytest.raises(ValueError, match="top"):
        token_logprobs(torch.zeros(3, 100), t, top=65)
    with pytest.raises(ValueError, match="ignore_index"):
        token_logprobs(x, t, ignore_index=1 << 63)
    p = torch.nn.Parameter(torch.zeros(4))
    p.grad = torch.ones(4)
    with pytest.raises(RuntimeError, match="HIP device"):
        clip_grad_norm_([p], 1.0)
    with pytest.raises(RuntimeError, match="HIP device"):
        grad_norm(p)
    for m in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            clip_grad_norm_([p], m)
        with pytest.raises(ValueError, match="max_norm"):
            clip_grads_with_norm_([p], m, torch.ones(()))
    p.grad = torch.ones(1).expand(4)
    with pytest.raises(ValueError, match="overlaps itself"):
        clip_grad_norm_([p], 1.0)
    q = torch.nn.Parameter(torch.zeros(4, 4))
    q.grad = torch.eye(4).to_sparse()
    with pytest.raises(ValueError, match="layout"):
        clip_grad_norm_([q], 1.0)


def test_no_gradients_have_a_norm_of_zero():
    p = torch.nn.Parameter(torch.zeros(4))
    assert float(clip_grad_norm_([p], 1.0)) == 0.0 and float(grad_norm([])) == 0.0 and float(grad_norm(iter([p]))) == 0.0


def test_references_against_torch():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(5, 11, generator=g).double().requires_grad_()
    t = torch.tensor([0, 10, 3, -100, 7])
    lp, ent = R.logprobs(x, t)
    want = -torch.nn.functional.cross_entropy(x, t, reduction="none", ignore_index=-100)
    assert torch.allclose(lp, want) and torch.allclose(ent, torch.distributions.Categorical(logits=x).entropy())
    a, b = torch.randn(5, generator=g).double(), torch.randn(5, generator=g).double()
    total = (a * want).sum()
    grad, = torch.autograd.grad((a * -torch.nn.functional.cross_entropy(x, t, reduction="none", ignore_index=-100)).sum()
                                + (b * torch.distributions.Categorical(logits=x).entropy()).sum(), x)
    assert total.isfinite() and torch.allclose(R.logprobs_grad(x, t, a, b), grad)
    y = x.detach().clone()
    y[0], y[1, 3], y[2, 1:3], y[4, 0] = -math.inf, math.nan, math.inf, -math.inf
    lp, ent = R.logprobs(y, torch.tensor([0, 0, 1, 2, 1]))
    assert lp[0] == -math.inf and ent[0] == 0 and lp[1].isnan() and ent[1].isnan()
    assert abs(lp[2] + math.log(2)) < 1e-12 and abs(ent[2] - math.log(2)) < 1e-12 and lp[4].isfinite()
    dx = R.logprobs_grad(y, torch.tensor([0, 0, 1, 2, 1]), torch.ones(5), torch.ones(5))
    assert (dx[0] == 0).all() and dx[1].isnan().all() and torch.allclose(dx[2, 1:3], torch.tensor([0.5, -0.5]).double())
    w = torch.randn(7, 3, generator=g)
    ids = torch.tensor([[1, 6, 1], [9, -1, 0]])
    y, _ = R.lookup(ids, w, 2.0)
    assert torch.equal(y[0], 2.0 * w[ids[0]].double()) and (y[1, :2] == 0).all()
    dy = torch.randn(2, 3, 3, generator=g)
    grad, _ = R.lookup_grad(ids, dy, 7, 2.0, padding=0)
    assert torch.allclose(grad[1], 2.0 * (dy[0, 0] + dy[0, 2]).double()) and (grad[[0, 2, 3, 4, 5]] == 0).all()
    p = torch.nn.Parameter(w.clone())
    p.grad = 3.0 * w
    norm, want, _ = R.clipped([p.grad.clone()], 1.0)
    assert math.isclose(norm, float(torch.nn.utils.clip_grad_norm_([p], 1.0)), rel_tol=1e-6)
    assert torch.allclose(p.grad.double(), want[0], rtol=1e-6)
