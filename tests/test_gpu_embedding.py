"""The embedding lookup and its gradient by sorted tokens, against their plain forms in 64 bits."""
import pytest
import torch

import ends_ref as R
from prime_moment_attention import _lib, embedding_lookup

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def make_ids(kind, shape, V, g):
    u = torch.rand(shape, generator=g, device="cuda")
    if kind == "same":
        return torch.full(shape, V // 2, device="cuda")
    if kind == "ranked":
        return (torch.exp(u * torch.log(torch.tensor(V + 1.0))) - 1).long().clamp(0, V - 1)
    if kind == "outside":  # a third of them below or above the table
        ids = torch.randint(0, V, shape, generator=g, device="cuda")
        return torch.where(u < 0.2, ids - V, torch.where(u > 0.85, ids + V, ids))
    ids = torch.randint(0, V, shape, generator=g, device="cuda")
    return ids.flatten().sort(descending=True).values.view(shape) if kind == "sorted" else ids


def check(ids, weight, dy, scale=1.0, padding=None):
    w = weight.detach().requires_grad_()
    y = embedding_lookup(ids, w, scale, padding)
    want, bound = R.lookup(ids, weight, scale)
    R.assert_within(y, want, bound, "rows")
    assert y.dtype is weight.dtype
    grad, = torch.autograd.grad(y, w, dy)
    want, bound = R.lookup_grad(ids, dy, weight.shape[0], scale, padding)
    R.assert_within(grad, want, bound(weight.dtype), "gradient")
    with torch.no_grad():
        assert torch.equal(embedding_lookup(ids, weight, scale, padding), y.detach())
    return grad


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n, V, C, kind", [
    (1, 1, 1, "same"), (1, 7, 3, "uniform"), (2, 2, 7, "uniform"), (31, 5, 8, "uniform"), (32, 1, 9, "same"),
    (33, 3, 16, "ranked"), (64, 300, 64, "uniform"), (65, 511, 33, "sorted"), (255, 512, 24, "outside"),
    (1000, 513, 100, "ranked"), (1024, 40, 128, "same"), (1025, 50304, 40, "ranked"), (4097, 1000, 65, "same"),
    (2331, 32000, 501, "ranked"), (5000, 262143, 5, "uniform"), (5000, 262144, 5, "uniform"), (3000, 300000, 8, "outside"),
    (70000, 50304, 64, "ranked"), (600000, 2000, 16, "ranked"), (131072, 128, 8, "uniform"), (131073, 129, 8, "uniform"),
    (140000, 3, 24, "outside"), (150000, 262145, 5, "outside"), (30000, 70000, 520, "ranked"), (17000, 65537, 1030, "ranked"),
    (16384, 20, 700, "outside"), (16383, 20, 700, "outside"), (9000, 100000, 16, "same"), (9000, 100000, 16, "ranked"),
    (16000, 100000, 20, "uniform"), (2200000, 70000, 3, "ranked")])
def test_lookup_and_gradient(dtype, n, V, C, kind):
    g = gen(n * 7 + V)
    ids = make_ids(kind, (n,), V, g)
    weight = torch.randn(V, C, generator=g, device="cuda").to(dtype)
    dy = torch.randn(n, C, generator=g, device="cuda").to(dtype)
    check(ids, weight, dy, scale=1.0 if n % 2 else 27.7, padding=None if C % 2 else V // 2 - V)


@pytest.mark.parametrize("dtype", DTYPES)
def test_views_and_types(dtype):
    """Rows that start anywhere, wide strides, ids of any shape, order and type, gradients that
    are views: broadcast, transposed, reversed in memory order."""
    g = gen(5)
    wide = torch.randn(301, 60, generator=g, device="cuda").to(dtype)
    ids = make_ids("ranked", (6, 40), 301, g)
    for C, at in ((37, 3), (32, 1), (1, 7), (3, 5)):
        view = wide[:, at:at + C]
        dy = torch.randn(6, 40, C, generator=g, device="cuda").to(dtype)
        for some in (ids, ids.t(), ids[:, ::3], ids.int(), ids[:, 5], ids[2, 3]):
            y = embedding_lookup(some, view, 0.5)
            assert torch.equal(y, embedding_lookup(some.long().contiguous(), view.contiguous(), 0.5))
        check(ids, view, dy)
        check(ids.t(), view, dy.transpose(0, 1))
        check(ids, view, dy[:1, :1].expand(6, 40, C))
        check(ids, view, torch.randn(6, 40, C + 2, generator=g, device="cuda").to(dtype)[..., 1:-1])
        check(ids, view, torch.randn(C, 40, 6, generator=g, device="cuda").to(dtype).permute(2, 1, 0))
    tall = torch.randn(60, 301, generator=g, device="cuda").to(dtype).t()  # columns far apart
    check(ids, tall, torch.randn(6, 40, 60, generator=g, device="cuda").to(dtype))


def test_nothing_to_look_up():
    for n, V, C in ((0, 5, 4), (3, 5, 0), (3, 0, 4), (0, 0, 0)):
        w = torch.randn(V, C, device="cuda").requires_grad_()
        y = embedding_lookup(torch.zeros(2, n, dtype=torch.int64, device="cuda"), w, 2.0)
        assert y.shape == (2, n, C) and (y == 0).all()
        grad, = torch.autograd.grad(y.sum(), w)
        assert grad.shape == (V, C) and (grad == 0).all()


def test_gradient_is_the_lookup_turned_round():
    """<dy, lookup(W + D) - lookup(W)> = <gradient, D>: whole numbers, so that all is exact."""
    g = gen(11)
    ids = make_ids("outside", (700,), 90, g)
    W, D = (torch.randint(-8, 9, (90, 21), generator=g, device="cuda").float() for _ in range(2))
    dy = torch.randint(-8, 9, (700, 21), generator=g, device="cuda").float()
    w = W.clone().requires_grad_()
    grad, = torch.autograd.grad(embedding_lookup(ids, w, 4.0), w, dy)
    step = embedding_lookup(ids, W + D, 4.0) - embedding_lookup(ids, W, 4.0)
    assert (dy.double() * step.double()).sum() == (grad.double() * D.double()).sum()


@pytest.mark.parametrize("n", [40, 700, 16383, 16384, 40000, 140000])
@pytest.mark.parametrize("ids64", [True, False])
def test_runs_of_every_length(n, ids64):
    """Ids that occur 1, 2, .. 100 times, in turn and at every place of a chunk, some of them
    thousands of times, some outside the table: whole numbers, so that the sums are exact."""
    g = gen(n)
    lengths = [*range(1, 101), 3000, 1, 64, 31, 32, 33, 7, 8, 9, 5000, 15, 16, 17, 65, 96, 97]
    runs = []
    while sum(runs) < n:
        runs += lengths[len(runs) % 7:]
    keys = torch.repeat_interleave(torch.arange(len(runs), device="cuda"), torch.tensor(runs, device="cuda"))[:n]
    V = int(keys.max()) + 1
    mixed = torch.randperm(V + 9, generator=g, device="cuda")[keys]  # (some above the table)
    ids = mixed[torch.randperm(n, generator=g, device="cuda")]
    dy = torch.randint(-4, 5, (n, 70), generator=g, device="cuda").float()
    w = torch.zeros(V, 70, device="cuda").requires_grad_()
    for order in (ids, mixed):
        grad, = torch.autograd.grad(embedding_lookup(order if ids64 else order.int(), w, 0.5), w, dy)
        want, _ = R.lookup_grad(order, dy, V, 0.5)
        assert torch.equal(grad.cpu().double(), want)


def test_values_that_are_not_finite_stay_in_their_rows():
    w = torch.randn(6, 40, device="cuda")
    w[2, 3], w[4, 5] = float("inf"), float("nan")
    ids = torch.tensor([2, 1, 4, 2], device="cuda")
    y = embedding_lookup(ids, w, 2.0)
    assert y[0, 3] == float("inf") and y[2, 5].isnan() and y[1].isfinite().all() and y.isfinite().sum() == 4 * 40 - 3
    dy = torch.ones(4, 40, device="cuda")
    dy[1, 0] = float("nan")
    w.requires_grad_()
    grad, = torch.autograd.grad(embedding_lookup(ids, w), w, dy)
    assert grad[1, 0].isnan() and grad.isfinite().sum() == 6 * 40 - 1


def test_same_bits_every_time():
    g = gen(2)
    ids = make_ids("ranked", (20000,), 700, g)
    w = torch.randn(700, 200, generator=g, device="cuda").requires_grad_()
    dy = torch.randn(20000, 200, generator=g, device="cuda")
    first, = torch.autograd.grad(embedding_lookup(ids, w), w, dy)
    for _ in range(5):
        again, = torch.autograd.grad(embedding_lookup(ids, w), w, dy)
        assert torch.equal(first, again)


def test_retained_graph_and_one_gradient_only():
    w = torch.randn(9, 4, device="cuda", requires_grad=True)
    y = embedding_lookup(torch.tensor([1, 1, 8], device="cuda"), w)
    first, = torch.autograd.grad(y.square().sum(), w, retain_graph=True)
    again, = torch.autograd.grad(y.square().sum(), w, create_graph=True)
    assert torch.equal(first, again)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        (again * again).sum().backward()
    ids = torch.tensor([1, 2], device="cuda")
    y = embedding_lookup(ids, w)
    ids.add_(1)  # the gradient is that of the ids as they were
    grad, = torch.autograd.grad(y.sum(), w)
    assert (grad[[1, 2]] == 1).all() and grad.sum() == 8


def test_order_outlives_the_forward():
    w = torch.randn(500, 33, device="cuda", requires_grad=True)
    for n in (40, 3000, 20000):
        ids, dy = torch.randint(0, 500, (n,), device="cuda"), torch.randn(n, 33, device="cuda")
        want, = torch.autograd.grad(embedding_lookup(ids, w), w, dy)
        y = embedding_lookup(ids, w)
        size = _lib.load().prime_embedding_order_size(n, 500)
        full = [torch.full((size,), 255, dtype=torch.uint8, device="cuda") for _ in range(8)]
        del full
        got, = torch.autograd.grad(y, w, dy)
        assert torch.equal(got, want)


def test_streams_side_by_side():
    g = gen(8)
    streams = [torch.cuda.Stream() for _ in range(3)]
    data = [(make_ids("ranked", (30000,), 5000, g), torch.randn(5000, 96, generator=g, device="cuda").requires_grad_(),
             torch.randn(30000, 96, generator=g, device="cuda")) for _ in streams]
    torch.cuda.synchronize()
    out = []
    for s, (ids, w, dy) in zip(streams, data):
        with torch.cuda.stream(s):
            out.append(torch.autograd.grad(embedding_lookup(ids, w), w, dy)[0])
    torch.cuda.synchronize()
    for got, (ids, w, dy) in zip(out, data):
        assert torch.equal(got, torch.autograd.grad(embedding_lookup(ids, w), w, dy)[0])


def test_captured_with_new_ids_at_each_replay():
    g = gen(4)
    ids = make_ids("ranked", (3000,), 800, g)
    w = torch.randn(800, 48, generator=g, device="cuda").requires_grad_()
    dy = torch.randn(3000, 48, generator=g, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(embedding_lookup(ids, w, 3.0), w, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = embedding_lookup(ids, w, 3.0)
        grad, = torch.autograd.grad(y, w, dy)
    for kind in ("uniform", "same", "sorted", "outside", "ranked"):
        ids.copy_(make_ids(kind, (3000,), 800, g))
        dy.normal_(generator=g)
        graph.replay()
        torch.cuda.synchronize()
        v = w.detach().clone().requires_grad_()
        want = embedding_lookup(ids, v, 3.0)
        assert torch.equal(y.detach(), want.detach())
        assert torch.equal(grad, torch.autograd.grad(want, v, dy)[0])


def test_tables_and_gradients_beyond_32_bits():
    """A table of 4.9 GB and rows near both ends of it; rows of dy behind 4 GB."""
    V, C = 600000, 4096
    w = torch.empty(V, C, device="cuda", dtype=torch.bfloat16).normal_().requires_grad_()
    ids = torch.tensor([V - 1, 0, V - 1, V // 2, 5], device="cuda")
    y = embedding_lookup(ids, w)
    assert torch.equal(y.detach(), w.detach()[ids])
    dy = torch.randn(5, C, device="cuda").bfloat16()
    grad, = torch.autograd.grad(y, w, dy)
    want, bound = R.lookup_grad(torch.tensor([3, 0, 3, 2, 1]), dy, 4)
    R.assert_within(grad[[0, 5, V // 2, V - 1]], want, bound(torch.bfloat16))
    assert grad.abs().amax(1).count_nonzero() == 4
    del grad, y
    small = w.detach()[:16].clone().requires_grad_()
    ids = torch.full((V,), 20, device="cuda")
    ids[[1, V - 2, V - 1]] = torch.tensor([3, 3, 15], device="cuda")
    grad, = torch.autograd.grad(embedding_lookup(ids, small), small, w.detach())
    want, bound = R.lookup_grad(torch.tensor([0, 0, 1]), w.detach()[[1, V - 2, V - 1]], 2)
    R.assert_within(grad[[3, 15]], want, bound(torch.bfloat16))
    assert grad.abs().amax(1).count_nonzero() == 2


@pytest.mark.parametrize("n", [5000, 50000])
def test_a_table_of_very_many_rows(n):
    """More rows than two digits tell apart; whole numbers, so that the sums are exact."""
    V = (1 << 25) + 1001
    g = gen(n)
    w = torch.zeros(V, 1, device="cuda", dtype=torch.bfloat16).requires_grad_()
    ids = torch.cat([torch.randint(0, V, (n // 2,), generator=g, device="cuda"), torch.full((n - n // 2,), V - 1, device="cuda")])
    ids = ids[torch.randperm(n, generator=g, device="cuda")]
    dy = torch.randint(-2, 3, (n, 1), generator=g, device="cuda").bfloat16()
    grad, = torch.autograd.grad(embedding_lookup(ids, w), w, dy)
    want = torch.zeros(V, 1, device="cuda").index_add_(0, ids, dy.float())
    assert torch.equal(grad, want.bfloat16())


def test_entry_point_leaves_what_is_not_its_own():
    """Rows of a wider buffer are read, guards around the outputs stay."""
    n, V, C = 77, 50, 19
    ids = make_ids("ranked", (n,), V, gen(1))
    w = torch.randn(V, C, device="cuda")
    buf = torch.full((n * C + 64,), 7.0, device="cuda")
    _lib.embedding(ids, w, 1.0, buf[32:-32].view(n, C))
    assert (buf[:32] == 7).all() and (buf[-32:] == 7).all() and torch.equal(buf[32:-32].view(n, C), w[ids])
    size = _lib.embedding_order(n, V, "cuda").numel()
    order = torch.full((size + 512,), 7, dtype=torch.uint8, device="cuda")
    _lib.embedding(ids, w, 1.0, torch.empty(n, C, device="cuda"), -1, order[256:-256])
    assert (order[:256] == 7).all() and (order[-256:] == 7).all()
    buf = torch.full((V * C + 64,), 7.0, device="cuda")
    _lib.embedding_backward(order[256:-256], torch.randn(n, C, device="cuda"), 1.0, buf[32:-32].view(V, C))
    assert (buf[:32] == 7).all() and (buf[-32:] == 7).all()
    with pytest.raises(ValueError):
        _lib.embedding(ids, w, 1.0, buf[:5])
    with pytest.raises(RuntimeError, match="order"):
        _lib.embedding_backward(order[:size - 1], torch.randn(n, C, device="cuda"), 1.0, w)
    with pytest.raises(RuntimeError, match="order"):
        _lib.embedding(ids, w, 1.0, torch.empty(n, C, device="cuda"), -1, order[1:])
