"""Log probabilities, entropy and gradients over the whole range of finite logits: masks of any
size, largest logits of any size, and both in the places where a lane, a wave or a batch of
vectors has nothing else."""
import pytest
import torch

import ends_ref as R
from prime_moment_attention import _lib, token_logprobs
from test_gpu_logprobs import check, gen

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def magnitudes(dtype, g):
    """Powers of two, whose product with log2(e) leaves no residual in fp32, masks in use, and
    sizes at random from 2^20 to 2^127."""
    out = [2.0 ** k for k in (*range(20, 121, 4), *range(121, 128))]
    out += [8e6, 1e7, 1.2e7, 1e8, 1e9, 1660944384.0, 1888815488.0, 2.5e9, 1e10, 1e30, 1e38, 1.7e38, 3e38]
    out += torch.exp2(20 + 107 * torch.rand(24, generator=g, device="cuda").double()).tolist()
    out += torch.exp2(29 + 5 * torch.rand(24, generator=g, device="cuda").double()).tolist()
    if dtype is F16:
        out = [2.0 ** k for k in range(8, 16)] + [1e4, 65504.0]
    return out


def rows_with(a, base, lane, wave):
    """Rows like `base` with a as a mask and as the largest logit; lane, wave: the places that one
    lane and one wave read."""
    V = base.numel()
    first = torch.arange(V, device="cuda") < V // 2
    keep = torch.zeros(V, dtype=torch.bool, device="cuda")
    keep[-1] = True
    masks = [first, ~first, lane, wave, ~keep]
    rows = [torch.where(m, -a, base) for m in masks]
    rows += [base.clone(), base.clone(), torch.full_like(base, -a), torch.full_like(base, a), base.clone()]
    rows[5][V // 2] = a
    rows[6][V // 3] = rows[6][V // 2] = a  # two share the probability
    rows[9][:] = -a
    rows[9][V // 2] = a
    return rows


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("V, threads", [(100, 64), (2048, 64), (9001, 256), (20001, 1024), (70001, 1024)])
def test_masks_and_largest_logits_of_any_size(dtype, V, threads):
    g = gen(V)
    base = (2 * torch.randn(V, generator=g, device="cuda")).to(dtype).float()
    owner = torch.arange(V, device="cuda") // (4 if dtype is F32 else 8) % threads
    lane, wave = owner == 3, owner // 64 == (1 if threads > 64 else 0)
    if threads == 64:
        wave = owner < 32
    x = torch.cat([torch.stack(rows_with(a, base, lane, wave)) for a in magnitudes(dtype, g)]).to(dtype)
    for part in x.split(300):
        n = part.shape[0]
        tokens = torch.randint(0, V, (n,), generator=g, device="cuda")
        tokens[::2] = part[::2].float().argmax(1)
        a, b = torch.randn(2, n, generator=g, device="cuda")
        check(part, tokens, 2, True, a, b)
        check(part, tokens, 0, True, None, b)


def test_masks_in_many_rows():
    """The form for many rows of a large vocabulary."""
    g = gen(3)
    n, V = 600, 17001
    x = 2 * torch.randn(n, V, generator=g, device="cuda")
    a = torch.exp2(20 + 107 * torch.rand(n, 1, generator=g, device="cuda"))
    a[::3] = torch.exp2(29 + 5 * torch.rand(n // 3, 1, generator=g, device="cuda"))
    x = torch.where(torch.arange(V, device="cuda") < V // 2, -a, x)
    tokens = torch.randint(0, V, (n,), generator=g, device="cuda")
    d = torch.randn(2, n, generator=g, device="cuda")
    check(x, tokens, 3, True, d[0], d[1])


@pytest.mark.parametrize("V", [100, 9001, 50304])
def test_a_finite_mask_is_as_good_as_minus_infinity(V):
    """Masked tokens have no probability, whatever the mask: the same bits as of -infinity."""
    g = gen(V)
    base = 3 * torch.randn(8, V, generator=g, device="cuda")
    banned = torch.rand(8, V, generator=g, device="cuda") < 0.7
    banned[:4, : V // 2] = True
    banned[:, -1] = False
    tokens = torch.full((8,), V - 1, device="cuda")
    d = torch.randn(2, 8, generator=g, device="cuda")

    def results(mask, dtype):
        x = torch.where(banned, mask, base).to(dtype).requires_grad_()
        r = token_logprobs(x, tokens, entropy=True)
        return r.logprobs.detach(), r.entropy.detach(), torch.autograd.grad([r.logprobs, r.entropy], x, [d[0], d[1]])[0]

    for dtype in (F32, BF16):
        want = results(-float("inf"), dtype)
        for mask in (-1e9, -1e10, -2.5e9, -1660944384.0, -1e30, -1e38, -2.0 ** 126, torch.finfo(dtype).min):
            for a, b in zip(results(mask, dtype), want):
                assert torch.equal(a, b), (dtype, mask)

def test_a_token_outside_the_vocabulary_has_an_entropy_all_the_same():
    """Its log probability is NaN; of the entropy alone the gradient is that of any other row."""
    for V in (70, 3000, 20000):
        x = torch.randn(4, V, generator=gen(V), device="cuda")
        tokens = torch.tensor([3, V, -1, -100], device="cuda")
        h = torch.randn(4, device="cuda")
        leaf = x.clone().requires_grad_()
        r = token_logprobs(leaf, tokens, entropy=True)
        dx, = torch.autograd.grad(r.entropy, leaf, h)
        want = R.logprobs_grad(x, tokens, None, h)
        assert want.isfinite().all()
        R.assert_within(dx, want, R.grad_bound(x, tokens, None, h, want), "gradient")


def test_as_many_rows_as_a_call_takes():
    """2^31 - 1 rows of one token each, whose probability is 1: 4 GB of logits, 17 GB of tokens."""
    n = (1 << 31) - 1
    x = torch.randn(n, 1, device="cuda", dtype=BF16)
    tokens = torch.zeros(n, dtype=torch.int64, device="cuda")
    tokens[-1] = tokens[(1 << 30) + 3] = -100
    tokens[5] = 1
    guard = torch.full((n + 8,), 7.0, device="cuda")
    lp = guard[:n]
    _lib.token_logprobs(x, tokens, -100, lp, None, None, 0, None, None)
    assert lp[5].isnan() and (guard[n:] == 7).all()
    lp[5] = 0.0
    # d - log2 S with S = 2^d (1 + e): |e| <= 2 u of the exponential, so that e / ln 2, log2's rounding
    # (2 u of |log2 S| < 1) and the difference's come to less than 6 u; times ln 2
    assert lp.abs().max() <= 6 * R.U32
