"""CPU checks of the gated recurrence's, dropout's and the sampler's entry points: they
refuse bad arguments before any device work, at the C ABI and in the Python layer, and
the tests' own references agree with second forms of themselves."""
import ctypes

import numpy as np
import pytest
import torch

from gated_ref import gated_forward, keep_mask, philox_words, sample_row
from prime_moment_attention import GatedLinearRecurrence, _lib, dropout_add, gated_recurrence, sample_tokens

BF, F32 = _lib.PRIME_BF16, _lib.PRIME_F32
AT = [(i + 1) << 24 for i in range(20)]  # addresses far apart; never dereferenced
B, L, C = 2, 400, 64


def seq(addr, sl=C, sb=L * C):
    return _lib.PrimeSeq(addr, sb, sl)


def scan(x=seq(AT[0]), s=seq(AT[1]), g=seq(AT[2]), dt=BF, b=B, l=L, c=C, tau=AT[3], si=AT[4], y=seq(AT[5]), so=AT[6],
         ck=AT[7], ws=AT[8], n=1 << 22):
    return _lib.load().prime_gated_scan(x, s, g, dt, b, l, c, tau, si, y, so, ck, ws, n, None)


def scan_bwd(x=seq(AT[0]), s=seq(AT[1]), g=seq(AT[2]), dt=BF, tau=AT[3], ck=AT[4], dy=seq(AT[5]), do=AT[6],
             dx=seq(AT[7]), ds=seq(AT[8]), dg=seq(AT[9]), dtau=AT[10], di=AT[11], ws=AT[12], n=1 << 22):
    return _lib.load().prime_gated_scan_backward(x, s, g, dt, B, L, C, tau, ck, dy, do, dx, ds, dg, dtau, di, ws, n,
                                                 None)


def test_gated_scan_refuses_before_device_work():
    assert scan(x=None) == -1 and scan(tau=None) == -1 and scan(y=seq(None)) == -1
    assert scan(b=1 << 23, l=5) == -1 and "grid" in _lib.last_error()
    assert scan(b=0) == -1 and scan(l=0) == -1 and scan(c=-1) == -1 and scan(l=(1 << 30) + 1) == -1
    assert scan(dt=9) == -3
    assert scan(x=seq(AT[0], sl=-1)) == -1 and "stride" in _lib.last_error()
    assert scan(x=seq(AT[0] + 1)) == -4 and scan(tau=AT[3] + 2) == -4 and scan(so=AT[6] + 1) == -4
    assert scan(y=seq(AT[0] + 2)) == -5 and scan(y=seq(AT[5], sl=C - 1)) == -5
    assert scan(so=AT[4] + 4) == -5  # partly the incoming state
    assert scan(ck=AT[6] + 8) == -5 and scan(so=AT[3]) == -5
    need = _lib.load().prime_gated_scan_workspace_size(B, L, C)
    assert need > 0 and scan(n=need - 1) == -1 and "workspace" in _lib.last_error()
    assert scan(ws=None) == -1 and scan(ws=AT[0] + 16) == -5


def test_gated_backward_refuses_before_device_work():
    assert scan_bwd(ck=None) == -1 and scan_bwd(dtau=None) == -1 and scan_bwd(dx=None) == -1
    assert scan_bwd(dt=7) == -3 and scan_bwd(dg=seq(AT[9] + 1)) == -4
    assert scan_bwd(ds=seq(AT[7])) == -5 and scan_bwd(dx=seq(AT[1])) == -5
    assert scan_bwd(di=AT[10]) == -5 and scan_bwd(dtau=AT[4]) == -5 and scan_bwd(ws=AT[9]) == -5
    # thirds of one buffer whose columns do overlap
    wide = lambda o: seq(AT[7] + 2 * o, sl=3 * C, sb=3 * C * L)
    assert scan_bwd(dx=wide(0), ds=wide(C - 1), dg=wide(2 * C)) == -5
    need = _lib.load().prime_gated_scan_backward_workspace_size(B, L, C)
    assert scan_bwd(n=need - 1) == -1 and scan_bwd(ws=AT[12] + 4) == -1


def test_dropout_refuses_before_device_work():
    def call(x=AT[0], ldx=64, r=AT[1], ldr=64, o=AT[2], ldo=64, dt=BF, rows=8, cols=64, p=0.1, rng=AT[3]):
        return _lib.load().prime_dropout_add(x, ldx, r, ldr, o, ldo, dt, rows, cols, p, rng, 0, None)
    assert call(x=None) == -1 and call(o=None) == -1 and call(rng=None) == -1
    assert call(rows=0) == -1 and call(cols=-2) == -1 and call(rows=1 << 30, cols=1 << 30) == -1
    assert call(rows=(1 << 28) + 1, ldx=1 << 20) == -1
    assert call(ldx=63) == -1 and call(ldr=1) == -1 and call(ldo=0) == -1
    for p in (-0.1, 1.1, float("nan")):
        assert call(p=p) == -1 and "outside" in _lib.last_error()
    assert call(dt=5) == -3
    assert call(x=AT[0] + 1) == -4 and call(rng=AT[3] + 4) == -4
    assert call(o=AT[0] + 2) == -5 and call(o=AT[1] + 64) == -5 and call(o=AT[3] - 64) == -5
    assert call(o=AT[0], ldo=65) == -5  # the same start, other rows


def test_sample_refuses_before_device_work():
    def call(lg=AT[0], dt=BF, n=4, V=100, st=100, u=AT[1], T=None, k=None, p=None, m=None, out=AT[2]):
        return _lib.load().prime_sample(lg, dt, n, V, st, u, 1.0, T, 0, k, 1.0, p, 0.0, m, out, None)
    assert call(lg=None) == -1 and call(u=None) == -1 and call(out=None) == -1
    assert call(n=0) == -1 and call(V=0) == -1 and call(V=(1 << 20) + 1, st=1 << 21) == -1 and call(st=-1) == -1
    assert call(n=1 << 22) == -1
    assert call(dt=3) == -3
    assert call(lg=AT[0] + 1) == -4 and call(out=AT[2] + 4) == -4 and call(T=AT[3] + 1) == -4 and call(k=AT[3] + 2) == -4
    assert call(out=AT[0] + 8) == -5 and call(out=AT[1]) == -5 and call(k=AT[2]) == -5


def test_python_layer_refuses_host_tensors_and_bad_shapes():
    z = torch.zeros(1, 4, 8)
    with pytest.raises(RuntimeError, match="HIP device"):
        gated_recurrence(z, z, z, torch.ones(8))
    with pytest.raises(ValueError, match="step"):
        gated_recurrence(z, z[:, :2], z, torch.ones(8))
    with pytest.raises(ValueError, match="dtype"):
        gated_recurrence(z, z.half(), z, torch.ones(8))
    with pytest.raises(ValueError, match="tau"):
        gated_recurrence(z, z, z, torch.ones(7))
    with pytest.raises(ValueError, match="state"):
        gated_recurrence(z, z, z, torch.ones(8), state=torch.ones(1, 8).double())
    with pytest.raises(RuntimeError, match="dtype"):
        gated_recurrence(z.double(), z.double(), z.double(), torch.ones(8))
    with pytest.raises(RuntimeError, match="HIP device"):
        dropout_add(z, None, 0.1, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="HIP device"):
        sample_tokens(torch.zeros(2, 9), torch.zeros(2))


def test_gated_module_parameters():
    m = GatedLinearRecurrence(32, width=24)
    assert sorted(n for n, _ in m.named_parameters()) == ["in_proj.bias", "in_proj.weight", "log_tau", "o_proj.weight"]
    tau = m.get_tau(torch.device("cpu"))
    assert tau.shape == (24,) and abs(tau[0] - 2.0) < 1e-4 and abs(tau[-1] - 2000.0) < 0.1
    step = torch.nn.functional.softplus(m.in_proj.bias[24:48])
    assert torch.allclose(step, torch.ones(24))


def test_references_against_second_forms():
    """The scan's closed form over a short sequence, the paper's Philox vectors, and the
    sampler on a case worked by hand."""
    g = torch.Generator().manual_seed(0)
    x, s, gt = (torch.randn(1, 5, 3, generator=g).double() for _ in range(3))
    tau = torch.tensor([2.0, 30.0, 900.0]).double()
    y, last = gated_forward(x, s, gt, tau)
    z = torch.log1p(torch.exp(s)).clamp(1e-4, 50.0) / tau
    b = torch.sqrt(1 - torch.exp(-2 * z)) / (1 + torch.exp(-gt)) * x
    cum = z.cumsum(1)
    for t in range(5):
        closed = (torch.exp(-(cum[:, t:t + 1] - cum[:, :t + 1])) * b[:, :t + 1]).sum(1)
        assert torch.allclose(y[:, t], closed, rtol=1e-12, atol=1e-12)
    assert torch.equal(last, y[:, -1])
    assert philox_words(0, 0, 0) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    keep, scale = keep_mask(10, 0.5, 0, 0, 0)
    assert scale == 2.0 and list(keep[:2]) == [0xE8D5 >= 32768, 0x6627 >= 32768]
    row = np.log(np.array([0.1, 0.4, 0.2, 0.3]))
    assert [sample_row(row, u) for u in (0.05, 0.3, 0.6, 0.8)] == [0, 1, 2, 3]
    assert [sample_row(row, u, top_k=2) for u in (0.5, 0.6)] == [1, 3]
    assert [sample_row(row, u, top_p=0.75) for u in (0.1, 0.5, 0.9)] == [1, 2, 3]
    assert [sample_row(row, u, min_p=0.6) for u in (0.5, 0.6)] == [1, 3]
