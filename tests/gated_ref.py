"""Plain float64 forms of the gated linear recurrence, of Philox4x32-10 dropout and of
the sampled token, for the tests (not collected: no test_ prefix)."""
import math

import numpy as np
import torch

STEP_MIN, STEP_MAX = 1e-4, 50.0


def gated_forward(x, step, gate, tau, state=None):
    """Token by token over [B, L, C]; differentiable by autograd."""
    soft = torch.logaddexp(step, torch.zeros_like(step))
    log_a = -soft.clamp(STEP_MIN, STEP_MAX) / tau
    a = log_a.exp()
    b = (-torch.expm1(2 * log_a)).sqrt() * torch.sigmoid(gate) * x
    h = torch.zeros_like(x[:, 0]) if state is None else state
    ys = []
    for at, bt in zip(a.unbind(1), b.unbind(1)):
        h = at * h + bt
        ys.append(h)
    return torch.stack(ys, 1), h


def philox_words(block, counter, seed):
    """Four 32-bit words of Philox4x32-10 for one block, in Python integers."""
    m = 0xFFFFFFFF
    c = [block & m, block >> 32 & m, counter & m, counter >> 32 & m]
    k = [seed & m, seed >> 32 & m]
    for _ in range(10):
        p0, p1 = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(p1 >> 32) ^ c[1] ^ k[0], p1 & m, (p0 >> 32) ^ c[3] ^ k[1], p0 & m]
        k = [(k[0] + 0x9E3779B9) & m, (k[1] + 0xBB67AE85) & m]
    return c


def keep_mask(n, p, seed, offset, call):
    """(keep [n], 1 / (1 - p)) with p in steps of 1/65536."""
    cut = int(p * 65536 + 0.5)
    counter = (offset + call) % (1 << 64)
    bits = np.empty((-(-n // 8), 8), dtype=np.int64)
    for j in range(bits.shape[0]):
        for i, w in enumerate(philox_words(j, counter, seed % (1 << 64))):
            bits[j, 2 * i], bits[j, 2 * i + 1] = w & 0xFFFF, w >> 16
    return bits.reshape(-1)[:n] >= cut, 65536.0 / (65536 - cut) if cut < 65536 else 0.0


def sample_row(row, u, T=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """The token of one row of float64 logits (ties to the lower index)."""
    row = np.where(np.isnan(row), -np.inf, row).astype(np.float64)
    if np.isneginf(row).all():
        row = np.zeros_like(row)
    order = np.argsort(-row, kind="stable")
    if not T > 0:
        top_k, T = 1, 1.0
    if top_k > 0:
        order = order[:top_k]
    top = row[order[0]]

    def weigh(i):
        with np.errstate(invalid="ignore"):
            return np.where(row[i] == top, 1.0, np.exp(np.nan_to_num((row[i] - top) / T, nan=-np.inf)))
    w = weigh(order)
    if top_p < 1:
        before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
        n = max(1, int((before < top_p * w.sum()).sum()))
        order, w = order[:n], w[:n]
    if min_p > 0:  # in exponents: next to a weight of 1, exp itself rounds to 1
        with np.errstate(invalid="ignore"):
            e = np.where(row[order] == top, 0.0, np.nan_to_num((row[order] - top) / T, nan=-np.inf))
        order = order[e >= math.log(min(min_p, 1.0))]
    kept = np.sort(order)
    mass = np.cumsum(weigh(kept))
    return int(kept[min(np.searchsorted(mass, u * mass[-1], side="right"), len(kept) - 1)])
