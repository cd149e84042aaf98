"""The operators at the two ends of a language model's training step, and the log
probabilities that a server gives with its tokens, as cases for timing them.

The kinds:
  embed     embedding_lookup: row i is scale * weight[ids[i]]; with "train" also its
            gradient, row v of which is scale times the sum of the rows of dy whose id is
            v (none for the padding id).
  logprobs  token_logprobs: per row of logits the log probability of a given token, the
            entropy and the `top` likeliest tokens (equal ones by index) with their log
            probabilities; with "train" the gradient of the logits for gradients of the
            log probabilities and, where it is computed, of the entropy.
  clip      clip_grad_norm_: the norm over the gradients of many parameters, and the
            gradients times min(1, max_norm / (norm + 1e-6)) in place.
"""
import math
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PACKAGE = os.path.join(ROOT, "prime-moment-attention_amd")
if PACKAGE not in sys.path:
    sys.path.insert(0, PACKAGE)

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
IGNORE = -100


def _embed(dtype, B, L, V, C, train=False, scale=1.0, pad=0.0):
    return {"kind": "embed", "dtype": dtype, "B": B, "L": L, "V": V, "C": C, "train": train, "scale": scale, "pad": pad}


def _logprobs(dtype, n, V, top=0, entropy=False, train=False):
    return {"kind": "logprobs", "dtype": dtype, "n": n, "V": V, "top": top, "entropy": entropy, "train": train}


def _clip(dtype, layers, width, V, clips=True):
    return {"kind": "clip", "dtype": dtype, "layers": layers, "width": width, "V": V, "clips": clips}


def listed():
    cases = {
        # the embedding of the next token of one conversation: the launch is what counts
        "embed_bf16_b1": _embed("bf16", 1, 1, 50304, 768),
        # the embedding of a batch of long prompts, scaled by the root of the width
        "embed_bf16_b8_8192": _embed("bf16", 8, 8192, 50304, 768, scale=math.sqrt(768)),
        # a training step at the model's context length: 65536 tokens, frequent ones many times
        "embed_train_bf16_b32_2048": _embed("bf16", 32, 2048, 50304, 768, train=True),
        # a small fp32 step, half of it padding, rows off every vector
        "embed_train_f32_b3_777": _embed("f32", 3, 777, 32000, 501, train=True, scale=2.5, pad=0.5),
        # the next token of one conversation, answered with its 20 likeliest alternatives
        "logprobs_bf16_b1": _logprobs("bf16", 1, 50304, top=20),
        # a full serving batch, with 5 alternatives and the entropy
        "logprobs_bf16_b256": _logprobs("bf16", 256, 50304, top=5, entropy=True),
        # the loss of a training step and its gradient
        "logprobs_train_bf16_8192": _logprobs("bf16", 8192, 50304, train=True),
        # a policy's step with an entropy bonus: fp32, an odd vocabulary, rows off every vector
        "logprobs_train_f32_777": _logprobs("f32", 777, 32001, entropy=True, train=True),
        # the gradients of a small model
        "clip_f32_small": _clip("f32", 2, 64, 500),
        # the gradients of a model of the PRIME-125M width, twelve layers
        "clip_bf16_125m": _clip("bf16", 12, 768, 50304),
        # the same in fp32
        "clip_f32_125m": _clip("f32", 12, 768, 50304),
        # bf16 gradients among fp32 ones of odd sizes, below the limit: the norm alone
        "clip_mixed_odd_idle": _clip("mixed", 6, 501, 32001, clips=False),
    }
    return [dict(case, name=name) for name, case in cases.items()]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["embed", "embed", "logprobs", "logprobs", "clip"])
    dtype = rng.choice(["bf16", "bf16", "f32", "f16"])
    if kind == "embed":
        C = _log(rng, 64, 4096)
        V = _log(rng, 256, min(160000, 80000000 // C))
        n = _log(rng, 1, 50000000 // C)
        B = _log(rng, 1, min(n, 64))
        return _embed(dtype, B, max(1, n // B), V, C, train=rng.random() < 0.6,
                      scale=rng.choice([1.0, round(math.sqrt(C), 3)]), pad=rng.choice([0.0, 0.0, 0.1, 0.5]))
    if kind == "logprobs":
        V = _log(rng, 256, 160000)
        if rng.random() < 0.5:
            return _logprobs(dtype, _log(rng, 1, 200000000 // V), V, entropy=rng.random() < 0.4, train=True)
        return _logprobs(dtype, _log(rng, 1, min(1024, 25000000 // V)), V, top=rng.choice([0, 1, 5, 10, 20]),
                         entropy=rng.random() < 0.5)
    width = _log(rng, 32, 1024)
    return _clip(rng.choice(["bf16", "f32", "f16", "mixed"]), rng.randint(1, 16), width,
                 _log(rng, 256, min(100000, 60000000 // width)), clips=rng.random() < 0.7)


# ---------------------------------------------------------------- inputs

def _tokens(rand, V):
    """Ids whose frequency falls with the id, as ranked words' does."""
    return (torch.exp(rand * math.log(V + 1)) - 1).long().clamp(0, V - 1)


def _shapes(case):
    """The parameters of a model: embeddings, then per layer the projections, the QK norms
    over heads of 64, the two norms and a gated MLP, then the last norm."""
    W, M = case["width"], 8 * case["width"] // 3
    layer = [(W, W)] * 4 + [(64,)] * 4 + [(W,)] * 2 + [(M, W), (M, W), (W, M)]
    return [(case["V"], W)] + layer * case["layers"] + [(W,)]


def _buckets(case):
    """The gradients' buckets, as (dtype, shapes): one after the other, up to a twentieth of the
    model each; in mixed models the vectors are fp32 in buckets of their own."""
    shapes = _shapes(case)
    limit = sum(math.prod(s) for s in shapes) // 20
    mixed = case["dtype"] == "mixed"
    kinds = [DTYPES["f32" if mixed and len(s) == 1 else "bf16" if mixed else case["dtype"]] for s in shapes]
    out = []
    for dt in dict.fromkeys(kinds):
        size = limit
        for s in (s for s, k in zip(shapes, kinds) if k is dt):
            if size >= limit:
                out.append((dt, []))
                size = 0
            out[-1][1].append(s)
            size += math.prod(s)
    return out


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(1000003 * seed + 29)
    randn = lambda *shape: torch.randn(*shape, generator=g, device="cuda")
    rand = lambda *shape: torch.rand(*shape, generator=g, device="cuda")
    if case["kind"] == "embed":
        dt, B, L, V, C = (case[k] for k in ("dtype", "B", "L", "V", "C"))
        ids = _tokens(rand(B, L), V)
        if case["pad"]:
            ids = torch.where(rand(B, L) < case["pad"], V - 1, ids)
        d = {"ids": ids, "weight": (0.02 * randn(V, C)).to(DTYPES[dt])}
        if case["train"]:
            d["dy"] = randn(B, L, C).to(DTYPES[dt])
        return d
    if case["kind"] == "logprobs":
        n, V = case["n"], case["V"]
        logits = randn(n, V) * (1.0 + 3.0 * rand(n, 1))
        if not case["train"]:  # a tenth of the rows with two thirds of the tokens banned
            logits.masked_fill_((rand(n, 1) < 0.1) & (rand(n, V) < 0.67), -math.inf)
        logits = logits.to(DTYPES[case["dtype"]])
        # tokens as the model draws them; in training a tenth of the rows has none
        tokens = (logits - torch.empty(n, V, device="cuda").exponential_(generator=g).log_()).argmax(1)
        d = {"logits": logits}
        if case["train"]:
            tokens = torch.where(rand(n) < 0.1, IGNORE, tokens)
            unit = (65536.0 if case["dtype"] == "f16" else 1.0) / n  # fp16 trains on a scaled loss
            d["dlogprobs"] = -unit * (0.5 + rand(n))
            if case["entropy"]:
                d["dentropy"] = -0.1 * unit * torch.ones(n, device="cuda")
        return dict(d, tokens=tokens)
    buckets = _buckets(case)
    count = sum(math.prod(s) for _, shapes in buckets for s in shapes)
    # a norm of about 8, spread unevenly over the buckets
    parts = [(8 / math.sqrt(count) * randn(sum(math.prod(s) for s in shapes)) * (0.2 + 1.6 * rand(1))).to(dt)
             for dt, shapes in buckets]
    return {"buckets": parts, "shapes": [shapes for _, shapes in buckets]}


def prepare(case, seed):
    d = _inputs(case, seed)
    if case["kind"] == "clip":
        params = []
        for bucket, shapes in zip(d["buckets"], d["shapes"]):
            for part, s in zip(bucket.split([math.prod(s) for s in shapes]), shapes):
                p = torch.nn.Parameter(torch.empty(s, device="cuda", dtype=bucket.dtype))
                p.grad = part.view(s)
                params.append(p)
        d.update(params=params, max_norm=1.0 if case["clips"] else 1000.0)
    elif case["train"]:
        d["weight" if case["kind"] == "embed" else "logits"].requires_grad_()
    return dict(d, case=case)


def _limit(d):
    """The limit of this pass: it falls a little from one to the next, so that gradients
    that the last pass clipped are over it again."""
    d["max_norm"] *= 1.0 if not d["case"]["clips"] else 0.99995 if d["case"]["dtype"] == "f16" else 0.9995
    return d["max_norm"]


# ---------------------------------------------------------------- plain forms

def _plain_embed(d):
    case, ids, weight = d["case"], d["ids"], d["weight"].detach()
    y = (weight[ids].float() * case["scale"]).to(weight.dtype)
    if not case["train"]:
        return y
    dy = d["dy"].float().view(-1, case["C"])
    if case["pad"]:
        dy = dy * (ids != case["V"] - 1).view(-1, 1)
    grad = torch.zeros(weight.shape, device=dy.device).index_add_(0, ids.view(-1), dy) * case["scale"]
    return y, grad.to(weight.dtype)


def _plain_logprobs(d):
    case, tokens = d["case"], d["tokens"]
    x = d["logits"].detach().float()
    n, V = x.shape
    shifted = x - x.amax(1, keepdim=True)
    e = torch.exp(shifted)
    total = e.sum(1, keepdim=True)
    log_total = torch.log(total)
    known = tokens != IGNORE
    at = tokens.clamp(min=0).unsqueeze(1)
    out = [torch.where(known, (shifted.gather(1, at) - log_total).squeeze(1), 0.0)]
    if case["entropy"]:
        mean = (torch.where(e > 0, e * shifted, 0.0).sum(1, keepdim=True) / total)
        out.append((log_total - mean).squeeze(1))
    if case["top"]:
        ranked, order = shifted.sort(dim=1, descending=True, stable=True)
        out += [ranked[:, :case["top"]] - log_total, order[:, :case["top"]]]
    if case["train"]:
        p = e / total
        g = torch.where(known, d["dlogprobs"], 0.0).unsqueeze(1)
        dx = -g * p
        dx.scatter_add_(1, at, g)
        if case["entropy"]:
            dx -= d["dentropy"].unsqueeze(1) * p * (shifted - mean)
        out.append(dx.to(d["logits"].dtype))
    return tuple(out)


def _plain_clip(d):
    limit, grads = _limit(d), [p.grad for p in d["params"]]
    norm = torch.stack([g.float().square().sum() for g in grads]).double().sum().sqrt()
    c = (limit / (norm + 1e-6)).clamp(max=1.0).float()
    [g.copy_(g.float() * c) for g in grads]
    return (norm.float(), *d["buckets"])


# ---------------------------------------------------------------- one pass

def _own_embed(d):
    from prime_moment_attention import embedding_lookup
    case = d["case"]
    y = embedding_lookup(d["ids"], d["weight"], scale=case["scale"],
                         padding_idx=case["V"] - 1 if case["pad"] else None)
    if not case["train"]:
        return y
    return y.detach(), *torch.autograd.grad(y, [d["weight"]], d["dy"])


def _own_logprobs(d):
    from prime_moment_attention import token_logprobs
    case = d["case"]
    r = token_logprobs(d["logits"], d["tokens"], top=case["top"], entropy=case["entropy"], ignore_index=IGNORE)
    out = [r.logprobs.detach()]
    if case["entropy"]:
        out.append(r.entropy.detach())
    if case["top"]:
        out += [r.top_logprobs, r.top_tokens]
    if case["train"]:
        outputs = [r.logprobs] + ([r.entropy] if case["entropy"] else [])
        out += torch.autograd.grad(outputs, [d["logits"]], [d[k] for k in ("dlogprobs", "dentropy") if k in d])
    return tuple(out)


def _own_clip(d):
    from prime_moment_attention import clip_grad_norm_
    return (clip_grad_norm_(d["params"], _limit(d)), *d["buckets"])


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"embed": _own_embed, "logprobs": _own_logprobs, "clip": _own_clip}[kind](state)
    return {"embed": _plain_embed, "logprobs": _plain_logprobs, "clip": _plain_clip}[kind](state)


# ---------------------------------------------------------------- float64

def _exact_embed(case, d):
    """The gradient as differences of the running sum over the tokens in sorted order."""
    rows = d["weight"].double().mul(case["scale"])
    y = rows.index_select(0, d["ids"].flatten()).view(*d["ids"].shape, -1)
    if not case["train"]:
        return y
    order = d["ids"].flatten().argsort()
    counts = torch.bincount(d["ids"].flatten(), minlength=case["V"])
    ends = counts.cumsum(0)
    sums = torch.zeros_like(rows)
    for c in range(0, case["C"], 128):
        part = d["dy"].view(-1, case["C"])[:, c:c + 128].double()[order].cumsum(0)
        part = torch.cat([torch.zeros_like(part[:1]), part])
        sums[:, c:c + 128] = part[ends] - part[ends - counts]
    if case["pad"]:
        sums[case["V"] - 1] = 0
    return y, sums * case["scale"]


def _exact_logprobs(case, d):
    """By logsumexp, and the gradients by autograd through it."""
    x = d["logits"].double().requires_grad_(case["train"])
    logp = x - torch.logsumexp(x, 1, keepdim=True)
    known = d["tokens"] >= 0
    rows = torch.arange(case["n"], device=x.device)
    out = [torch.where(known, logp[rows, torch.where(known, d["tokens"], 0)], 0.0)]
    if case["entropy"]:
        out.append(-torch.xlogy(logp.exp(), logp.exp()).sum(1) if not case["train"] else -(logp.exp() * logp).sum(1))
    outputs = list(out)
    if case["top"]:
        out += [logp.topk(case["top"], 1).values, None]
    if case["train"]:
        out += torch.autograd.grad(outputs, [x], [d[k].double() for k in ("dlogprobs", "dentropy") if k in d])
    return tuple(None if t is None else t.detach() for t in out)


def _exact_clip(case, d):
    norm = math.sqrt(sum(float(torch.linalg.vector_norm(b.double())) ** 2 for b in d["buckets"]))
    limit = 1000.0 if not case["clips"] else 0.99995 if case["dtype"] == "f16" else 0.9995
    factor = min(1.0, limit / (norm + 1e-6))
    return (norm, *(b.double() * factor for b in d["buckets"]))


def exact(case, seed):
    d = _inputs(case, seed)
    return {"embed": _exact_embed, "logprobs": _exact_logprobs, "clip": _exact_clip}[case["kind"]](case, d)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    if case["kind"] == "embed":
        es, n, V, C = DTYPES[case["dtype"]].itemsize, case["B"] * case["L"], case["V"], case["C"]
        # the rows that are asked for at all, by the ids' distribution
        v = torch.arange(1, V + 1, dtype=torch.float64)
        share = (1 - case["pad"]) * torch.log1p(1 / v) / math.log(V + 1)
        forward = 8 * n + es * C * (n + int((1 - (1 - share) ** n).sum()))
        return {"bytes": forward + (es * C * (n + V) if case["train"] else 0), "flops": n * C * (2 if case["train"] else 1)}
    if case["kind"] == "logprobs":
        es, n, V = DTYPES[case["dtype"]].itemsize, case["n"], case["V"]
        out = n * (12 + 4 * case["entropy"] + 12 * case["top"])
        return {"bytes": n * V * es * (2 if case["train"] else 1) + out,
                "flops": n * V * (4 + 2 * case["entropy"]) * (2 if case["train"] else 1)}
    count = [(dt.itemsize, sum(math.prod(s) for s in shapes)) for dt, shapes in _buckets(case)]
    return {"bytes": sum(es * n for es, n in count) * (2 if case["clips"] else 1) + 4,
            "flops": sum(n for _, n in count) * (3 if case["clips"] else 2)}
