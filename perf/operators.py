"""What the operators of a training step over packed documents cost: cases, inputs, plain forms and 64-bit values.

Two operators are measured, each through the call a user makes:

* ``attention``: :func:`economize_b200.ops.packed_attention`, causal attention over packed documents with grouped
  heads, the forward pass alone (scoring prompts) or with the gradients of queries, keys and values (training);
* ``readout``: :func:`economize_b200.ops.linear_cross_entropy`, the softmax cross-entropy of a vocabulary readout:
  the losses alone (scoring), with the gradient of the hidden states (a frozen head) or with the head's too.

``run`` computes them in elementary 32-bit operations while ``own`` is false and makes the package's calls while it
is true. ``exact`` holds the same outputs in 64 bits.
"""

from __future__ import annotations

import math
import random

import torch

own = False

IGNORE = -100

# Four head layouts: multi-head, and 4 or 8 query heads on a key head; head dimensions a tile holds whole or not.
ATTENTION = [
    # one token of each of four rows and two short drafts: what one call costs at least
    dict(name="attention few tokens", op="attention", tokens=24, docs=6, pad=0, heads=8, kv_heads=2, dim=64,
         grad=False),
    # scoring eight prompts packed into one row, heads of an 8B decoder
    dict(name="attention prompts", op="attention", tokens=8192, docs=8, pad=0, heads=32, kv_heads=8, dim=128,
         grad=False),
    # a training row of chat turns, many shorter than a tile, and the row's padding
    dict(name="attention chat turns", op="attention", tokens=4096, docs=48, pad=131, heads=32, kv_heads=8, dim=128,
         grad=True),
    # a training row of documents
    dict(name="attention documents", op="attention", tokens=8192, docs=5, pad=0, heads=32, kv_heads=8, dim=128,
         grad=True),
    # a small multi-head draft model on an odd number of tokens, head dimension 64
    dict(name="attention draft model", op="attention", tokens=5003, docs=3, pad=0, heads=12, kv_heads=12, dim=64,
         grad=True),
    # one long document
    dict(name="attention long document", op="attention", tokens=16384, docs=1, pad=0, heads=16, kv_heads=4, dim=128,
         grad=True),
]
READOUT = [
    # a handful of rows over a small head: what one call costs at least
    dict(name="readout few rows", op="readout", rows=16, hidden=1024, vocab=32000, masked=0.0, grad="both"),
    # scoring 1024 tokens of a prompt with a large vocabulary: losses only
    dict(name="readout scoring", op="readout", rows=1024, hidden=4096, vocab=128256, masked=0.0, grad="none"),
    # a drafter's own head over its draft vocabulary
    dict(name="readout draft head", op="readout", rows=4096, hidden=4096, vocab=32000, masked=0.0, grad="both"),
    # a frozen head under recovery adapters, the prompts' half of the rows masked
    dict(name="readout frozen head", op="readout", rows=8192, hidden=4096, vocab=128256, masked=0.5, grad="hidden"),
    # a vocabulary and a row count that no tile divides
    dict(name="readout odd sizes", op="readout", rows=2047, hidden=1000, vocab=50257, masked=0.1, grad="both"),
    # a whole batch with a trained head and a large vocabulary
    dict(name="readout trained head", op="readout", rows=8192, hidden=4096, vocab=128256, masked=0.0, grad="both"),
]


def listed():
    return [dict(c) for c in ATTENTION + READOUT]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    if rng.random() < 0.5:
        heads, kv_heads = rng.choice([(8, 8), (12, 12), (12, 4), (14, 2), (8, 1), (16, 4), (32, 8), (32, 4)])
        case = dict(op="attention", tokens=_log_uniform(rng, 16, 16384), docs=_log_uniform(rng, 1, 64), pad=0,
                    heads=heads, kv_heads=kv_heads, dim=rng.choice([64, 64, 80, 96, 128, 128, 128]),
                    grad=rng.random() < 0.7)
        case["docs"] = min(case["docs"], case["tokens"])
        # the plain form's padded scores: no more of them than the longest listed document's
        while case["docs"] * heads * max(lengths(case)) ** 2 > 16 * 16384 ** 2:
            case["tokens"] = case["tokens"] * 3 // 4
            case["docs"] = min(case["docs"], case["tokens"])
        if rng.random() < 0.4:
            case["pad"] = rng.randrange(1, 1 + case["tokens"] // 8)
        return case
    case = dict(op="readout", rows=_log_uniform(rng, 8, 8192), hidden=8 * _log_uniform(rng, 32, 512),
                vocab=_log_uniform(rng, 1000, 151936), masked=rng.choice([0.0, 0.0, 0.1, 0.5, 0.9]),
                grad=rng.choice(["none", "hidden", "both", "both"]))
    while case["rows"] * case["hidden"] * case["vocab"] > 8192 * 4096 * 128256:
        case["rows"] = case["rows"] * 3 // 4
    return case


def lengths(case):
    """The documents' lengths: spread over their logarithm, adding up to ``tokens``, by the case alone."""
    n, docs = case["tokens"], case["docs"]
    rng = random.Random(n * 1000003 + docs)
    weights = [math.exp(rng.uniform(0.0, 3.0)) for _ in range(docs)]
    total, out, used, seen = sum(weights), [], 0, 0.0
    for w in weights:
        seen += w
        upto = min(n, int(round(n * seen / total)))
        out.append(upto - used)
        used = upto
    out[-1] += n - used
    return out


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, device="cuda", generator=gen) * std).to(torch.bfloat16)

    if case["op"] == "attention":
        lens = lengths(case)
        rows, h, g, d = case["tokens"] + case["pad"], case["heads"], case["kv_heads"], case["dim"]
        cu = torch.tensor([0] + lens, device="cuda").cumsum(0).to(torch.int32)
        # rotated queries and keys are contiguous, values a part of the fused projection's rows
        q = normal(rows, h, d).requires_grad_(case["grad"])
        k = normal(rows, g, d).requires_grad_(case["grad"])
        fused = normal(rows, (h + 2 * g) * d)
        v = fused[:, (h + g) * d:].view(rows, g, d).detach().requires_grad_(case["grad"])
        state = dict(op="attention", q=q, k=k, v=v, cu=cu, longest=max(lens), grad=case["grad"])
        if case["grad"]:
            state["dout"] = normal(rows, h, d, std=0.02)
        return state
    n, h, v = case["rows"], case["hidden"], case["vocab"]
    weight = normal(v, h, std=0.02)
    targets = torch.randint(0, v, (n,), device="cuda", generator=gen)
    # normalised states that lean towards their target's row, from not at all to surely
    lean = torch.rand(n, 1, device="cuda", generator=gen) * 12.0
    rows = weight[targets].float()
    hidden = torch.randn(n, h, device="cuda", generator=gen) + lean * rows / rows.norm(dim=-1, keepdim=True)
    hidden = hidden.to(torch.bfloat16)
    order = torch.randperm(n, device="cuda", generator=gen)
    targets[order[: int(n * case["masked"])]] = IGNORE
    return dict(op="readout", hidden=hidden.requires_grad_(case["grad"] != "none"),
                weight=weight.requires_grad_(case["grad"] == "both"), targets=targets, grad=case["grad"])


def run(state):
    if own:
        return _own(state)
    return _attention(state) if state["op"] == "attention" else _readout(state)


def _own(state):
    from economize_b200 import ops

    if state["op"] == "attention":
        out = ops.packed_attention(state["q"], state["k"], state["v"], state["cu"])
        if not state["grad"]:
            return {"out": out}
        dq, dk, dv = torch.autograd.grad(out, (state["q"], state["k"], state["v"]), state["dout"])
        return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}
    if state["grad"] == "none":
        return {"losses": ops.linear_cross_entropy(state["hidden"], state["weight"], state["targets"],
                                                   ignore_index=IGNORE, reduction="none")}
    loss = ops.linear_cross_entropy(state["hidden"], state["weight"], state["targets"], ignore_index=IGNORE)
    if state["grad"] == "hidden":
        (dx,) = torch.autograd.grad(loss, (state["hidden"],))
        return {"loss": loss.detach(), "dx": dx}
    dx, dw = torch.autograd.grad(loss, (state["hidden"], state["weight"]))
    return {"loss": loss.detach(), "dx": dx, "dw": dw}


@torch.no_grad()
def _attention(state):
    """The documents padded to the longest: ``[B, H_kv, G, L, L]`` scores, a causal mask, softmax, and back."""
    q, k, v, cu = state["q"], state["k"], state["v"], state["cu"].long()
    n, heads, dim = q.shape
    kv, longest = k.shape[1], state["longest"]
    group, docs = heads // kv, cu.numel() - 1
    steps = torch.arange(longest, device=q.device)
    at = cu[:-1, None] + steps  # [B, L] the packed row of every padded position
    real = at < cu[1:, None]
    at = torch.where(real, at, 0)

    def padded(x, per):
        x = torch.where(real[..., None, None], x.float()[at], 0.0)  # [B, L, heads, D]
        return x.view(docs, longest, kv, per, dim).permute(0, 2, 3, 1, 4)

    def packed(x, per):
        x = x.permute(0, 3, 1, 2, 4).reshape(docs, longest, kv * per, dim)
        y = torch.zeros(n + 1, kv * per, dim, device=x.device)
        return y.index_copy_(0, torch.where(real, at, n).reshape(-1), x.flatten(0, 1))[:n].to(torch.bfloat16)

    scale = dim ** -0.5
    qs, ks, vs = padded(q, group), padded(k, 1), padded(v, 1)
    p = torch.matmul(qs, ks.transpose(-1, -2)).mul_(scale)
    p.masked_fill_(steps[None, :] > steps[:, None], float("-inf"))
    p.sub_(p.amax(-1, keepdim=True)).exp_()
    p.div_(p.sum(-1, keepdim=True))
    o = torch.matmul(p, vs)
    if not state["grad"]:
        return {"out": packed(o, group)}
    do = padded(state["dout"], group)
    dv = torch.matmul(p.flatten(2, 3).transpose(-1, -2), do.flatten(2, 3))
    ds = torch.matmul(do, vs.transpose(-1, -2)).sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    del p
    dq = torch.matmul(ds, ks)
    dk = torch.matmul(ds.flatten(2, 3).transpose(-1, -2), qs.flatten(2, 3))
    return {"out": packed(o, group), "dq": packed(dq, group), "dk": packed(dk[:, :, None], 1),
            "dv": packed(dv[:, :, None], 1)}


@torch.no_grad()
def _readout(state):
    """All logits at once, their softmax, and the two products of the gradients."""
    x, w, targets = state["hidden"].float(), state["weight"].float(), state["targets"]
    valid = targets != IGNORE
    at = torch.where(valid, targets, 0)[:, None]
    z = torch.matmul(x, w.t())
    picked = z.gather(1, at)[:, 0]
    top = z.amax(-1, keepdim=True)
    e = z.sub_(top).exp_()
    total = e.sum(-1, keepdim=True)
    nll = torch.where(valid, torch.log(total[:, 0]) + top[:, 0] - picked, 0.0)
    if state["grad"] == "none":
        return {"losses": nll}
    count = valid.sum().clamp_min(1)
    loss = nll.sum() / count
    dz = e.div_(total)
    dz.scatter_add_(1, at, torch.full_like(picked, -1.0)[:, None])
    dz.mul_((valid / count)[:, None])
    out = {"loss": loss, "dx": torch.matmul(dz, w).to(torch.bfloat16)}
    if state["grad"] == "both":
        out["dw"] = torch.matmul(dz.t(), x).to(torch.bfloat16)
    return out


def work(case):
    if case["op"] == "attention":
        rows, h, g, d = case["tokens"] + case["pad"], case["heads"], case["kv_heads"], case["dim"]
        pairs = h * sum(n * (n + 1) // 2 for n in lengths(case))
        # queries and output; keys and values; with gradients the output's and those of all three inputs too
        size = 2 * rows * d * (2 * h + 2 * g)
        if not case["grad"]:
            return {"bytes": size, "flops": 4 * d * pairs}
        return {"bytes": 2 * size, "flops": 14 * d * pairs}
    n = case["rows"] - int(case["rows"] * case["masked"])
    h, v = case["hidden"], case["vocab"]
    products = {"none": 1, "hidden": 2, "both": 3}[case["grad"]]
    size = 2 * n * h + 2 * v * h + 8 * case["rows"]
    if case["grad"] == "none":
        size += 4 * case["rows"]
    else:
        size += 4 + 2 * case["rows"] * h + (2 * v * h if case["grad"] == "both" else 0)
    return {"bytes": size, "flops": products * 2 * n * h * v}


@torch.no_grad()
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(state, lengths(case))
    return _exact_readout(state)


def _exact_attention(state, lens):
    """Document by document and head by head, in 64 bits."""
    q, k, v = (state[x].detach().double() for x in "qkv")
    heads, dim = q.shape[1], q.shape[2]
    group, scale = heads // k.shape[1], 1.0 / math.sqrt(dim)
    out = torch.zeros_like(q)
    grad = state["grad"]
    if grad:
        dout = state["dout"].double()
        dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    start = 0
    for n in lens:
        span = slice(start, start + n)
        start += n
        many = max(1, min(heads, 200_000_000 // max(1, n * n)))  # heads at a time
        for h0 in range(0, heads if n else 0, many):
            hs = torch.arange(h0, min(heads, h0 + many), device=q.device)
            qs, ks, vs = q[span][:, hs], k[span][:, hs // group], v[span][:, hs // group]
            s = torch.einsum("ihd,jhd->hij", qs, ks) * scale
            s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1), -math.inf)
            p = torch.exp(s - torch.logsumexp(s, -1, keepdim=True))
            del s
            out[span, h0:h0 + many] = torch.einsum("hij,jhd->ihd", p, vs)
            if grad:
                do = dout[span][:, hs]
                dp = torch.einsum("ihd,jhd->hij", do, vs)
                dv[span].index_add_(1, hs // group, torch.einsum("hij,ihd->jhd", p, do))
                ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
                del p, dp
                dq[span, h0:h0 + many] = torch.einsum("hij,jhd->ihd", ds, ks)
                dk[span].index_add_(1, hs // group, torch.einsum("hij,ihd->jhd", ds, qs))
    return {"out": out, "dq": dq, "dk": dk, "dv": dv} if grad else {"out": out}


def _exact_readout(state):
    """A thousand rows at a time, in 64 bits."""
    x, w, targets = state["hidden"].detach().double(), state["weight"].detach().double(), state["targets"]
    keep = (targets != IGNORE).nonzero()[:, 0]
    losses = torch.zeros(targets.numel(), dtype=torch.float64, device=x.device)
    dx = torch.zeros_like(x)
    dw = torch.zeros_like(w) if state["grad"] == "both" else None
    for rows in keep.split(1024):
        z = x[rows] @ w.t()
        logp = z.log_softmax(-1)
        del z
        losses[rows] = -logp.gather(1, targets[rows, None])[:, 0]
        if state["grad"] != "none":
            dz = logp.exp_()
            dz[torch.arange(rows.numel(), device=x.device), targets[rows]] -= 1.0
            dz /= max(1, keep.numel())
            dx[rows] = dz @ w
            if dw is not None:
                dw.addmm_(dz.t(), x[rows])
    if state["grad"] == "none":
        return {"losses": losses}
    out = {"loss": losses.sum() / max(1, keep.numel()), "dx": dx}
    if dw is not None:
        out["dw"] = dw
    return out
