"""What the operators between and inside 4-bit decoder blocks cost: cases, inputs, plain forms and 64-bit values.

Four operators are measured, each through the call a user makes:

* ``quantize``: :func:`economize_b200.ops.fp4_quantize` of activations, and its values (``dequantize``);
* ``product``: :func:`economize_b200.ops.linear` of bf16 activations with an
  :class:`~economize_b200.ops.fp4.FP4Weight`: the activations are quantised and both operands multiplied in 4 bits;
* ``norm``: :func:`economize_b200.ops.block_norm`, the norm after a block, its gate and residual scale, the residual
  sum and the norm before the next block, alone or with all gradients;
* ``chain``: the same norm with its result in 4 bits, and the product that reads it.

``run`` computes them in elementary 32-bit operations while ``own`` is false and makes the package's calls while it
is true. ``exact`` holds the same outputs in 64 bits.

The 4-bit formats hold E2M1 values (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives; ties to the even code). ``mxfp4``:
one power of two per 32 columns, ``2^(E - 2)`` for a largest magnitude of exponent ``E``, twice that when its mantissa
is 1.75 or more. ``nvfp4``: one power of two per row, the smallest that is no less than the row's largest magnitude
over 2688, and one e4m3 scale per 16 columns, their largest magnitude over 6 in units of the row's (at least 2^-9).
"""

from __future__ import annotations

import math

import torch

own = False

EPS = 1e-5
GROUP = {"nvfp4": 16, "mxfp4": 32}

CASES = [
    # one token before an attention projection: what a call costs at least
    dict(name="quantize one token", op="quantize", rows=1, cols=4096, fmt="nvfp4"),
    # a prompt before the down projection of an 8B decoder
    dict(name="quantize prompt", op="quantize", rows=8192, cols=14336, fmt="mxfp4"),
    # the output projection of one decoded token
    dict(name="product one token", op="product", rows=1, cols=4096, out=4096, fmt="nvfp4"),
    # gate and up projections of a verified draft tree
    dict(name="product draft tree", op="product", rows=61, cols=4096, out=28672, fmt="nvfp4"),
    # sizes that no tile divides
    dict(name="product odd sizes", op="product", rows=1003, cols=1056, out=1000, fmt="mxfp4"),
    # gate and up projections of a long prompt
    dict(name="product prompt", op="product", rows=8192, cols=4096, out=28672, fmt="nvfp4"),
    # norms on both sides of a block, a draft tree
    dict(name="norm draft tree", op="norm", rows=61, hidden=4096, dtype="bf16", post=True, gate="none", scale=1.0,
         grad=False),
    # a scaled residual and the next block's norm, a long prompt
    dict(name="norm prompt", op="norm", rows=8192, hidden=4096, dtype="bf16", post=False, gate="none", scale=0.22,
         grad=False),
    # a pre-norm block of a packed training row
    dict(name="norm training row", op="norm", rows=8192, hidden=4096, dtype="bf16", post=False, gate="none",
         scale=1.0, grad=True),
    # a gated block with both norms, trained in 32 bits, sizes that no vector divides
    dict(name="norm gated training", op="norm", rows=2047, hidden=1001, dtype="fp32", post=True, gate="token",
         scale=0.5, grad=True),
    # a draft tree's norm and attention projection
    dict(name="chain draft tree", op="chain", rows=61, cols=4096, out=6144, fmt="nvfp4", post=False),
    # a prompt's norms on both sides of a block and the next attention projection
    dict(name="chain prompt", op="chain", rows=4096, cols=4096, out=6144, fmt="mxfp4", post=True),
]

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [dict(c) for c in CASES]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["quantize", "product", "product", "norm", "norm", "chain"])
    if op == "norm":
        case = dict(op=op, rows=_log_uniform(rng, 1, 16384), hidden=_log_uniform(rng, 64, 8192),
                    dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), post=rng.random() < 0.5,
                    gate=rng.choice(["none", "none", "token", "full"]), scale=rng.choice([1.0, 1.0, 0.22, 0.5]),
                    grad=rng.random() < 0.5)
        if rng.random() < 0.5:
            case["hidden"] = (case["hidden"] + 63) // 64 * 64
        limit = 8192 * 4096 // (2 if case["dtype"] == "fp32" or case["gate"] == "full" else 1)
        while case["rows"] * case["hidden"] > limit:
            case["rows"] = case["rows"] * 3 // 4
        return case
    case = dict(op=op, rows=_log_uniform(rng, 1, 8192), cols=32 * _log_uniform(rng, 4, 448),
                fmt=rng.choice(["nvfp4", "mxfp4"]))
    if op == "quantize":
        return case
    case["out"] = _log_uniform(rng, 64, 28672)
    if rng.random() < 0.5:
        case["out"] = (case["out"] + 127) // 128 * 128
    if op == "chain":
        case["post"] = rng.random() < 0.5
    while case["rows"] * case["cols"] * case["out"] > 8192 * 4096 * 28672:
        case["rows"] = case["rows"] * 3 // 4
    return case


# ---- inputs --------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(*shape, device="cuda", generator=gen) * std

    def activations(rows, cols, dtype=torch.bfloat16):
        # tokens of different size, a few large channels
        size = torch.exp(0.5 * normal(rows, 1))
        channel = torch.exp(0.6 * normal(1, cols))
        return (normal(rows, cols) * size * channel).to(dtype)

    state = dict(case)
    if case["op"] == "norm":
        n, h, dtype = case["rows"], case["hidden"], DTYPES[case["dtype"]]
        grad = case["grad"]
        state["x"] = activations(n, h, dtype).requires_grad_(grad)
        state["residual"] = (2.0 * activations(n, h).float()).to(dtype).requires_grad_(grad)
        state["weight"] = (1.0 + normal(h, std=0.2)).to(dtype).requires_grad_(grad)
        state["post_weight"] = (0.5 + normal(h, std=0.1)).to(dtype).requires_grad_(grad) if case["post"] else None
        state["gate_values"] = None
        if case["gate"] != "none":
            width = 1 if case["gate"] == "token" else h
            state["gate_values"] = torch.sigmoid(normal(n, width)).to(dtype).requires_grad_(grad)
        if grad:
            state["dnormed"] = normal(n, h, std=0.02).to(dtype)
            state["dstream"] = normal(n, h, std=0.02).to(dtype)
        return state
    state["x"] = activations(case["rows"], case["cols"])
    if case["op"] == "quantize":
        return state
    state["w"] = normal(case["out"], case["cols"], std=0.02).to(torch.bfloat16)
    if case["op"] == "chain":
        h = case["cols"]
        state["residual"] = (2.0 * activations(case["rows"], h).float()).to(torch.bfloat16)
        state["weight"] = (1.0 + normal(h, std=0.2)).to(torch.bfloat16)
        state["post_weight"] = (0.5 + normal(h, std=0.1)).to(torch.bfloat16) if case["post"] else None
    if own:
        state["handle"] = _handle(state)  # the 4-bit weight that a model keeps
    else:
        state["values"] = _fp4_values(state["w"], case["fmt"])
    return state


def _handle(state):
    from economize_b200.ops.fp4 import FP4Weight

    return FP4Weight.from_weight(state["w"], state["fmt"])


# ---- the calls -----------------------------------------------------------------------------------------------------
def run(state):
    if own:
        return _own(state)
    return {"quantize": _quantize, "product": _product, "norm": _norm, "chain": _chain}[state["op"]](state)


def _own(state):
    from economize_b200 import ops

    op = state["op"]
    if op == "quantize":
        return {"values": ops.fp4_quantize(state["x"], state["fmt"]).dequantize()}
    if op == "norm":
        normed, stream = ops.block_norm(state["x"], state["residual"], state["weight"],
                                        post_weight=state["post_weight"], gate=state["gate_values"],
                                        scale=state["scale"], eps=EPS)
        if not state["grad"]:
            return {"normed": normed, "stream": stream}
        wanted = _wanted(state)
        grads = torch.autograd.grad((normed, stream), list(wanted.values()), (state["dnormed"], state["dstream"]))
        return {"normed": normed.detach(), "stream": stream.detach(), **dict(zip(wanted, grads))}
    handle = state["handle"] if "handle" in state else _handle(state)
    if op == "product":
        return {"y": ops.linear(state["x"], handle)}
    normed, stream = ops.block_norm(state["x"], state["residual"], state["weight"], post_weight=state["post_weight"],
                                    eps=EPS, quantize=state["fmt"])
    return {"y": ops.linear(normed, handle), "stream": stream}


def _wanted(state):
    names = {"dx": "x", "dresidual": "residual", "dweight": "weight", "dpost": "post_weight", "dgate": "gate_values"}
    return {out: state[name] for out, name in names.items() if state[name] is not None}


# ---- plain forms ---------------------------------------------------------------------------------------------------
def _e2m1(a):
    """Magnitudes to the nearest E2M1 value, in 32 bits."""
    out = torch.zeros_like(a)
    for border, even_below, step in ((0.25, True, 0.5), (0.75, False, 0.5), (1.25, True, 0.5), (1.75, False, 0.5),
                                     (2.5, True, 1.0), (3.5, False, 1.0), (5.0, True, 2.0)):
        out += torch.where(a > border if even_below else a >= border, step, 0.0)
    return out


def _power(x):
    """2^x of whole x between -126 and 127, exactly."""
    return ((x.to(torch.int32) + 127) << 23).view(torch.float32)


def _fp4_values(x, fmt):
    """The values that ``x`` has in 4 bits."""
    rows, cols = x.shape
    g = x.float().view(rows, cols // GROUP[fmt], GROUP[fmt])
    top = g.abs().amax(-1, keepdim=True)
    if fmt == "mxfp4":
        mantissa, exponent = torch.frexp(top)  # in [0.5, 1)
        unit = _power((exponent - 3 + (mantissa >= 0.875)).clamp(-126, 125))
        q = _e2m1((g / unit).abs())
        return (torch.copysign(q, g) * unit).view(rows, cols).to(x.dtype)
    mantissa, exponent = torch.frexp(top.amax(1, keepdim=True) / 2688.0)
    row = _power((exponent - (mantissa == 0.5).int()).clamp(-100, 120))
    g = g / row
    scale = (top / row / 6.0).clamp(2.0 ** -9, 448.0).to(torch.float8_e4m3fn).float()
    q = _e2m1((g / scale).abs())
    return (torch.copysign(q, g) * scale * row).view(rows, cols).to(x.dtype)


@torch.no_grad()
def _quantize(state):
    return {"values": _fp4_values(state["x"], state["fmt"])}


@torch.no_grad()
def _product(state):
    x = _fp4_values(state["x"], state["fmt"]).float()
    return {"y": torch.matmul(x, state["values"].float().t()).to(torch.bfloat16)}


def _rms(v):
    return torch.rsqrt(v.pow(2).mean(-1, keepdim=True) + EPS)


@torch.no_grad()
def _norm(state):
    x, residual, w = (state[k].float() for k in ("x", "residual", "weight"))
    post = None if state["post_weight"] is None else state["post_weight"].float()
    gate = None if state["gate_values"] is None else state["gate_values"].float()
    factor = state["scale"] if gate is None else gate * state["scale"]
    xhat, ix = None, None
    branch = x
    if post is not None:
        ix = _rms(x)
        xhat = x * ix
        branch = xhat * post
    stream = residual + factor * branch
    inv = _rms(stream)
    shat = stream * inv
    dtype = state["x"].dtype
    out = {"normed": (shat * w).to(dtype), "stream": stream.to(dtype)}
    if not state["grad"]:
        return out
    dn = state["dnormed"].float()
    g = dn * w
    ds = state["dstream"].float() + inv * (g - shat * (g * shat).mean(-1, keepdim=True))
    db = ds * factor
    dx = db
    if post is not None:
        h = db * post
        dx = ix * (h - xhat * (h * xhat).mean(-1, keepdim=True))
    out["dx"] = dx.to(dtype)
    out["dresidual"] = ds.to(dtype)
    out["dweight"] = (dn * shat).sum(0).to(dtype)
    if post is not None:
        out["dpost"] = (db * xhat).sum(0).to(dtype)
    if gate is not None:
        dgate = ds * branch * state["scale"]
        out["dgate"] = (dgate.sum(-1, keepdim=True) if gate.shape[1] == 1 else dgate).to(dtype)
    return out


@torch.no_grad()
def _chain(state):
    out = _norm({**state, "gate_values": None, "scale": 1.0, "grad": False})
    x = _fp4_values(out["normed"], state["fmt"]).float()
    y = torch.matmul(x, state["values"].float().t()).to(torch.bfloat16)
    return {"y": y, "stream": out["stream"]}


# ---- what a pass cannot do without ---------------------------------------------------------------------------------
def work(case):
    n = case["rows"]
    if case["op"] == "norm":
        h, size = case["hidden"], 4 if case["dtype"] == "fp32" else 2
        whole, gates = n * h * size, {"none": 0, "token": n * size, "full": n * h * size}[case["gate"]]
        weights = h * size * (2 if case["post"] else 1)
        total, flops = 4 * whole + gates + weights, 10 * n * h
        if case["grad"]:  # the outputs' gradients read, all inputs' written (one tensor where two are the same)
            same = not case["post"] and case["gate"] == "none" and case["scale"] == 1.0
            total += (3 if same else 4) * whole + gates + weights
            flops += 30 * n * h
        return {"bytes": total, "flops": flops}
    k, fmt = case["cols"], case["fmt"]
    if case["op"] == "quantize":
        return {"bytes": 4 * n * k, "flops": 4 * n * k}
    out = case["out"]
    stored = out * (k // 2 + k // GROUP[fmt]) + (4 * out if fmt == "nvfp4" else 0)
    total, flops = 2 * n * k + stored + 2 * n * out, 2 * n * k * out
    if case["op"] == "chain":
        total += 4 * n * k + 2 * k * (2 if case["post"] else 1)
    return {"bytes": total, "flops": flops}


# ---- 64 bits -------------------------------------------------------------------------------------------------------
@torch.no_grad()
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "quantize":
        return {"values": _exact_fp4(state["x"], case["fmt"])}
    if case["op"] == "norm":
        return _exact_norm(state)
    w = _exact_fp4(state["w"], case["fmt"])
    if case["op"] == "product":
        return {"y": _exact_matmul(_exact_fp4(state["x"], case["fmt"]), w)}
    parts = _exact_norm({**state, "gate_values": None, "scale": 1.0, "grad": False})
    # the norm's result is rounded to the input's type before it is quantised
    normed = parts["normed"].to(torch.float32).to(torch.bfloat16)
    return {"y": _exact_matmul(_exact_fp4(normed, case["fmt"]), w), "stream": parts["stream"]}


def _exact_matmul(x, w):
    return torch.cat([rows @ w.t() for rows in x.split(4096)])


def _exact_fp4(x, fmt):
    """The nearest values of the format, found by distance."""
    size = GROUP[fmt]
    v = x.detach().double().unflatten(-1, (-1, size))
    top = v.abs().amax(-1, keepdim=True)
    if fmt == "mxfp4":
        exponent = torch.floor(torch.log2(top.clamp_min(2.0 ** -124)))
        exponent += (top >= 1.75 * torch.exp2(exponent)).double()
        unit = torch.exp2((exponent - 2).clamp(-126, 125))
    else:
        row = top.amax(1, keepdim=True) / 2688
        row = torch.exp2(torch.ceil(torch.log2(row.clamp_min(2.0 ** -100))))
        scale = (top / (6 * row)).clamp(2.0 ** -9, 448)
        spacing = torch.exp2(torch.floor(torch.log2(scale)).clamp_min(-6) - 3)
        unit = torch.round(scale / spacing) * spacing * row
    v = v / unit
    a = v.abs().clamp(max=6)
    # spacing of the values: 0.5 below 2, 1 below 4, 2 above; halves go to the even multiple
    spacing = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).double()
    q = torch.round(a / spacing) * spacing
    return (torch.sign(v) * q * unit).flatten(-2)


def _exact_norm(state):
    with torch.enable_grad():
        leaf = {}
        for name in ("x", "residual", "weight", "post_weight", "gate_values"):
            if state[name] is not None:
                leaf[name] = state[name].detach().double().requires_grad_(state["grad"])
        branch = leaf["x"]
        if "post_weight" in leaf:
            branch = branch / torch.sqrt(branch.square().mean(-1, keepdim=True) + EPS) * leaf["post_weight"]
        if "gate_values" in leaf:
            branch = branch * leaf["gate_values"]
        stream = leaf["residual"] + state["scale"] * branch
        normed = stream / torch.sqrt(stream.square().mean(-1, keepdim=True) + EPS) * leaf["weight"]
        out = {"normed": normed.detach(), "stream": stream.detach()}
        if state["grad"]:
            names = {"dx": "x", "dresidual": "residual", "dweight": "weight", "dpost": "post_weight",
                     "dgate": "gate_values"}
            names = {k: n for k, n in names.items() if n in leaf}
            grads = torch.autograd.grad((normed, stream), [leaf[n] for n in names.values()],
                                        (state["dnormed"].double(), state["dstream"].double()))
            out.update(zip(names, grads))
    return out
