"""The norms around a block against the same formulas in 64 bits, element by element, and their gradients.

Tolerances. ``half`` is the most a rounding to the operands' type moves a value by, ``eps / 2`` of it. What is computed
in fp32 (a norm: a sum of up to 16384 squares in at most 64 terms a thread, 32 lanes and 32 warps, a reciprocal square
root of 2 units; a handful of products) stays within ``2^-17`` of the sum of its terms' magnitudes; sums over tokens add
``T 2^-24`` of theirs. Without post norm and gate the backward pass reads the stream as it was rounded: ``half`` of it.
Values below the type's normal range are off by its smallest spacing besides.
"""

import pytest
import torch

from economize_b200 import ops
from economize_b200.ops.fp4 import FP4Weight

pytestmark = pytest.mark.gpu

F32 = 2.0 ** -17


def _make(dev, rows, hidden, dtype, post, gate, residual=True, seed=0, grad=False):
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, mean=0.0, std=1.0):
        return (mean + std * torch.randn(*shape, device=dev, generator=g)).to(dtype)

    t = dict(x=normal(rows, hidden, std=1.5), residual=normal(rows, hidden, std=2.0) if residual else None,
             weight=normal(hidden, mean=1.0, std=0.3), post_weight=normal(hidden, mean=0.6, std=0.2) if post else None,
             gate=None)
    if gate != "none":
        t["gate"] = torch.sigmoid(normal(rows, 1 if gate == "token" else hidden).float()).to(dtype)
    if grad:
        t = {k: None if v is None else v.requires_grad_() for k, v in t.items()}
    return t, normal(rows, hidden, std=0.1), normal(rows, hidden, std=0.1)


def _oracle(t, scale, eps, dn=None, ds_up=None):
    """64-bit outputs (and gradients), each with the bound of its error."""
    d = {k: None if v is None else v.detach().double() for k, v in t.items()}
    dtype = t["x"].dtype
    half, tiny = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    x, w = d["x"], d["weight"]
    gate = 1.0 if d["gate"] is None else d["gate"]
    post = d["post_weight"]
    ix = torch.ones_like(x[:, :1])
    if post is not None:
        ix = torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
    xh = x * ix
    pw = 1.0 if post is None else post
    b = xh * pw
    s = scale * gate * b + (0.0 if d["residual"] is None else d["residual"])
    s_mag = abs(scale) * gate * b.abs() + (0.0 if d["residual"] is None else d["residual"].abs())
    inv = torch.rsqrt(s.square().mean(-1, keepdim=True) + eps)
    sh, sh_mag = s * inv, s_mag * inv
    n = sh * w
    out = {"stream": (s, s.abs() * half + s_mag * F32 + tiny),
           "normed": (n, n.abs() * half + sh_mag * w.abs() * 2 * F32 + tiny)}
    if dn is None and ds_up is None:
        return out
    dn = torch.zeros_like(x) if dn is None else dn.double()
    up = torch.zeros_like(x) if ds_up is None else ds_up.double()
    simple = post is None and d["gate"] is None
    sh_err = sh_mag * 2 * F32 + (sh.abs() * half if simple else 0.0)
    rows = x.shape[0]
    g = dn * w
    m = (g * sh).mean(-1, keepdim=True)
    m_err = (g.abs() * sh_err).mean(-1, keepdim=True) + (g * sh).abs().mean(-1, keepdim=True) * F32
    ds = up + inv * (g - sh * m)
    ds_mag = up.abs() + inv * (g.abs() + sh.abs() * m.abs())
    ds_err = ds_mag * 2 * F32 + inv * (sh_err * m.abs() + (sh.abs() + sh_err) * m_err)
    total = rows * 2.0 ** -24 + F32

    def rounded(v, err):
        return v, v.abs() * half * 1.01 + err + tiny

    out["dresidual"] = rounded(ds, ds_err)
    out["dweight"] = rounded((dn * sh).sum(0), (dn.abs() * sh_err).sum(0) + (dn * sh).abs().sum(0) * total)
    db, db_err = scale * gate * ds, abs(scale) * gate * (ds_err + ds.abs() * F32)
    if d["gate"] is not None:
        dg, dg_err = scale * b * ds, abs(scale) * b.abs() * (ds_err + 2 * F32 * ds.abs())
        if d["gate"].shape[1] == 1:
            dg_err = dg_err.sum(-1, keepdim=True) + dg.abs().sum(-1, keepdim=True) * F32
            dg = dg.sum(-1, keepdim=True)
        out["dgate"] = rounded(dg, dg_err)
    if post is None:
        out["dx"] = rounded(db, db_err)
        return out
    h, h_err = db * post, db_err * post.abs()
    m = (h * xh).mean(-1, keepdim=True)
    m_err = (h_err * xh.abs()).mean(-1, keepdim=True) + (h * xh).abs().mean(-1, keepdim=True) * 2 * F32
    dx = ix * (h - xh * m)
    out["dx"] = rounded(dx, ix * (h_err + xh.abs() * m_err + (h.abs() + xh.abs() * m.abs()) * 2 * F32))
    out["dpost_weight"] = rounded((db * xh).sum(0), (db_err * xh.abs()).sum(0) + (db * xh).abs().sum(0) * total)
    return out


def _within(got, want, what):
    value, err = want
    off = (got.double() - value).abs()
    assert (off <= err).all(), f"{what}: {(off / err).max().item():.2f} times the bound"


def _call(t, scale, eps, **kw):
    return ops.block_norm(t["x"], t["residual"], t["weight"], post_weight=t["post_weight"], gate=t["gate"], scale=scale,
                          eps=eps, **kw)


DTYPES = [torch.bfloat16, torch.float16, torch.float32]
SIZES = [(1, 1), (1, 8), (2, 31), (3, 64), (7, 100), (5, 1000), (61, 4096), (33, 1001), (130, 2048), (700, 520), (9, 8200),
         (4, 16384), (3, 16383), (1300, 333), (1200, 4096)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,hidden", SIZES)
def test_forward(cuda, dtype, rows, hidden):
    for i, (post, gate, residual, scale) in enumerate([(False, "none", True, 1.0), (True, "none", True, 1.0),
                                                       (False, "token", True, 0.5), (True, "full", True, 0.22),
                                                       (True, "token", False, 2.0), (False, "none", False, 1.0)]):
        t, _, _ = _make(cuda, rows, hidden, dtype, post, gate, residual, seed=i)
        normed, stream = _call(t, scale, 1e-5)
        want = _oracle(t, scale, 1e-5)
        _within(normed, want["normed"], "normed")
        _within(stream, want["stream"], "stream")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,hidden", SIZES)
def test_gradients(cuda, dtype, rows, hidden):
    names = {"dx": "x", "dresidual": "residual", "dweight": "weight", "dpost_weight": "post_weight", "dgate": "gate"}
    for i, (post, gate, residual, scale) in enumerate([(False, "none", True, 1.0), (False, "none", True, 0.22),
                                                       (True, "none", True, 1.0), (False, "token", True, 0.5),
                                                       (False, "full", True, 1.0), (True, "token", True, 0.7),
                                                       (True, "full", True, 0.22), (True, "token", False, 1.0),
                                                       (False, "none", False, 1.0)]):
        t, dn, up = _make(cuda, rows, hidden, dtype, post, gate, residual, seed=10 + i, grad=True)
        wanted = {k: n for k, n in names.items() if t[n] is not None}
        normed, stream = _call(t, scale, 1e-5)
        got = torch.autograd.grad((normed, stream), [t[n] for n in wanted.values()], (dn, up))
        want = _oracle(t, scale, 1e-5, dn, up)
        for k, v in zip(wanted, got):
            assert v.dtype == dtype and v.shape == t[wanted[k]].shape
            _within(v, want[k], f"{k} (post={post} gate={gate} residual={residual} scale={scale})")


def test_one_output_and_single_gradients(cuda):
    for post, gate in ((False, "none"), (True, "token")):
        t, dn, up = _make(cuda, 40, 512, torch.bfloat16, post, gate, seed=30, grad=True)
        every = [v for v in t.values() if v is not None]
        for a, b in ((dn, None), (None, up)):
            normed, stream = _call(t, 0.5, 1e-5)
            got = torch.autograd.grad(normed if b is None else stream, [t["x"], t["residual"]], a if b is None else b,
                                      retain_graph=True)
            want = _oracle(t, 0.5, 1e-5, a, b)
            _within(got[0], want["dx"], "dx")
            _within(got[1], want["dresidual"], "dresidual")
            unused = torch.autograd.grad(normed if b is None else stream, every, a if b is None else b, allow_unused=True)
            assert all(v is not None for v in unused)
        full = torch.autograd.grad(_call(t, 0.5, 1e-5), every, (dn, up))
        for leaf, want in zip(every, full):  # one input that requires a gradient at a time
            solo = {k: None if v is None else v.detach().requires_grad_(v is leaf) for k, v in t.items()}
            (key,) = (k for k, v in t.items() if v is leaf)
            (got,) = torch.autograd.grad(_call(solo, 0.5, 1e-5), [solo[key]], (dn, up))
            assert torch.equal(got, want)


def test_gradients_against_differences(cuda):
    """Directional derivatives by central differences of the 32-bit operator: truncation of order step^2, rounding of
    2^-21 of the loss over the step."""
    t, dn, up = _make(cuda, 6, 96, torch.float32, True, "token", seed=31, grad=True)
    loss = lambda t: sum((o.double() * g.double()).sum() for o, g in zip(_call(t, 0.7, 1e-5), (dn, up)))  # noqa: E731
    grads = torch.autograd.grad(_call(t, 0.7, 1e-5), list(t.values()), (dn, up))
    mag = sum((o.double() * g.double()).abs().sum() for o, g in zip(_call(t, 0.7, 1e-5), (dn, up))).item()
    step = 2.0 ** -7
    g = torch.Generator(device=cuda).manual_seed(1)
    for name, grad in zip(t, grads):
        v = torch.randn(t[name].shape, device=cuda, generator=g)
        v = v / v.norm()
        with torch.no_grad():
            ends = [loss({**t, name: t[name] + f * v}) for f in (step, -step)]
            wide = [loss({**t, name: t[name] + f * v}) for f in (2 * step, -2 * step)]
        slope, coarse = ((a - b).item() for a, b in (ends, wide))
        slope, coarse = slope / (2 * step), coarse / (4 * step)
        want = (grad.double() * v.double()).sum().item()
        # the truncation error falls by four from the coarse step to the fine one: a third of their difference
        assert abs(slope - want) <= 0.5 * abs(slope - coarse) + mag * 2.0 ** -21 / step, name


def test_strides_and_offsets(cuda):
    g = torch.Generator(device=cuda).manual_seed(40)
    wide = torch.randn(50, 3 * 264, device=cuda, generator=g).bfloat16()
    w = torch.rand(264, device=cuda, generator=g).bfloat16()
    for x, r in ((wide[:, :264], wide[:, 264:528]), (wide[:, 3:267], wide[:, 264:528]), (wide[::2, :264], wide[1::2, 264:528]),
                 (wide[:1, :264], wide[1:2, 1:265]), (wide.t()[:264].t(), wide[:, 8:272])):
        a = ops.block_norm(x, r, w)
        b = ops.block_norm(x.contiguous(), r.contiguous(), w)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    # an odd base of the weights, a token gate out of a wider tensor, a broadcast gate
    odd = torch.rand(265, device=cuda, generator=g).bfloat16()[1:]
    gate = wide[:, 700:701]
    a = ops.block_norm(wide[:, :264], wide[:, 264:528], odd, gate=gate)
    b = ops.block_norm(wide[:, :264], wide[:, 264:528], odd.clone(), gate=gate.clone())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    half = torch.full((1, 1), 0.5, device=cuda, dtype=torch.bfloat16, requires_grad=True)
    x = wide[:, :264].clone().requires_grad_()
    normed, stream = ops.block_norm(x, wide[:, 264:528], w, gate=half.expand(50, 1))
    c = ops.block_norm(wide[:, :264], wide[:, 264:528], w, scale=0.5)
    assert torch.equal(normed, c[0]) and torch.equal(stream, c[1])
    (normed.float().sum() + stream.float().sum()).backward()
    assert half.grad.shape == (1, 1) and x.grad.shape == (50, 264)
    # upstream gradients that are broadcast or transposed
    y = wide[:, :264].clone().requires_grad_()
    n, s = ops.block_norm(y, None, w)
    (n.sum() + s.sum()).backward()
    z = wide[:, :264].clone().requires_grad_()
    one = torch.ones(50, 264, device=cuda, dtype=torch.bfloat16)
    torch.autograd.backward(ops.block_norm(z, None, w), (one, one))
    assert torch.equal(y.grad, z.grad)


def test_shapes_without_rows(cuda):
    w = torch.ones(64, device=cuda, requires_grad=True)
    x = torch.empty(0, 64, device=cuda, requires_grad=True)
    normed, stream = ops.block_norm(x, x, w)
    (normed.sum() + stream.sum()).backward()
    assert x.grad.shape == (0, 64) and torch.equal(w.grad, torch.zeros_like(w))
    y = torch.randn(2, 3, 5, 64, device=cuda)
    a, b = ops.block_norm(y, y, w.detach()), ops.block_norm(y.view(-1, 64), y.view(-1, 64), w.detach())
    assert a[0].shape == y.shape and torch.equal(a[0].view(-1, 64), b[0]) and torch.equal(a[1].view(-1, 64), b[1])
    assert torch.equal(ops.block_norm(y[0, 0, 0], None, w.detach())[0], b[0][0] * 0 + ops.block_norm(
        y.view(-1, 64)[:1], None, w.detach())[0][0])


def test_rows_that_are_not_finite_stay_by_themselves(cuda):
    t, dn, up = _make(cuda, 12, 256, torch.bfloat16, True, "token", seed=50)
    clean = [v.clone() for v in _call(t, 1.0, 1e-5)]
    t["x"][3, 7] = float("nan")
    t["residual"][5] = float("inf")
    got = _call(t, 1.0, 1e-5)
    keep = torch.ones(12, dtype=torch.bool, device=cuda)
    keep[[3, 5]] = False
    for a, b in zip(got, clean):
        assert torch.equal(a[keep], b[keep])
        assert not a[3].isfinite().any()
    assert not got[0][5].isfinite().any()
    zero = torch.zeros(2, 256, device=cuda, dtype=torch.bfloat16)  # a row of zeros: 0 / sqrt(eps)
    n, s = ops.block_norm(zero, zero, t["weight"], post_weight=t["post_weight"])
    assert not n.any() and not s.any()


def test_equal_bits_on_repeats_and_saved_memory(cuda):
    t, dn, up = _make(cuda, 3000, 1024, torch.bfloat16, True, "full", seed=60, grad=True)
    leaves = list(t.values())
    first = torch.autograd.grad(_call(t, 0.5, 1e-5), leaves, (dn, up))
    for _ in range(3):
        for a, b in zip(first, torch.autograd.grad(_call(t, 0.5, 1e-5), leaves, (dn, up))):
            assert torch.equal(a, b)
    out = _call(t, 0.5, 1e-5)
    twice = [torch.autograd.grad(out, leaves, (dn, up), retain_graph=True) for _ in range(2)]
    assert all(torch.equal(a, b) for a, b in zip(*twice))
    with torch.no_grad():
        t["x"].add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, leaves, (dn, up))


def test_training_graph(cuda):
    """Forward and backward passes captured into one CUDA graph and replayed on new inputs."""
    t, dn, up = _make(cuda, 300, 512, torch.bfloat16, True, "token", seed=70, grad=True)
    leaves = list(t.values())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(_call(t, 0.5, 1e-5), leaves, (dn, up))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _call(t, 0.5, 1e-5)
        grads = torch.autograd.grad(out, leaves, (dn, up))
    for seed in (71, 72):
        fresh, _, _ = _make(cuda, 300, 512, torch.bfloat16, True, "token", seed=seed, grad=True)
        with torch.no_grad():
            for k in t:
                t[k].copy_(fresh[k])
        graph.replay()
        want = _call(fresh, 0.5, 1e-5)
        for a, b in zip((*out, *grads), (*want, *torch.autograd.grad(want, list(fresh.values()), (dn, up)))):
            assert torch.equal(a, b)


def test_capture_beside_a_living_graph(cuda):
    """A captured call is refused while a graph of the default stream holds its leaves, and runs once that is gone."""
    t, dn, up = _make(cuda, 40, 64, torch.bfloat16, False, "none", seed=75, grad=True)
    leaves = [v for v in t.values() if v is not None]
    living = _call(t, 1.0, 1e-5)
    want = torch.autograd.grad(living, leaves, (dn, up), retain_graph=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with pytest.raises(RuntimeError, match="still holds a leaf"), torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
        _call(t, 1.0, 1e-5)
    with torch.no_grad():
        inference = torch.cuda.CUDAGraph()
        with torch.cuda.graph(inference, stream=side):
            again = _call(t, 1.0, 1e-5)
    inference.replay()
    assert all(torch.equal(a, b) for a, b in zip(again, living))
    del living
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        grads = torch.autograd.grad(_call(t, 1.0, 1e-5), leaves, (dn, up))
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(grads, want))


def test_autocast_and_refusals(cuda):
    t, dn, up = _make(cuda, 8, 64, torch.float32, True, "token", seed=80, grad=True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        normed, stream = _call(t, 1.0, 1e-5)
    assert normed.dtype == torch.bfloat16
    grads = torch.autograd.grad((normed, stream), list(t.values()), (dn.bfloat16(), up.bfloat16()))
    assert all(g.dtype == torch.float32 for g in grads)
    x, w = torch.randn(4, 64, device=cuda), torch.ones(64, device=cuda)
    for args, kw in (((x, None, w[:32]), {}), ((x, x[:2], w), {}), ((x, None, w.bfloat16()), {}),
                     ((x, None, w.cpu()), {}), ((x, None, w), {"post_weight": w[:1]}),
                     ((x, None, w), {"gate": x[:, :2]}), ((x, None, w), {"gate": x[:2, :1]}),
                     ((x, None, w), {"scale": float("inf")}), ((x, None, w), {"eps": -1.0}),
                     ((x, None, w), {"quantize": "int4"}), ((x.long(), None, w.long()), {})):
        with pytest.raises(ValueError):
            ops.block_norm(*args, **kw)
    with pytest.raises(ValueError):
        ops.block_norm(x.double(), None, w.double())
    with pytest.raises(ValueError):
        ops.block_norm(torch.zeros(1, 16392, device=cuda), None, torch.zeros(16392, device=cuda))
    with pytest.raises(ValueError):
        ops.block_norm(x, None, w, quantize="nvfp4")  # 4-bit results come from bf16
    y = torch.randn(4, 64, device=cuda, requires_grad=True)
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad(ops.block_norm(y, None, w)[0].sum(), y, create_graph=True)
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(lambda v: ops.block_norm(v, None, w)[0], (x,), (x,))


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("rows,hidden", [(1, 32), (3, 96), (61, 4096), (130, 1056), (700, 2048), (2, 16384), (1300, 64)])
def test_four_bits(cuda, fmt, rows, hidden):
    """The result in 4 bits is the 16-bit result quantised, bit for bit."""
    for i, (post, gate, residual) in enumerate([(False, "none", True), (True, "token", True), (True, "full", False)]):
        t, _, _ = _make(cuda, rows, hidden, torch.bfloat16, post, gate, residual, seed=90 + i)
        normed, stream = _call(t, 0.5, 1e-5)
        q, s4 = _call(t, 0.5, 1e-5, quantize=fmt)
        want = ops.fp4_quantize(normed, fmt)
        assert torch.equal(s4, stream) and q.shape == normed.shape
        assert torch.equal(q.codes, want.codes) and torch.equal(q.scales, want.scales)
        assert torch.equal(q.row_scale, want.row_scale)
    wide = torch.randn(9, 200, device=cuda).bfloat16()
    q, s = ops.block_norm(wide[:, 3:131], wide[:, 5:133], torch.ones(129, device=cuda).bfloat16()[1:], quantize=fmt)
    n, s2 = ops.block_norm(wide[:, 3:131], wide[:, 5:133], torch.ones(128, device=cuda).bfloat16())
    assert torch.equal(s, s2) and torch.equal(q.codes, ops.fp4_quantize(n, fmt).codes)


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_chain(cuda, fmt):
    """Block after block in 4 bits: norm, product, norm, product, as a decoder runs them, alone and as a CUDA graph."""
    t, _, _ = _make(cuda, 61, 1024, torch.bfloat16, True, "none", seed=100)
    g = torch.Generator(device=cuda).manual_seed(2)
    up = FP4Weight.from_weight((torch.randn(2048, 1024, device=cuda, generator=g) * 0.03).bfloat16(), fmt)
    down = FP4Weight.from_weight((torch.randn(1024, 1024, device=cuda, generator=g) * 0.03).bfloat16(), fmt)

    def step(x, fused):
        stream = t["residual"]
        for _ in range(3):
            if fused:
                n, stream = ops.block_norm(x, stream, t["weight"], post_weight=t["post_weight"], quantize=fmt)
            else:
                n, stream = ops.block_norm(x, stream, t["weight"], post_weight=t["post_weight"])
            x = ops.linear(ops.silu_mul(ops.linear(n, up)), down)
        return x, stream

    want = step(t["x"], False)
    got = step(t["x"], True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    static = t["x"].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static, True)
    graph.replay()
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    assert ops.require().status(0) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,hidden", [(9, 37), (1, 1), (7, 1), (700, 301), (3, 4095), (40, 6)])
def test_rows_that_share_words(cuda, dtype, rows, hidden):
    """16-bit rows of odd or short lengths: views with any offset and stride give the bits of tensors without gaps, and a
    row that is not finite leaves its neighbours, with which it shares words, as they are."""
    t, dn, up = _make(cuda, rows, hidden, dtype, True, "full", seed=90, grad=True)
    leaves = list(t.values())
    want = _call(t, 0.5, 1e-5)
    grads = torch.autograd.grad(want, leaves, (dn, up))
    for offset, stride in ((0, hidden + 1), (1, hidden + 2), (3, hidden + 3), (2, hidden + 4)):
        def view(x):
            flat = torch.full((rows * stride + 8,), float("nan"), device=cuda, dtype=dtype)
            wide = flat[offset:offset + rows * stride].view(rows, stride)
            wide[:, :hidden] = x.detach()
            return wide[:, :hidden]

        v = {k: view(x).requires_grad_() if x.dim() == 2 else x for k, x in t.items()}
        got = _call(v, 0.5, 1e-5)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        again = torch.autograd.grad(got, list(v.values()), (view(dn), view(up)))
        assert all(torch.equal(a, b) for a, b in zip(again, grads))
    if rows >= 3:
        with torch.no_grad():
            t["x"][rows // 2] = float("nan")
        got = _call(t, 0.5, 1e-5)
        again = torch.autograd.grad(got, leaves, (dn, up))
        others = torch.arange(rows, device=cuda) != rows // 2
        for a, b in zip((*got, again[0], again[1], again[4]), (*want, grads[0], grads[1], grads[4])):
            assert torch.equal(a[others], b[others])
        assert not got[0][rows // 2].isfinite().any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,hidden", [(16, 4096), (3, 1001), (700, 520), (5, 16384)])
def test_gradients_take_the_unrounded_stream(cuda, dtype, rows, hidden):
    """Without a norm behind the block and a gate too, nothing but the results is rounded to the operands' type: with one
    output at a time the bounds hold without the stream's rounding (``half`` of every term of dweight)."""
    half, tiny = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    for i, (residual, scale) in enumerate(((True, 1.0), (True, 0.22), (False, 1.0))):
        t, dn, _ = _make(cuda, rows, hidden, dtype, False, "none", residual, seed=110 + i, grad=True)
        normed, stream = _call(t, scale, 1e-5)
        leaves = [t["weight"], t["x"]] + ([t["residual"]] if residual else [])
        dw, dx, *dr = torch.autograd.grad(normed, leaves, dn)
        with torch.no_grad():
            x, w, g = t["x"].double(), t["weight"].double(), dn.double()
            s = scale * x + (t["residual"].double() if residual else 0.0)
            mag = abs(scale) * x.abs() + (t["residual"].double().abs() if residual else 0.0)
            inv = torch.rsqrt(s.square().mean(-1, keepdim=True) + 1e-5)
            sh, sh_err = s * inv, mag * inv * 2 * F32
            want = (g * sh).sum(0)
            err = (g.abs() * sh_err).sum(0) + (g * sh).abs().sum(0) * (rows * 2.0 ** -24 + F32)
            _within(dw, (want, want.abs() * half * 1.01 + err + tiny), "dweight")
            m = (g * w * sh).mean(-1, keepdim=True)
            m_err = (g * w * sh).abs().mean(-1, keepdim=True) * F32 + ((g * w).abs() * sh_err).mean(-1, keepdim=True)
            ds = inv * (g * w - sh * m)
            err = inv * ((g * w).abs() + (sh * m).abs()) * 2 * F32 + inv * (sh_err * m.abs() + (sh.abs() + sh_err) * m_err)
            for got, f in ((dx, scale), *((d, 1.0) for d in dr)):
                _within(got, (f * ds, abs(f) * (ds.abs() * half * 1.01 + err) + tiny), "dx or dresidual")


@pytest.mark.parametrize("form", ["three dimensions", "autocast", "view", "autocast weight"])
def test_capture_beside_a_living_graph_of_views_and_casts(cuda, form):
    """The operands of a captured call are refused like leaves where they are views or casts of leaves that a graph of the
    default stream holds, and taken once that graph is gone. (Only the forward pass is captured beside the graph.)"""
    dtype = torch.float32 if form.startswith("autocast") else torch.bfloat16
    leaf = torch.randn(2, 5, 64, device=cuda).to(dtype).requires_grad_(form != "autocast weight")
    weight = torch.ones(64, device=cuda, dtype=dtype, requires_grad=form == "autocast weight")

    def call():
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=form.startswith("autocast")):
            return ops.block_norm(leaf.view(10, 64) if form == "view" else leaf, None, weight)[0]

    living = call()
    (want,) = torch.autograd.grad(living.sum(), leaf if leaf.requires_grad else weight, retain_graph=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with pytest.raises(RuntimeError, match="still holds a leaf"), torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
        call()
    del living
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        (got,) = torch.autograd.grad(call().sum(), leaf if leaf.requires_grad else weight)
    graph.replay()
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,hidden", [(1, 5), (7, 1001), (1300, 333), (2500, 77), (600, 4095), (9, 200)])
def test_operands_that_are_not_there(cuda, dtype, rows, hidden):
    """A residual or an upstream gradient that is not given is one of zeros, bit for bit: rows copied ahead, those behind
    the last and odd ones that start in the middle of a word among them."""
    for post, gate in ((False, "none"), (True, "token"), (False, "full")):
        t, dn, up = _make(cuda, rows, hidden, dtype, post, gate, False, seed=120, grad=True)
        zeros = torch.zeros(rows, hidden, device=cuda, dtype=dtype)
        leaves = [v for v in t.values() if v is not None]
        without, given = _call(t, 0.5, 1e-5), _call({**t, "residual": zeros}, 0.5, 1e-5)
        assert all(torch.equal(a, b) for a, b in zip(without, given))
        for i, g in ((0, dn), (1, up)):
            alone = torch.autograd.grad(without[i], leaves, g, retain_graph=True)
            both = torch.autograd.grad(given, leaves, (g, zeros) if i == 0 else (zeros, g), retain_graph=True)
            assert all(torch.equal(a, b) for a, b in zip(alone, both))


def test_half_autocast(cuda):
    """Under fp16 autocast operands of several types, as a projection and an fp32 stream are, run in fp16 and get their
    gradients in their own types; operands of one type stay as they are, and 4-bit results are made from bf16 alone."""
    t, dn, up = _make(cuda, 8, 64, torch.float32, True, "token", seed=81, grad=True)
    x = t["x"].detach().half().requires_grad_()
    with torch.autocast("cuda", dtype=torch.float16):
        normed, stream = _call({**t, "x": x}, 1.0, 1e-5)
        plain = _call(t, 1.0, 1e-5)
        with pytest.raises(ValueError, match="bfloat16"):
            ops.block_norm(x, None, t["weight"], quantize="nvfp4")
    assert normed.dtype == stream.dtype == torch.float16 and plain[0].dtype == torch.float32
    half = {k: v.detach().half() for k, v in t.items()}
    assert all(torch.equal(a, b) for a, b in zip((normed, stream), _call(half, 1.0, 1e-5)))
    leaves = [x] + [t[k] for k in ("residual", "weight", "post_weight", "gate")]
    grads = torch.autograd.grad((normed, stream), leaves, (dn.half(), up.half()))
    assert [g.dtype for g in grads] == [torch.float16] + [torch.float32] * 4
