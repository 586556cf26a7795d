"""4-bit operands on the GPU: codes and scales against the rules in 64 bits, products against 64-bit products of the
values the codes stand for.

Tolerances. Quantisation: none, the values are equal (its borders are exact in fp32). Products: one rounding to bf16,
``2^-8`` of the value, and fp32 sums: the tensor cores may cut off ``2^-23`` of the running magnitude at every 16
products, so at most ``(K / 16 + 2) 2^-23`` of the sum of the products' magnitudes; the same again for sums in parts.
"""

import pytest
import torch

from economize_b200 import ops
from economize_b200.errors import ConfigError
from economize_b200.ops import fp4
from economize_b200.ops.fp4 import FP4Weight

pytestmark = pytest.mark.gpu

GROUP = {"nvfp4": 16, "mxfp4": 32}


def _values(x, fmt):
    """The nearest 4-bit values of ``x`` in 64 bits, by distance."""
    v = x.double().unflatten(-1, (-1, GROUP[fmt]))
    top = v.abs().amax(-1, keepdim=True)
    if fmt == "mxfp4":
        e = torch.floor(torch.log2(top.clamp_min(2.0 ** -124)))
        e += (top >= 1.75 * torch.exp2(e)).double()
        unit = torch.exp2((e - 2).clamp(-126, 125))
    else:
        row = torch.exp2(torch.ceil(torch.log2((top.amax(-2, keepdim=True) / 2688).clamp_min(2.0 ** -100))))
        row = torch.where(top.amax(-2, keepdim=True) > 0, row, 1.0)
        scale = (top / (6 * row)).clamp(2.0 ** -9, 448)
        step = torch.exp2(torch.floor(torch.log2(scale)).clamp_min(-6) - 3)
        unit = torch.round(scale / step) * step * row
    v = v / unit
    a = v.abs().clamp(max=6)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).double()
    return (torch.sign(v) * torch.round(a / step) * step * unit).flatten(-2)


def _normal(dev, *shape, seed=0, spread=0.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn(*shape, device=dev, generator=g)
    if spread:
        x = x * torch.exp(spread * torch.randn(*shape, device=dev, generator=g))
    return x.bfloat16()


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("rows,cols", [(1, 32), (1, 64), (2, 96), (3, 256), (5, 288), (127, 416), (128, 512), (129, 1056),
                                       (61, 4096), (700, 2080), (1000, 14336), (2, 33056), (1, 65536)])
def test_quantize(cuda, fmt, rows, cols):
    x = _normal(cuda, rows, cols, seed=rows + cols, spread=1.5)
    q = ops.fp4_quantize(x, fmt)
    assert torch.equal(q.dequantize().double(), _values(x, fmt))
    cpu = ops.fp4_quantize(x.cpu(), fmt)  # scales byte for byte, padding included
    assert torch.equal(q.scales.cpu(), cpu.scales) and torch.equal(q.row_scale.cpu(), cpu.row_scale)
    assert torch.equal(cpu.dequantize(), q.dequantize().cpu())


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_quantize_every_magnitude(cuda, fmt):
    """All finite bf16 values, each as its group's largest and below another's. (The oracle is rounded to bf16 as the
    result is: groups of the very largest have values beyond bf16's range, 6 x 5.85e37, which become infinite; all others
    have at most 6 significant bits and stay.)"""
    bits = torch.arange(0, 0x7F80, device=cuda, dtype=torch.int32)
    every = bits.to(torch.int16).view(torch.bfloat16)
    g = torch.Generator(device=cuda).manual_seed(0)
    pad = (-every.numel()) % 32
    every = torch.cat([every, every[:pad]])
    sign = torch.where(torch.rand(every.numel(), device=cuda, generator=g) < 0.5, -1, 1).bfloat16()
    for x in (every * sign, (every * sign)[torch.randperm(every.numel(), device=cuda, generator=g)]):
        rows = x.view(-1, 32)  # a row per 32: every scale of rows
        want = _values(rows, fmt)
        assert torch.equal(ops.fp4_quantize(rows, fmt).dequantize(), want.bfloat16())
        assert torch.equal(want.bfloat16().double()[want.abs() < 3.3e38], want[want.abs() < 3.3e38])
    # all bf16 significands against all e4m3 scales of a row: ties between codes
    s = torch.arange(128, 256, device=cuda).bfloat16()
    tops = torch.arange(96, 192, device=cuda).bfloat16()
    grid = torch.stack([s[None].expand(96, 128) * 2.0 ** k for k in range(-9, 1)], 1)  # [tops, k, 128]
    x = torch.zeros(96, 10, 128 // 8, 16, device=cuda, dtype=torch.bfloat16)
    x[..., :8] = grid.view(96, 10, 16, 8)
    x[..., 8] = 2 * tops[:, None, None]
    x = x.view(96, -1)
    x[:, -1] = 448.0
    assert torch.equal(ops.fp4_quantize(x, fmt).dequantize().double(), _values(x, fmt))


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_quantize_zeros_and_not_finite(cuda, fmt):
    x = _normal(cuda, 4, 128, seed=1)
    x[0] = 0.0
    x[1, 5] = float("nan")
    x[2, 40] = float("inf")
    x[3, 100] = -float("inf")
    q = ops.fp4_quantize(x, fmt)
    d = q.dequantize()
    assert torch.equal(d[0], torch.zeros_like(d[0]))
    bad = ~x.isfinite()
    group = bad.view(4, -1, GROUP[fmt]).any(-1, keepdim=True).expand(-1, -1, GROUP[fmt]).reshape(4, -1)
    assert d[group].isnan().all()
    clean = torch.where(bad, 0.0, x)
    assert torch.equal(d[~group].double(), _values(clean, fmt)[~group])
    assert torch.equal(q.scales.cpu(), ops.fp4_quantize(x.cpu(), fmt).scales)
    # products: the rows that read them are NaN, the others are what they are without them
    w = FP4Weight.from_weight(_normal(cuda, 40, 128, seed=2), fmt)
    y = ops.linear(x, w)
    assert y[1:].isnan().all() and torch.equal(y[:1], torch.zeros_like(y[:1]))
    x[1:3] = 1.0
    assert torch.equal(ops.linear(x, w)[:3], ops.linear(x[:3], w))


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_quantize_strided_and_empty(cuda, fmt):
    wide = _normal(cuda, 37, 1000, seed=3)
    for x in (wide[:, 8:8 + 96], wide[:, 3:3 + 96], wide[::2, :128], wide.t()[:960].t()[:, :64], wide[:1, 1:33]):
        assert torch.equal(ops.fp4_quantize(x, fmt).dequantize(), ops.fp4_quantize(x.contiguous(), fmt).dequantize())
    x = wide[:36, :192].reshape(2, 3, 6, 192)
    q = ops.fp4_quantize(x, fmt)
    assert q.shape == x.shape and q.dequantize().shape == x.shape
    empty = ops.fp4_quantize(wide[:0, :64], fmt)
    assert empty.dequantize().shape == (0, 64)
    w = FP4Weight.from_weight(wide[:, :64], fmt)
    assert ops.linear(wide[:0, :64], w).shape == (0, 37) and ops.linear(empty, w).shape == (0, 37)


def _check_product(x, w, fmt, y=None):
    weight = FP4Weight.from_weight(w, fmt)
    y = ops.linear(x, weight) if y is None else y
    xd, wd = _values(x.reshape(-1, x.shape[-1]), fmt), _values(w, fmt)
    want, mag = xd @ wd.t(), xd.abs() @ wd.abs().t()
    bound = want.abs() * 2.0 ** -8 + mag * (2 * (x.shape[-1] / 16 + 2) * 2.0 ** -23)
    off = (y.reshape(want.shape).double() - want).abs()
    assert (off <= bound).all(), f"{(off / (bound + 1e-300)).max().item():.2f} times the bound"
    return weight, y


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("rows,cols,out", [(1, 32, 1), (1, 256, 128), (3, 64, 130), (16, 512, 4096), (17, 288, 100),
                                           (32, 1024, 1000), (61, 4096, 6144), (64, 2080, 257), (100, 1312, 384),
                                           (128, 256, 256), (129, 544, 129), (256, 4096, 512), (300, 1056, 1000),
                                           (1003, 1056, 1000), (640, 14336, 256)])
def test_product(cuda, fmt, rows, cols, out):
    x = _normal(cuda, rows, cols, seed=rows, spread=0.7)
    w = _normal(cuda, out, cols, seed=out, spread=0.3) * 0.05
    _check_product(x, w, fmt)


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("path", [1, 2])
@pytest.mark.parametrize("rows,cols,out", [(1, 32, 1), (130, 288, 385), (257, 1056, 768), (300, 4096, 1000), (2100, 544, 3200),
                                           (1003, 2080, 6001)])
def test_product_paths(cuda, fmt, path, rows, cols, out):
    """Every kernel at sizes that it would not be chosen for, several tiles to a CTA pair among them."""
    x = _normal(cuda, rows, cols, seed=rows, spread=0.7)
    w = _normal(cuda, out, cols, seed=out, spread=0.3) * 0.05
    a, b = ops.fp4_quantize(x, fmt), FP4Weight.from_weight(w, fmt)
    y = ops.require().fp4_matmul(a.data, rows, cols, b.codes, b.scales, b.row_scale, fp4.FORMATS[fmt], path)
    _check_product(x, w, fmt, y)


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_product_exact(cuda, fmt):
    """One product in a sum, rounded once: every element, group and row scale in its place."""
    g = torch.Generator(device=cuda).manual_seed(5)
    for rows, cols, out in ((61, 768, 200), (200, 1280, 384), (513, 512, 300)):
        x = torch.zeros(rows, cols, device=cuda)
        at = torch.randint(0, cols, (rows,), device=cuda, generator=g)
        x[torch.arange(rows, device=cuda), at] = torch.exp2(torch.randint(-3, 9, (rows,), device=cuda, generator=g).float())
        w = torch.randint(-6, 7, (out, cols), device=cuda, generator=g).float()
        w = torch.where(w.abs() == 5, 4.0, w)
        w = w.view(out, -1, 16)
        w[..., 0] = 6.0
        w = w * torch.exp2(torch.randint(-2, 3, (out, w.shape[1], 1), device=cuda, generator=g).float())
        if fmt == "mxfp4":  # one scale per 32
            w = w.view(out, -1, 2, 16) / w.view(out, -1, 2, 16).abs().amax((2, 3), keepdim=True) * 6
            w = fp4.quantize(w.reshape(out, cols).bfloat16(), fmt).dequantize().float()
        w = w.reshape(out, cols).bfloat16()
        y = ops.linear(x.bfloat16(), FP4Weight.from_weight(w, fmt))
        want = _values(x.bfloat16(), fmt) @ _values(w, fmt).t()  # one product each
        assert torch.equal(y.double(), want.bfloat16().double())


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_rows_do_not_depend_on_their_number(cuda, fmt):
    x = _normal(cuda, 128, 4096, seed=6)
    w = FP4Weight.from_weight(_normal(cuda, 1024, 4096, seed=7), fmt)
    every = ops.linear(x, w)
    for n in (1, 2, 16, 17, 33, 61, 64, 65, 127):
        assert torch.equal(ops.linear(x[:n], w), every[:n])
        assert torch.equal(ops.linear(x[128 - n:], w), every[128 - n:])


def test_leading_dimensions_and_types(cuda):
    x = _normal(cuda, 2, 3, 128, seed=8)
    w = FP4Weight.from_weight(_normal(cuda, 64, 128, seed=9))
    y = ops.linear(x, w)
    assert y.shape == (2, 3, 64) and y.dtype == torch.bfloat16
    assert torch.equal(y, ops.linear(ops.fp4_quantize(x), w))
    assert ops.linear(x.float(), w).dtype == torch.float32 and torch.equal(ops.linear(x.float(), w).bfloat16(), y)
    bias = _normal(cuda, 64, seed=10)
    assert torch.equal(ops.linear(x, w, bias), y + bias)
    assert torch.equal(ops.linear(x[0, 0], w), y[0, 0])


def test_weight_state(cuda):
    w = _normal(cuda, 200, 416, seed=11)
    for fmt in ("nvfp4", "mxfp4"):
        a = FP4Weight.from_weight(w, fmt)
        b = FP4Weight.from_weight(w.cpu(), fmt)  # values, not codes: the sign of a zero code may differ
        assert torch.equal(a.dequantize().cpu(), b.dequantize())
        b = b.to(cuda)
        x = _normal(cuda, 5, 416, seed=12)
        assert torch.equal(ops.linear(x, a), ops.linear(x, b))
        assert a.nbytes() == a.codes.numel() + a.scales.numel() + 4 * a.row_scale.numel()


def test_refusals(cuda):
    x = _normal(cuda, 4, 64)
    w = FP4Weight.from_weight(_normal(cuda, 8, 64))
    with pytest.raises(ConfigError):
        ops.fp4_quantize(x, "int4")
    with pytest.raises(ConfigError):
        ops.fp4_quantize(x[:, :48])
    with pytest.raises(RuntimeError, match="bfloat16"):
        ops.fp4_quantize(x.float())
    with pytest.raises(ConfigError):
        ops.linear(_normal(cuda, 4, 96), w)
    with pytest.raises(ConfigError):
        ops.linear(ops.fp4_quantize(x, "mxfp4"), w)
    with pytest.raises(ConfigError):
        ops.linear(x.cpu(), w)
    C, q = ops.require(), ops.fp4_quantize(x)
    good = (q.data, 4, 64, w.codes, w.scales, w.row_scale, 1)
    for i, bad in ((0, q.data[:-16]), (0, q.data.cpu()), (0, q.data.float()), (1, 5), (1, -1), (2, 96), (2, 40),
                   (3, w.codes.cpu()), (3, w.codes[:, :16]), (4, w.scales.float()), (4, w.scales[:, :2]),
                   (5, w.row_scale.double()), (5, w.row_scale[:2]), (5, w.row_scale.cpu()), (6, 3), (6, 2)):
        args = list(good)
        args[i] = bad
        with pytest.raises((RuntimeError, ValueError)):
            C.fp4_matmul(*args)


def test_streams_and_graphs(cuda):
    x = _normal(cuda, 61, 1024, seed=13)
    w = FP4Weight.from_weight(_normal(cuda, 768, 1024, seed=14))
    want = ops.linear(x, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = ops.linear(x, w)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, want)
    static = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.linear(static, w)
    for seed in (15, 16):
        fresh = _normal(cuda, 61, 1024, seed=seed)
        static.copy_(fresh)
        graph.replay()
        assert torch.equal(out, ops.linear(fresh, w))
    assert ops.require().status(0) == 0


def test_weight_made_and_used_at_once(cuda):
    """A weight is read by the product right behind the kernels that made it."""
    x = _normal(cuda, 1, 4096, seed=17)
    base = _normal(cuda, 4096, 4096, seed=18)
    want = None
    for i in range(20):
        w = FP4Weight.from_weight(base)
        y = ops.linear(x, w)
        want = y if want is None else want
        assert torch.equal(y, want)
        del w
        torch.empty(4096 * 2048, device=cuda, dtype=torch.uint8).fill_(0xFF)  # where the codes were


def test_long_offsets(cuda):
    """Codes and outputs beyond 2^31 bytes."""
    rows, cols = 70000, 65536
    x = torch.zeros(rows, cols, device=cuda, dtype=torch.bfloat16)
    x[-3:] = _normal(cuda, 3, cols, seed=19)
    q = ops.fp4_quantize(x)
    tail = ops.fp4_quantize(x[-3:])
    assert torch.equal(q.codes[-3:], tail.codes)
    w = _normal(cuda, 48, cols, seed=20)
    _check_product(x[-3:], w, "nvfp4", ops.linear(q, FP4Weight.from_weight(w))[-3:])
    d = q.dequantize()
    assert torch.equal(d[-3:], tail.dequantize()) and not d[:-3].any()


@pytest.mark.parametrize("path", [1, 2])
@pytest.mark.parametrize("rows,out", [(3, 8), (129, 257), (300, 64)])
def test_rows_of_any_magnitude(cuda, path, rows, out):
    """Rows and weights near either end of what nvfp4's powers of two reach, against rows of the other end and their own,
    on both kernels: results inside bf16's range are right although one row's power alone, or both together, would leave
    it, those beyond it are infinite, and sums of zero are zero. Every sum is exact in fp32 (64 equal terms of 12 bits, all
    of one sign or half of them of the other), so the result is rounded once, from what fp32 holds: below bf16's normal
    range that is off by half its smallest spacing and half of fp32's."""
    cols = 64
    e = torch.tensor([-110, -97, -89, -52, -20, 0, 33, 60, 75, 90, 101, 115, 120], device=cuda)
    ex, ew = e[torch.arange(rows, device=cuda) * 6 % 13], e[torch.arange(out, device=cuda) * 5 % 13]
    for signs in (1, 2):
        x = torch.exp2(ex.double())[:, None].expand(rows, cols).clone()
        x[:, ::2] *= -1 if signs == 2 else 1
        w = torch.exp2(ew.double())[:, None].expand(out, cols)
        a, b = ops.fp4_quantize(x.bfloat16(), "nvfp4"), FP4Weight.from_weight(w.bfloat16())
        y = ops.require().fp4_matmul(a.data, rows, cols, b.codes, b.scales, b.row_scale, 1, path)
        want = _values(x, "nvfp4") @ _values(w, "nvfp4").t()
        normal = want.abs() >= torch.finfo(torch.bfloat16).smallest_normal
        assert torch.equal(y[normal].double(), want.float().bfloat16().double()[normal])
        off = (y.double() - want).abs()
        assert (off[~normal] <= 2.0 ** -134 + 2.0 ** -150).all()
        assert not y.isnan().any() and (signs == 2 or y.isinf().any() and (y == 0).any())
        assert signs == 1 or not y.any()


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("rows", [1, 61, 200])
def test_weight_written_between_products(cuda, fmt, rows):
    """A weight written in place directly in front of a product, and one kernel before it, is what the product reads, in a
    captured sequence too: nothing of it is taken from what was there before."""
    x = _normal(cuda, rows, 2048, seed=21)
    q = ops.fp4_quantize(x, fmt)
    sources = [FP4Weight.from_weight(_normal(cuda, 1536, 2048, seed=s), fmt) for s in (22, 23, 24)]
    want = [ops.linear(q, s) for s in sources]
    w = FP4Weight.from_weight(_normal(cuda, 1536, 2048, seed=25), fmt)

    def sequence():
        out = []
        for s in sources:
            w.row_scale.copy_(s.row_scale)
            w.scales.copy_(s.scales)
            w.codes.copy_(s.codes)
            out.append(ops.linear(q, w))  # codes directly in front of the product
        for s in sources:
            w.row_scale.copy_(s.row_scale)
            w.codes.copy_(s.codes)
            w.scales.copy_(s.scales)
            out.append(ops.linear(x, w))  # scales in front of the quantisation in front of the product
        return out

    for _ in range(10):
        assert all(torch.equal(a, b) for a, b in zip(sequence(), want + want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sequence()
    for _ in range(10):
        for o in out:
            o.zero_()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, want + want))
    assert ops.require().status(0) == 0
