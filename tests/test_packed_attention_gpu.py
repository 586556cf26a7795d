"""Packed causal attention and its gradients against the formulas in 64 bits, element by element.

Tolerances (bf16 inputs are exact in 64 bits, so only the kernels round; u = 2^-8 is bf16's half spacing):

* a score is an fp32 accumulation of D products: at most ``D 2^-23`` of the sum of their magnitudes (``eps`` below,
  times the scale); a probability is off by 2 eps of itself (score and log-sum-exp) and the exponential's ``2^-20``;
* P and dS are rounded to bf16 once as operands (u relative), products accumulate in fp32 (``2^-14`` of the sum of
  magnitudes covers thousands of terms), every output is rounded once more (u);
* delta is allowed the rounded output's error times the gradient's magnitude.
"""

import math

import pytest
import torch

from economize_b200 import ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -8


def _inputs(dev, lens, heads, kv_heads, dim, pad=0, seed=0, spread=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    t = sum(lens) + pad

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, device=dev, generator=g) * std).bfloat16()

    q, k, v = normal(t, heads, dim, std=spread), normal(t, kv_heads, dim), normal(t, kv_heads, dim)
    cu = torch.tensor([0, *lens], device=dev).cumsum(0).int()
    return q, k, v, cu, normal(t, heads, dim)


def _oracle(q, k, v, lens, dout, scale):
    """Outputs and gradients in 64 bits with the bound of each one's error."""
    t, heads, dim = q.shape
    group = heads // k.shape[1]
    z = {n: torch.zeros(x.shape, dtype=torch.float64, device=q.device)
         for n, x in (("out", q), ("dq", q), ("dk", k), ("dv", v), ("out_err", q), ("dq_err", q), ("dk_err", k),
                      ("dv_err", v))}
    a = 0
    for n in lens:
        for h in range(heads if n else 0):
            s, j = slice(a, a + n), h // group
            qs, ks, vs, do = q[s, h].double(), k[s, j].double(), v[s, j].double(), dout[s, h].double()
            hide = torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1)
            sc = (qs @ ks.t() * scale).masked_fill(hide, -math.inf)
            eps = (qs.abs() @ ks.abs().t() * scale).masked_fill(hide, 0).amax(-1, keepdim=True) * dim * 2.0 ** -23
            rel = 2.5 * eps + 2.0 ** -19  # of a probability
            p = torch.softmax(sc, -1)
            o = p @ vs
            o_err = (p * (U + rel + 2.0 ** -14)) @ vs.abs() + U * o.abs()
            dp = do @ vs.t()
            delta = (do * o).sum(-1, keepdim=True)
            ds = p * (dp - delta) * scale
            dp_err = do.abs() @ vs.abs().t() * dim * 2.0 ** -23
            delta_err = (do.abs() * o_err).sum(-1, keepdim=True) + (do * o).abs().sum(-1, keepdim=True) * 2.0 ** -16
            ds_err = ds.abs() * (U + rel + 2.0 ** -14) + p * (dp_err + delta_err) * scale * (1 + U)
            z["out"][s, h], z["out_err"][s, h] = o, o_err
            z["dq"][s, h] = ds @ ks
            z["dq_err"][s, h] = ds_err @ ks.abs() + U * z["dq"][s, h].abs()
            z["dk"][s, j] += ds.t() @ qs
            z["dk_err"][s, j] += ds_err.t() @ qs.abs()
            z["dv"][s, j] += p.t() @ do
            z["dv_err"][s, j] += (p * (U + rel + 2.0 ** -14)).t() @ do.abs()
        a += n
    for n in ("dk", "dv"):
        z[n + "_err"] += U * z[n].abs()
    return z


def _within(got, z, name):
    off, err = (got.double() - z[name]).abs(), z[name + "_err"] + 1e-30
    assert (off <= err).all(), f"{name}: {(off / err).max().item():.2f} times the bound"


def _run(q, k, v, cu, dout, scale=None, tiles=0):
    q, k, v = (x.detach().requires_grad_() for x in (q, k, v))
    out = ops.packed_attention(q, k, v, cu, scale) if tiles == 0 else \
        ops.require().packed_attention(q, k, v, cu, scale or q.shape[-1] ** -0.5, tiles)
    return (out.detach(), *torch.autograd.grad(out, (q, k, v), dout))


LENS = [[1], [2], [127], [128], [129], [1, 1, 1], [16, 0, 15, 17], [300, 5, 0, 0, 64], [256, 256], [700], [1, 900, 33]]


@pytest.mark.parametrize("lens", LENS, ids=str)
@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 1, 128), (3, 3, 64), (4, 2, 128), (3, 1, 128), (8, 1, 64)])
def test_outputs_and_gradients(cuda, lens, heads, kv_heads, dim):
    q, k, v, cu, dout = _inputs(cuda, lens, heads, kv_heads, dim)
    z = _oracle(q, k, v, lens, dout, dim ** -0.5)
    got = _run(q, k, v, cu, dout)
    for name, x in zip(("out", "dq", "dk", "dv"), got):
        _within(x, z, name)
    assert torch.equal(ops.packed_attention(q, k, v, cu), got[0])  # without gradients
    assert ops.require().status(0) == 0


@pytest.mark.parametrize("tiles", [1, 2])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 128), (3, 3, 64), (6, 2, 96)])
def test_both_forms_of_the_forward_pass(cuda, tiles, heads, kv_heads, dim):
    """A CTA works on one query tile or on two, chosen by the mean length; every shape goes through either."""
    for lens, pad in (([700], 0), ([5, 300, 129, 0, 64, 1], 20), ([256] * 3, 0), ([1] * 200, 3)):
        q, k, v, cu, dout = _inputs(cuda, lens, heads, kv_heads, dim, pad=pad, seed=20)
        z = _oracle(q, k, v, lens, dout, dim ** -0.5)
        for name, got in zip(("out", "dq", "dk", "dv"), _run(q, k, v, cu, dout, tiles=tiles)):
            _within(got, z, name)
    assert ops.require().status(0) == 0


@pytest.mark.parametrize("lens,heads,kv_heads,dim", [
    ([700], 8, 1, 128),               # two CTAs share a key tile's queries
    ([2049], 8, 1, 64),               # eight
    ([5, 1300, 1, 0, 1294], 16, 1, 64),  # four, of which some get none of a short sequence's
    ([1000, 700], 12, 2, 96),         # two, six heads in packs of two
    ([1600], 32, 4, 80),              # six
])
def test_gradients_of_few_key_tiles(cuda, lens, heads, kv_heads, dim):
    """A key tile's queries are shared by several CTAs where there are few key tiles; their sums are joined in order."""
    q, k, v, cu, dout = _inputs(cuda, lens, heads, kv_heads, dim, pad=9, seed=21)
    z = _oracle(q, k, v, lens, dout, dim ** -0.5)
    first = _run(q, k, v, cu, dout)
    for name, got in zip(("out", "dq", "dk", "dv"), first):
        _within(got, z, name)
        assert got[-9:].count_nonzero() == 0
    for _ in range(20):
        for got, want in zip(_run(q, k, v, cu, dout), first):
            assert torch.equal(got, want)
    assert ops.require().status(0) == 0


def test_more_tiles_than_ctas(cuda):
    """CTAs take their tiles as they come free; which one takes a tile leaves the results alone."""
    g = torch.Generator().manual_seed(3)
    lens = torch.randint(0, 260, (150,), generator=g).tolist()
    q, k, v, cu, dout = _inputs(cuda, lens, 6, 3, 64, pad=5, seed=22)
    z = _oracle(q, k, v, lens, dout, 64 ** -0.5)
    first = _run(q, k, v, cu, dout)
    for name, got in zip(("out", "dq", "dk", "dv"), first):
        _within(got, z, name)
    for _ in range(20):
        for got, want in zip(_run(q, k, v, cu, dout), first):
            assert torch.equal(got, want)
    assert ops.require().status(0) == 0


@pytest.mark.parametrize("dim", [8, 16, 24, 32, 40, 56, 64, 72, 80, 96, 104, 120, 128])
def test_head_dimensions(cuda, dim):
    lens = [140, 3, 77]
    q, k, v, cu, dout = _inputs(cuda, lens, 4, 2, dim, seed=1)
    z = _oracle(q, k, v, lens, dout, dim ** -0.5)
    for name, got in zip(("out", "dq", "dk", "dv"), _run(q, k, v, cu, dout)):
        _within(got, z, name)


@pytest.mark.parametrize("spread,scale", [(1.0, 0.02), (8.0, None), (30.0, 0.3)])
def test_flat_and_peaked_scores(cuda, spread, scale):
    """Rows whose maximum rises by far more than the lazy rescaling allows, and rows that weigh all keys alike."""
    lens = [513, 200]
    q, k, v, cu, dout = _inputs(cuda, lens, 4, 2, 64, seed=2, spread=spread)
    ramp = torch.linspace(0.1, 2.0, 713, device=cuda)[:, None, None]
    k = (k * ramp).bfloat16()
    z = _oracle(q, k, v, lens, dout, scale or 0.125)
    for name, got in zip(("out", "dq", "dk", "dv"), _run(q, k, v, cu, dout, scale)):
        _within(got, z, name)


@pytest.mark.parametrize("lens,pad", [([200, 30], 70), ([128], 1), ([5, 0, 250], 300)])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 128), (3, 3, 64)])
def test_padding_and_other_sequences_hold_anything(cuda, lens, pad, heads, kv_heads, dim):
    """NaN in the row's padding reaches nothing (its own results are zero), NaN in one sequence no other."""
    q, k, v, cu, dout = _inputs(cuda, lens, heads, kv_heads, dim, pad=pad, seed=3)
    n = sum(lens)
    clean = _run(q, k, v, cu, dout)
    for x in (q, k, v, dout):
        x[n:] = float("nan")
    dirty = _run(q, k, v, cu, dout)
    for a, b in zip(clean, dirty):
        assert torch.equal(a, b)
        assert (b[n:] == 0).all() and torch.isfinite(b).all()
    if len(lens) > 1:
        last = slice(n - lens[-1], n)
        for x in (q, k, v, dout):
            x[last] = float("inf")
        for a, b in zip(clean, _run(q, k, v, cu, dout)):
            assert torch.equal(a[: last.start], b[: last.start])


def test_leading_rows_outside_the_sequences(cuda):
    lens = [40, 150]
    q, k, v, cu, dout = _inputs(cuda, [25, *lens, 10], 2, 1, 64, seed=4)
    want = _run(*(x[25:215] for x in (q, k, v)), torch.tensor([0, 40, 190], device=cuda).int(), dout[25:215])
    got = _run(q, k, v, cu[1:4].contiguous(), dout)
    for a, b in zip(want, got):
        assert torch.equal(a, b[25:215])
        assert (b[:25] == 0).all() and (b[215:] == 0).all()


def test_no_sequences_and_no_tokens(cuda):
    q, k, v, _, dout = _inputs(cuda, [20], 4, 2, 64)
    for cu in ([0], [0, 0], [20, 20, 20]):
        for x in _run(q, k, v, torch.tensor(cu, device=cuda).int(), dout):
            assert (x == 0).all()
    empty = _run(q[:0], k[:0], v[:0], torch.tensor([0, 0], device=cuda).int(), dout[:0])
    assert [x.shape[0] for x in empty] == [0, 0, 0, 0]


def test_many_sequences(cuda):
    """More sequences than the plan kernel has threads."""
    lens = [(i * 7) % 5 for i in range(2500)]
    q, k, v, cu, dout = _inputs(cuda, lens, 2, 1, 16, seed=5)
    z = _oracle(q[:, :1], k, v, lens[:400], dout[:, :1], 0.25)  # the oracle of the first sequences' first head
    got = _run(q[:, :1], k, v, cu, dout[:, :1])
    n = sum(lens[:400])
    for name, x in zip(("out", "dq", "dk", "dv"), got):
        z[name], z[name + "_err"] = z[name][:n], z[name + "_err"][:n]
        _within(x[:n], z, name)
    assert ops.require().status(0) == 0


def test_strided_views(cuda):
    """Parts of a fused projection, heads-major storage, unaligned views and a broadcast gradient."""
    lens, h, g, d = [150, 61], 4, 2, 64
    q, k, v, cu, dout = _inputs(cuda, lens, h, g, d, seed=6)
    want = _run(q, k, v, cu, dout)
    fused = torch.cat([q.flatten(1), k.flatten(1), v.flatten(1)], 1)
    parts = [x.view(211, -1, d) for x in fused.split([h * d, g * d, g * d], 1)]
    major = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
    wide = torch.empty(211, h, d + 3, device=cuda, dtype=torch.bfloat16)
    wide[..., 3:] = q
    for args in (parts, major, [wide[..., 3:], k, v]):
        for a, b in zip(want, _run(*args, cu, dout)):
            assert torch.equal(a, b)
    ones = torch.ones((), device=cuda, dtype=torch.bfloat16).expand(211, h, d)
    for a, b in zip(_run(q, k, v, cu, ones.contiguous()), _run(q, k, v, cu, ones)):
        assert torch.equal(a, b)


def test_broadcast_keys(cuda):
    """One K/V head expanded over two: the gradient of the shared head is the sum of both."""
    lens = [130, 20]
    q, k, v, cu, dout = _inputs(cuda, lens, 4, 1, 64, seed=7)
    k1, v1 = k.clone().requires_grad_(), v.clone().requires_grad_()
    out = ops.packed_attention(q, k1.expand(-1, 2, -1), v1.expand(-1, 2, -1), cu)
    dk, dv = torch.autograd.grad(out, (k1, v1), dout)
    z = _oracle(q, k, v, lens, dout, 0.125)
    z["dk_err"] += 2 * U * (z["dk"].abs() + z["dk_err"])  # two rounded halves and their sum
    z["dv_err"] += 2 * U * (z["dv"].abs() + z["dv_err"])
    parts = [torch.autograd.grad(ops.packed_attention(q[:, s], k1, v1, cu), (k1, v1), dout[:, s])
             for s in (slice(0, 2), slice(2, 4))]
    for got, name, i in ((dk, "dk", 0), (dv, "dv", 1)):
        z[name + "_err"] += U * (parts[0][i].double().abs() + parts[1][i].double().abs())
        _within(got, z, name)


def test_only_what_is_asked_for(cuda):
    lens = [90, 140]
    q, k, v, cu, dout = _inputs(cuda, lens, 4, 2, 64, seed=8)
    want = _run(q, k, v, cu, dout)
    for i in range(3):
        args = [x.detach().clone() for x in (q, k, v)]
        args[i].requires_grad_()
        out = ops.packed_attention(*args, cu)
        (g,) = torch.autograd.grad(out, (args[i],), dout)
        assert torch.equal(out.detach(), want[0]) and torch.equal(g, want[i + 1])


def test_same_bits_every_time(cuda):
    q, k, v, cu, dout = _inputs(cuda, [600, 41, 333], 8, 2, 128, seed=9)
    first = _run(q, k, v, cu, dout)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, _run(q, k, v, cu, dout)))


@pytest.mark.parametrize("lens", [[2] * 40, [1, 2, 3, 4] * 10, [1] * 30 + [2], [3] * 50], ids=lambda x: f"{len(x)} of {x[0]}-{x[-1]}")
def test_gradients_of_sequences_of_a_few_tokens(cuda, lens):
    """dp - delta cancels there: delta needs more of the output than its bf16 rounding keeps. The whole gradient is as
    near its 64-bit value as two roundings to bf16 leave it (u / sqrt(3) each, operand and result, a fifth added)."""
    q, k, v, cu, dout = _inputs(cuda, lens, 8, 2, 64, seed=21)
    z = _oracle(q, k, v, lens, dout, 0.125)
    for name, got in zip(("dq", "dk", "dv"), _run(q, k, v, cu, dout)[1:]):
        assert (got.double() - z[name]).norm() <= 1.2 * U * math.sqrt(2 / 3) * z[name].norm(), name


def test_gradients_by_differences(cuda):
    """The slope of the 64-bit formula along random directions, against the kernels' gradients."""
    lens, dim, h = [70, 131], 64, 1e-4
    q, k, v, cu, dout = _inputs(cuda, lens, 4, 2, dim, seed=10)
    z = _oracle(q, k, v, lens, dout, dim ** -0.5)
    grads = _run(q, k, v, cu, dout)[1:]
    g = torch.Generator(device=cuda).manual_seed(0)
    for i, name in enumerate(("dq", "dk", "dv")):
        args = [x.double() for x in (q, k, v)]
        step = torch.randn(args[i].shape, device=cuda, generator=g, dtype=torch.float64)
        ends = []
        for sign in (1, -1):
            moved = [x + sign * h * step if j == i else x for j, x in enumerate(args)]
            ends.append((ops.reference.packed_attention(*moved, cu, dim ** -0.5) * dout.double()).sum())
        slope = (ends[0] - ends[1]) / (2 * h)
        got = (grads[i].double() * step).sum()
        assert abs(got - slope) <= (z[name + "_err"] * step.abs()).sum() + 1e-5 * abs(slope)


def test_twice_through_one_graph_and_as_a_cuda_graph(cuda):
    """The counters from which CTAs take their tiles start anew with every pass and every replay."""
    lens = [400, 3, 0, 129, 77] * 8
    q, k, v, cu, dout = _inputs(cuda, lens, 8, 2, 64, pad=4, seed=30)
    want = _run(q, k, v, cu, dout)
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    out = ops.packed_attention(*leaves, cu)
    for _ in range(2):
        for got, ref in zip(torch.autograd.grad(out, leaves, dout, retain_graph=True), want[1:]):
            assert torch.equal(got, ref)
    for got, ref in zip(torch.autograd.grad(out, leaves[1:], dout), want[2:]):  # dQ not asked for
        assert torch.equal(got, ref)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _run(q, k, v, cu, dout)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results = _run(q, k, v, cu, dout)
    for _ in range(3):
        for x in results:
            x.zero_()
        graph.replay()
        for got, ref in zip(results, want):
            assert torch.equal(got, ref)
    assert ops.require().status(0) == 0


def test_another_stream(cuda):
    q, k, v, cu, dout = _inputs(cuda, [300, 77], 4, 2, 128, seed=11)
    want = _run(q, k, v, cu, dout)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(q, k, v, cu, dout)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_autocast(cuda):
    q, k, v, cu, dout = _inputs(cuda, [50], 2, 1, 64, seed=12)
    wide = [x.float().requires_grad_() for x in (q, k, v)]
    with torch.autocast("cuda", dtype=torch.bfloat16):
        out = ops.packed_attention(*wide, cu)
    grads = torch.autograd.grad(out, wide, dout)
    want = _run(q, k, v, cu, dout)
    assert torch.equal(out.detach(), want[0])
    for a, b in zip(grads, want[1:]):
        assert a.dtype == torch.float32 and torch.equal(a, b.float())


@pytest.mark.parametrize("offsets", [[0, 40, 30, 60], [0, 30, 90], [-5, 20, 60], [0, 200, 300]])
def test_bad_offsets_are_clamped_and_reported(cuda, offsets):
    q, k, v, _, dout = _inputs(cuda, [60], 2, 1, 64, seed=13)
    ops.require().status(0)
    bad = _run(q, k, v, torch.tensor(offsets, device=cuda).int(), dout)
    assert ops.require().status(0) & 32
    fixed = torch.tensor(offsets).clamp(0, 60).cummax(0).values.int().to(cuda)
    for a, b in zip(bad, _run(q, k, v, fixed, dout)):
        assert torch.equal(a, b)
    assert ops.require().status(0) == 0


def test_refusals(cuda):
    q, k, v, cu, _ = _inputs(cuda, [30], 4, 2, 64)
    call = ops.packed_attention
    with pytest.raises(RuntimeError, match="bfloat16"):
        call(q.float(), k, v, cu)
    with pytest.raises(RuntimeError, match="int32"):
        call(q, k, v, cu.long())
    with pytest.raises(RuntimeError, match="device"):
        call(q, k, v, cu.cpu())
    with pytest.raises(RuntimeError, match="do not match"):
        call(q, k[:20], v[:20], cu)
    with pytest.raises(RuntimeError, match="do not match"):
        call(q, k, v[..., :32], cu)
    with pytest.raises(RuntimeError, match="query heads"):
        call(q[:, :3], k, v, cu)
    with pytest.raises(RuntimeError, match="head dimensions"):
        call(*(x[..., :60].contiguous() for x in (q, k, v)), cu)
    with pytest.raises(RuntimeError, match="head dimensions"):
        call(*(torch.cat([x, x, x], -1) for x in (q, k, v)), cu)
    with pytest.raises(RuntimeError, match="scale"):
        call(q, k, v, cu, -1.0)
    with pytest.raises(RuntimeError, match="expects"):
        call(q[None], k[None], v[None], cu)


def _held(dev, make):
    """What ``make`` returns and the bytes that stay allocated for it."""
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated(dev)
    result = make()
    return result, torch.cuda.memory_allocated(dev) - before


def test_the_backward_pass_releases_what_the_forward_pass_kept(cuda):
    """The output's rest and the log-sum-exps go with the graph's buffers, not with the output's last reference."""
    q, k, v, cu, dout = _inputs(cuda, [512] * 8, 32, 4, 64, seed=40)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    size = q.numel() * 2

    def step():
        out = ops.packed_attention(*leaves, cu)
        torch.autograd.grad(out, leaves, dout)
        return out

    step()
    out, held = _held(cuda, step)
    assert held < 1.25 * size and out.grad_fn is not None
    with pytest.raises(RuntimeError, match="a second time"):
        torch.autograd.grad(out, leaves, dout)


def test_saved_tensor_hooks_and_checkpointing(cuda):
    """Hooks see every large tensor that the backward pass reads; offloaded or recomputed, the gradients are the same."""
    from torch.utils.checkpoint import checkpoint

    q, k, v, cu, dout = _inputs(cuda, [512] * 8, 32, 4, 64, seed=41)
    want = _run(q, k, v, cu, dout)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    size = q.numel() * 2
    seen = []
    with torch.autograd.graph.saved_tensors_hooks(lambda x: seen.append(x) or x, lambda x: x):
        ops.packed_attention(*leaves, cu)
    assert sum(x.shape == q.shape for x in seen) == 3  # queries, output, what its rounding left
    assert sum(x.shape == (32, 4096) and x.dtype == torch.float32 for x in seen) == 1
    seen.clear()
    recomputed, held = _held(cuda, lambda: checkpoint(ops.packed_attention, *leaves, cu, use_reentrant=False))
    assert held < 1.25 * size
    with torch.autograd.graph.save_on_cpu():
        offloaded, held = _held(cuda, lambda: ops.packed_attention(*leaves, cu))
    assert held < 1.25 * size
    for out in (recomputed, offloaded):
        assert torch.equal(out.detach(), want[0])
        for got, ref in zip(torch.autograd.grad(out, leaves, dout), want[1:]):
            assert torch.equal(got, ref)
    assert ops.require().status(0) == 0


def test_a_hook_that_returns_something_else_is_refused(cuda):
    """Saved tensors that come back on another device, of another type or size reach no kernel."""
    q, k, v, cu, dout = _inputs(cuda, [40], 2, 1, 64, seed=42)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    for wrong in (lambda x: x.cpu(), lambda x: x.to(torch.float64), lambda x: x.flatten()[1:]):
        for i in range(3, 7):  # output, rest, log-sum-exps, plan
            count = iter(range(100))
            with torch.autograd.graph.saved_tensors_hooks(lambda x: (next(count), x),
                                                          lambda s: wrong(s[1]) if s[0] == i else s[1]):
                out = ops.packed_attention(*leaves, cu)
            with pytest.raises(RuntimeError, match="saved"):
                torch.autograd.grad(out, leaves, dout)


def test_forward_mode_and_second_derivatives_are_refused(cuda):
    """No tangent is dropped, no second derivative left out, without a word."""
    import torch.autograd.forward_ad as fwd

    q, k, v, cu, dout = _inputs(cuda, [30], 4, 2, 64, seed=43)
    with fwd.dual_level():
        for i in range(3):
            for requires_grad in (False, True):
                args = [q.detach().clone().requires_grad_(requires_grad), k, v]
                args[i] = fwd.make_dual(args[i], torch.ones_like(args[i]))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    ops.packed_attention(*args, cu)
    q.requires_grad_()
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad(ops.packed_attention(q, k, v, cu), (q,), dout, create_graph=True)


@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 64), (8, 1, 128), (3, 3, 80)])
@pytest.mark.parametrize("first", [True, False])
def test_one_long_sequence_beside_many_short_ones(cuda, heads, kv_heads, dim, first):
    """The mean length, by which CTAs take one query tile or two and share key tiles or not, is that of neither."""
    short = [1 + i % 5 for i in range(400)] + [0] * 30
    lens = [2500, *short] if first else [*short[:200], 2500, *short[200:]]
    q, k, v, cu, dout = _inputs(cuda, lens, heads, kv_heads, dim, pad=3, seed=44)
    z = _oracle(q, k, v, lens, dout, dim ** -0.5)
    for name, got in zip(("out", "dq", "dk", "dv"), _run(q, k, v, cu, dout)):
        _within(got, z, name)
    assert ops.require().status(0) == 0
