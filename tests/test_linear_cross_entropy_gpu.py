"""The readout cross-entropy against the same formula in 64 bits, element by element.

Tolerances (bf16 inputs are exact in 64 bits, so only the kernels round):

* a logit is an fp32 accumulation of H products: at most ``H 2^-23`` of the sum of their magnitudes;
* ``dz`` is rounded to bf16 once (8 significant bits: ``2^-8`` relative) from an fp16 probability (``2^-11`` relative, ``2^-25`` of its
  piece's largest absolute) and a log-sum-exp off by a logit's error;
* ``dx`` and ``dW`` sum ``dz`` times exact factors in fp32 and are rounded to bf16 once more.
"""

import pytest
import torch

from economize_b200 import ops

pytestmark = pytest.mark.gpu


def _inputs(dev, rows, hidden, vocab, masked=0.0, seed=0, lean=8.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    w = (torch.randn(vocab, hidden, device=dev, generator=g) * 0.05).bfloat16()
    y = torch.randint(0, vocab, (rows,), device=dev, generator=g)
    x = torch.randn(rows, hidden, device=dev, generator=g)
    near = w[y].float()
    x = x + lean * torch.rand(rows, 1, device=dev, generator=g) * near / near.norm(dim=-1, keepdim=True)
    y[torch.rand(rows, device=dev, generator=g) < masked] = -100
    return x.bfloat16(), w, y


def _oracle(x, w, y, scale, g_rows):
    """64-bit losses and gradients, and the bounds of each output's error."""
    keep = y != -100
    h = x.shape[1]
    xd, wd = torch.where(keep[:, None], x, 0).double(), w.double()
    z = scale * xd @ wd.t()
    eps = abs(scale) * (xd.abs() @ wd.t().abs()).amax(-1) * h * 2.0 ** -23 + z.abs().amax(-1) * 2.0 ** -22
    logp = torch.log_softmax(z, -1)
    at = torch.where(keep, y, 0)
    nll = torch.where(keep, -logp.gather(1, at[:, None])[:, 0], 0.0)
    p = logp.exp()
    dz = p.clone()
    dz[torch.arange(len(y)), at] -= 1
    g = torch.where(keep, g_rows.double(), 0.0)[:, None] * scale
    dz, p = dz * g, p * g.abs()
    rel = 2.0 ** -8 + 2.0 ** -11 + 2.0 ** -16  # dz, e, the exponentials and factors
    dz_err = dz.abs() * rel + p * (2.5 * eps[:, None]) + g.abs() * 2.0 ** -25
    dx, dw = dz @ wd, dz.t() @ xd
    dx_err = dz_err @ wd.abs() + dx.abs() * 2.0 ** -8 + dz.abs() @ wd.abs() * 2.0 ** -14
    dw_err = dz_err.t() @ xd.abs() + dw.abs() * 2.0 ** -8 + dz.abs().t() @ xd.abs() * 2.0 ** -14
    return dict(nll=nll, dx=dx, dw=dw, nll_err=2.5 * eps + nll.abs() * 2.0 ** -20 + 2.0 ** -21, dx_err=dx_err,
                dw_err=dw_err, keep=keep)


def _within(got, want, err, what):
    off = (got.double() - want).abs()
    assert (off <= err + 1e-30).all(), f"{what}: {(off / (err + 1e-30)).max().item():.2f} times the bound"


SIZES = [(1, 8, 1), (1, 64, 7), (3, 72, 129), (16, 256, 1000), (65, 136, 255), (128, 64, 256), (129, 512, 4099),
         (300, 1000, 50257), (513, 256, 2048)]


@pytest.mark.parametrize("rows,hidden,vocab", SIZES)
@pytest.mark.parametrize("masked", [0.0, 0.4])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_losses_and_gradients(cuda, rows, hidden, vocab, masked, reduction):
    x, w, y = _inputs(cuda, rows, hidden, vocab, masked)
    x.requires_grad_()
    w.requires_grad_()
    scale = 0.75 if masked else 1.0
    loss = ops.linear_cross_entropy(x, w, y, reduction=reduction, logit_scale=scale)
    count = max(1, int((y != -100).sum()))
    if reduction == "none":
        up = torch.linspace(-1.0, 2.0, rows, device=cuda)
        g_rows = up
    else:
        up = torch.tensor(1.0, device=cuda)
        g_rows = torch.full((rows,), 1.0 / count if reduction == "mean" else 1.0, device=cuda)
    dx, dw = torch.autograd.grad(loss, (x, w), up)
    o = _oracle(x.detach(), w.detach(), y, scale, g_rows)
    if reduction == "none":
        _within(loss, o["nll"], o["nll_err"], "losses")
    else:
        div = count if reduction == "mean" else 1
        total, err = o["nll"].sum() / div, o["nll_err"][o["keep"]].sum() / div
        _within(loss, total, err + total.abs() * 2.0 ** -20, "loss")
    _within(dx, o["dx"], o["dx_err"], "dx")
    _within(dw, o["dw"], o["dw_err"], "dw")
    assert ops.require().status(0) == 0


@pytest.mark.parametrize("rows", [37, 119])
def test_what_all_rows_share_is_not_rounded(cuda, rows):
    """The mean's 1 / rows is no part of the gradients' rounded factor. Rounding dz ~ -1 / rows to bf16 shifts a whole
    gradient (1 / 37 and 1 / 119 by 2 parts in 1000); the independent roundings of E elements move the slope of
    one gradient against another by about 2^-8 / sqrt(E) = 2e-5 for the E here: 2e-4 is ten times that."""
    x, w, y = _inputs(cuda, rows, 1024, 600, seed=9)

    def grads(reduction):
        a, b = x.detach().requires_grad_(), w.detach().requires_grad_()
        loss = ops.linear_cross_entropy(a, b, y, reduction="none" if reduction == "rows" else reduction)
        return torch.autograd.grad(loss.mean() if reduction == "rows" else loss, (a, b))

    want = [g.double() for g in grads("sum")]
    for reduction in ("mean", "rows"):
        for got, ref in zip(grads(reduction), want):
            slope = (got.double() * rows * ref).sum() / ref.square().sum()
            assert abs(slope.item() - 1) < 2e-4


@pytest.mark.parametrize("first", [0.0, 1e-30, 3e-9, -2e5, 1e30])
def test_the_first_rows_gradient_is_any(cuda, first):
    """Rows' gradients are kept relative to the first row's where that is neither zero nor extreme."""
    x, w, y = _inputs(cuda, 40, 256, 700, seed=10)
    g = torch.randn(40, device=cuda)
    g[0] = first
    a, b = x.detach().requires_grad_(), w.detach().requires_grad_()
    dx, dw = torch.autograd.grad(ops.linear_cross_entropy(a, b, y, reduction="none"), (a, b), g)
    o = _oracle(x, w, y, 1.0, g)
    _within(dx, o["dx"], o["dx_err"], "dx")
    _within(dw, o["dw"], o["dw_err"], "dw")


@pytest.mark.parametrize("chunk", [64, 128, 320])
def test_chunks_of_rows(cuda, chunk):
    """Several chunks: every output as from one, weight gradients summed in fp32 in between."""
    x, w, y = _inputs(cuda, 333, 200, 1500, 0.2, seed=3)
    x.requires_grad_()
    w.requires_grad_()
    loss = ops.linear_cross_entropy(x, w, y, chunk_rows=chunk)
    dx, dw = torch.autograd.grad(loss, (x, w))
    count = int((y != -100).sum())
    o = _oracle(x.detach(), w.detach(), y, 1.0, torch.full((333,), 1.0 / count, device=cuda))
    _within(loss, o["nll"].sum() / count, o["nll_err"].sum() / count + 1e-6, "loss")
    _within(dx, o["dx"], o["dx_err"], "dx")
    _within(dw, o["dw"], o["dw_err"], "dw")


@pytest.mark.parametrize("rows", [1, 70, 300])
def test_no_row_has_a_target(cuda, rows):
    x, w, y = _inputs(cuda, rows, 64, 500)
    y.fill_(-100)
    x.fill_(float("nan"))
    x.requires_grad_()
    w.requires_grad_()
    for reduction in ("mean", "sum", "none"):
        loss = ops.linear_cross_entropy(x, w, y, reduction=reduction)
        dx, dw = torch.autograd.grad(loss.sum(), (x, w))
        assert (loss == 0).all() and (dx == 0).all() and (dw == 0).all()


def test_no_rows_at_all(cuda):
    w = torch.randn(40, 64, device=cuda).bfloat16().requires_grad_()
    x = torch.empty(0, 64, device=cuda, dtype=torch.bfloat16, requires_grad=True)
    y = torch.empty(0, dtype=torch.long, device=cuda)
    dx, dw = torch.autograd.grad(ops.linear_cross_entropy(x, w, y), (x, w))
    assert dx.shape == x.shape and (dw == 0).all()
    assert ops.linear_cross_entropy(x, w, y, reduction="none").shape == (0,)


def test_masked_rows_hold_anything(cuda):
    """NaN and infinities in ignored rows reach neither the loss nor a gradient."""
    x, w, y = _inputs(cuda, 200, 128, 700, 0.3, seed=5)
    clean = torch.where((y == -100)[:, None], torch.zeros_like(x), x)
    dirty = x.clone()
    dirty[y == -100] = float("nan")
    dirty[(y == -100).nonzero()[::2, 0]] = float("inf")
    out = []
    for states in (clean, dirty):
        s, v = states.clone().requires_grad_(), w.clone().requires_grad_()
        loss = ops.linear_cross_entropy(s, v, y)
        out.append((loss.detach(), *torch.autograd.grad(loss, (s, v))))
    for a, b in zip(*out):
        assert torch.equal(a, b)
    assert torch.isfinite(out[1][0])


def test_a_row_with_nan_states(cuda):
    """Its loss is NaN, as the formula's is, and only its own row of dx."""
    x, w, y = _inputs(cuda, 40, 64, 300, seed=6)
    x[7, 3] = float("nan")
    x.requires_grad_()
    losses = ops.linear_cross_entropy(x, w, y, reduction="none")
    (dx,) = torch.autograd.grad(losses, (x,), torch.ones_like(losses))
    bad = torch.arange(40, device=cuda) == 7
    assert torch.equal(torch.isnan(losses), bad)
    assert torch.equal(torch.isnan(dx).any(-1), bad)


def test_infinite_logits(cuda):
    """Vocabulary rows whose logit is minus infinity have probability zero (their gradient is that of zero weight)."""
    x, w, y = _inputs(cuda, 33, 64, 400, seed=7)
    x = x.abs()
    w[5:300] = float("-inf")
    y = torch.where((y >= 5) & (y < 300), 0, y)
    losses = ops.linear_cross_entropy(x, w, y, reduction="none")
    keep = torch.cat([torch.arange(5), torch.arange(300, 400)]).to(cuda)
    z = x.double() @ w[keep].double().t()
    at = torch.where(y < 5, y, y - 295)
    want = torch.logsumexp(z, -1) - z.gather(1, at[:, None])[:, 0]
    assert ((losses.double() - want).abs() <= 64 * 2.0 ** -22 * z.abs().amax(-1) + 1e-6).all()


def test_large_logits_do_not_overflow(cuda):
    x, w, y = _inputs(cuda, 60, 256, 900, seed=8)
    x, w = x * 40, w * 40
    x.requires_grad_()
    loss = ops.linear_cross_entropy(x, w, y)
    (dx,) = torch.autograd.grad(loss, (x,))
    o = _oracle(x.detach(), w, y, 1.0, torch.full((60,), 1 / 60, device=cuda))
    _within(loss, o["nll"].mean(), o["nll_err"].mean() + o["nll"].mean() * 2.0 ** -20, "loss")
    assert torch.isfinite(dx).all()


def test_strided_operands_and_leading_dimensions(cuda):
    x, w, y = _inputs(cuda, 96, 128, 640, 0.1, seed=9)
    wide_x = torch.full((96, 256), float("nan"), device=cuda, dtype=torch.bfloat16)
    wide_w = torch.full((640, 136), float("nan"), device=cuda, dtype=torch.bfloat16)
    wide_x[:, 64:192] = x
    wide_w[:, 8:] = w
    odd_x = torch.empty(96 * 129, device=cuda, dtype=torch.bfloat16)[: 96 * 129].view(96, 129)
    odd_x[:, 1:] = x
    want = ops.linear_cross_entropy(x, w, y)
    assert torch.equal(want, ops.linear_cross_entropy(wide_x[:, 64:192], wide_w[:, 8:], y))
    assert torch.equal(want, ops.linear_cross_entropy(odd_x[:, 1:], w.t().contiguous().t(), y))
    both = ops.linear_cross_entropy(x.view(4, 24, 128), w, y.view(4, 24), reduction="none")
    assert both.shape == (4, 24)
    assert torch.equal(both.flatten(), ops.linear_cross_entropy(x, w, y, reduction="none"))


def test_same_bits_every_time_and_twice_through_one_graph(cuda):
    x, w, y = _inputs(cuda, 257, 264, 3001, 0.2, seed=10)
    x.requires_grad_()
    w.requires_grad_()
    runs = []
    for _ in range(3):
        loss = ops.linear_cross_entropy(x, w, y)
        runs.append((loss, *torch.autograd.grad(loss, (x, w))))
    for a in runs[1:]:
        assert all(torch.equal(p, q) for p, q in zip(a, runs[0]))
    loss = ops.linear_cross_entropy(x, w, y)
    first = [t.clone() for t in torch.autograd.grad(loss * 2, (x, w), retain_graph=True)]
    second = torch.autograd.grad(loss * 2, (x, w))
    assert all(torch.equal(p, q) for p, q in zip(first, second))
    assert torch.equal(first[0], runs[0][1] * 2) and torch.equal(first[1], runs[0][2] * 2)


@pytest.mark.parametrize("rows", [40, 2500])
def test_as_a_cuda_graph(cuda, rows):
    x, w, y = _inputs(cuda, rows, 256, 1100, 0.3, seed=12)

    def step():
        a, b = x.detach().requires_grad_(), w.detach().requires_grad_()
        loss = ops.linear_cross_entropy(a, b, y)
        return (loss.detach(), *torch.autograd.grad(loss, (a, b)))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results = step()
    for _ in range(3):
        for t in results:
            t.zero_()
        graph.replay()
        for got, ref in zip(results, want):
            assert torch.equal(got, ref)
    assert ops.require().status(0) == 0


def test_only_what_is_asked_for(cuda):
    """A frozen weight or frozen states get no gradient; without any the losses are the same."""
    x, w, y = _inputs(cuda, 100, 128, 1000, 0.1, seed=11)
    base = ops.linear_cross_entropy(x, w, y)
    a = x.clone().requires_grad_()
    la = ops.linear_cross_entropy(a, w, y)
    la.backward()
    b = w.clone().requires_grad_()
    lb = ops.linear_cross_entropy(x, b, y)
    lb.backward()
    assert torch.equal(base, la.detach()) and torch.equal(base, lb.detach())
    with torch.no_grad():
        assert not ops.linear_cross_entropy(a, b, y).requires_grad


def test_autocast_takes_fp32_masters(cuda):
    x, w, y = _inputs(cuda, 50, 64, 300, seed=12)
    xf, wf = x.float().requires_grad_(), w.float().requires_grad_()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = ops.linear_cross_entropy(xf, wf, y)
    loss.backward()
    xb, wb = x.clone().requires_grad_(), w.clone().requires_grad_()
    ops.linear_cross_entropy(xb, wb, y).backward()
    assert xf.grad.dtype == torch.float32
    assert torch.equal(xf.grad, xb.grad.float()) and torch.equal(wf.grad, wb.grad.float())


def test_on_another_stream(cuda):
    x, w, y = _inputs(cuda, 120, 128, 2000, seed=13)
    want = ops.linear_cross_entropy(x, w, y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.linear_cross_entropy(x, w, y)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(want, got)


def test_target_out_of_range_is_ignored_and_reported(cuda):
    x, w, y = _inputs(cuda, 30, 64, 200, seed=14)
    y[4], y[9] = 200, -3
    masked = y.clone()
    masked[4] = masked[9] = -100
    ops.require().status(0)
    got = ops.linear_cross_entropy(x, w, y)
    assert ops.require().status(0) & 32
    assert torch.equal(got, ops.linear_cross_entropy(x, w, masked))
    assert ops.require().status(0) == 0


def test_refusals(cuda):
    x, w, y = _inputs(cuda, 10, 64, 50, seed=15)
    with pytest.raises(ValueError, match="reduction"):
        ops.linear_cross_entropy(x, w, y, reduction="max")
    with pytest.raises(ValueError, match="do not match"):
        ops.linear_cross_entropy(x[:, :32], w, y)
    with pytest.raises(ValueError, match="do not match"):
        ops.linear_cross_entropy(x, w, y[:5])
    with pytest.raises(RuntimeError, match="bfloat16"):
        ops.linear_cross_entropy(x.float(), w, y)
    with pytest.raises(RuntimeError, match="bfloat16"):
        ops.linear_cross_entropy(x, w.half(), y)
    with pytest.raises(RuntimeError, match="int64"):
        ops.linear_cross_entropy(x, w, y.int())
    with pytest.raises(RuntimeError, match="device"):
        ops.linear_cross_entropy(x, w.cpu(), y)
    with pytest.raises(RuntimeError, match="multiple of 8"):
        ops.linear_cross_entropy(x[:, :60].contiguous(), w[:, :60].contiguous(), y)


def test_saved_tensor_hooks_and_checkpointing(cuda):
    """The gradients that a mean or sum computes in its forward pass are saved as any other tensor: hooks see them, and
    what is offloaded or recomputed gives the same."""
    from torch.utils.checkpoint import checkpoint

    x, w, y = _inputs(cuda, 256, 512, 40000, 0.2, seed=16)
    x.requires_grad_()
    w.requires_grad_()
    want = torch.autograd.grad(ops.linear_cross_entropy(x, w, y), (x, w))
    seen = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: seen.append(t.shape) or t, lambda t: t):
        ops.linear_cross_entropy(x, w, y)
    assert sorted(seen) == sorted([x.shape, w.shape])

    def held(make):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated(cuda)
        loss = make()
        return loss, torch.cuda.memory_allocated(cuda) - before

    size = w.numel() * 2
    recomputed, kept = held(lambda: checkpoint(ops.linear_cross_entropy, x, w, y, use_reentrant=False))
    assert kept < size / 4
    with torch.autograd.graph.save_on_cpu():
        offloaded, kept = held(lambda: ops.linear_cross_entropy(x, w, y))
    assert kept < size / 4
    for loss in (recomputed, offloaded):
        for got, ref in zip(torch.autograd.grad(loss, (x, w)), want):
            assert torch.equal(got, ref)


@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_a_kept_graph_gives_the_same_again(cuda, reduction):
    """What a pass over a kept graph returns is the caller's: writing to it leaves the next pass alone. After a pass that
    does not keep it the graph is spent."""
    x, w, y = _inputs(cuda, 70, 128, 900, 0.2, seed=17)
    x.requires_grad_()
    w.requires_grad_()
    loss = ops.linear_cross_entropy(x, w, y, reduction=reduction).sum()
    want = [g.clone() for g in torch.autograd.grad(loss, (x, w), retain_graph=True)]
    for _ in range(2):
        got = torch.autograd.grad(loss, (x, w), retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        for g in got:
            g.fill_(3.0)
    (dx,) = torch.autograd.grad(loss, (x,))  # dW not asked for
    assert torch.equal(dx, want[0])
    with pytest.raises(RuntimeError, match="a second time"):
        torch.autograd.grad(loss, (x, w))


def test_forward_mode_and_second_derivatives_are_refused(cuda):
    """No tangent is dropped, no second derivative left out, without a word."""
    import torch.autograd.forward_ad as fwd

    x, w, y = _inputs(cuda, 10, 64, 50, seed=18)
    with fwd.dual_level():
        for i in range(2):
            for requires_grad in (False, True):
                args = [x.detach().clone().requires_grad_(requires_grad), w]
                args[i] = fwd.make_dual(args[i], torch.ones_like(args[i]))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    ops.linear_cross_entropy(*args, y)
    assert torch.isfinite(ops.linear_cross_entropy(x, w, y))
    x.requires_grad_()
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad(ops.linear_cross_entropy(x, w, y), (x,), create_graph=True)


def _rowwise(x, w, y, scale, g_rows, rows=600):
    """:func:`_oracle` over many rows, `rows` at a time."""
    parts = [_oracle(x[i:i + rows], w, y[i:i + rows], scale, g_rows[i:i + rows]) for i in range(0, len(y), rows)]
    o = {k: torch.cat([p[k] for p in parts]) for k in ("nll", "nll_err", "dx", "dx_err", "keep")}
    o["dw"] = sum(p["dw"] for p in parts)
    # the output is rounded once, not once for every part
    o["dw_err"] = sum(p["dw_err"] - p["dw"].abs() * 2.0 ** -8 for p in parts) + o["dw"].abs() * 2.0 ** -8
    return o


@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_rows_planned_by_a_kernel_of_their_own(cuda, reduction):
    """More rows than the gather kernel counts itself, and dW of few tiles, split along the rows."""
    x, w, y = _inputs(cuda, 2500, 256, 1100, 0.3, seed=19)
    x.requires_grad_()
    w.requires_grad_()
    count = int((y != -100).sum())
    up = torch.linspace(-1.0, 2.0, 2500, device=cuda) if reduction == "none" else torch.tensor(1.0, device=cuda)
    loss = ops.linear_cross_entropy(x, w, y, reduction=reduction)
    dx, dw = torch.autograd.grad(loss, (x, w), up)
    o = _oracle(x.detach(), w.detach(), y, 1.0, up if reduction == "none" else up.expand(2500) / count)
    if reduction == "none":
        _within(loss, o["nll"], o["nll_err"], "losses")
    else:
        total = o["nll"].sum() / count
        _within(loss, total, o["nll_err"][o["keep"]].sum() / count + total * 2.0 ** -20, "loss")
    _within(dx, o["dx"], o["dx_err"], "dx")
    _within(dw, o["dw"], o["dw_err"], "dw")
    assert ops.require().status(0) == 0


def _whole_and_splits(m, n, k, pairs):
    """Tiles of a product that are computed in one piece, and into how many the rest are split along K."""
    tiles, blocks = -(-m // 256) * -(-n // 256), -(-k // 64)
    rest = tiles % pairs
    splits = max(1, min(pairs // rest, blocks // 8)) if rest and (rest == tiles or blocks >= 64) else 1
    return (tiles - rest if splits > 1 else tiles), splits


def test_split_tiles_behind_whole_rounds(cuda):
    """Products of more tiles than CTA pairs whose last round is split along K: dX over the vocabulary, dW over the rows
    that the device counts."""
    rows, hidden, vocab = 5000, 1032, 5000
    x, w, y = _inputs(cuda, rows, hidden, vocab, 0.1, seed=20)
    count = int((y != -100).sum())
    pairs = torch.cuda.get_device_properties(cuda).multi_processor_count // 2
    if pairs == 74:
        for m, n, k in ((count, hidden, vocab), (vocab, hidden, count)):
            whole, splits = _whole_and_splits(m, n, k, pairs)
            assert whole == pairs and splits > 1
    x.requires_grad_()
    w.requires_grad_()
    loss = ops.linear_cross_entropy(x, w, y)
    dx, dw = torch.autograd.grad(loss, (x, w))
    o = _rowwise(x.detach(), w.detach(), y, 1.0, torch.full((rows,), 1.0 / count, device=cuda), rows=1000)
    total = o["nll"].sum() / count
    _within(loss, total, o["nll_err"][o["keep"]].sum() / count + total * 2.0 ** -20, "loss")
    _within(dx, o["dx"], o["dx_err"], "dx")
    _within(dw, o["dw"], o["dw_err"], "dw")
    assert ops.require().status(0) == 0


@pytest.mark.parametrize("masked", [0.02, 0.2])
def test_chunks_of_the_default_size(cuda, masked):
    """More than 1 GiB of probabilities: 3840 rows to a chunk here, the second one with rows or left with none."""
    rows, vocab = 4200, 131100
    x, w, y = _inputs(cuda, rows, 72, vocab, masked, seed=21)
    count = int((y != -100).sum())
    assert (count > 3840) == (masked < 0.1)
    x.requires_grad_()
    w.requires_grad_()
    loss = ops.linear_cross_entropy(x, w, y, reduction="sum")
    dx, dw = torch.autograd.grad(loss, (x, w))
    o = _rowwise(x.detach(), w.detach(), y, 1.0, torch.ones(rows, device=cuda))
    total = o["nll"].sum()
    _within(loss, total, o["nll_err"][o["keep"]].sum() + total * 2.0 ** -20, "loss")
    _within(dx, o["dx"], o["dx_err"], "dx")
    _within(dw, o["dw"], o["dw_err"], "dw")
    assert ops.require().status(0) == 0


def test_losses_in_chunks_of_the_default_size(cuda):
    """Losses alone keep 8 bytes for 128 logits: more than 1 GiB of them."""
    rows, vocab = 140000, 131100
    x, w, y = _inputs(cuda, rows, 64, vocab, 0.02, seed=22)
    losses = ops.linear_cross_entropy(x, w, y, reduction="none")
    keep, wd = y != -100, w.double()
    for i in range(0, rows, 2000):
        s = slice(i, i + 2000)
        xd, at = x[s].double(), torch.where(keep[s], y[s], 0)
        z = xd @ wd.t()
        want = torch.where(keep[s], torch.logsumexp(z, -1) - z.gather(1, at[:, None])[:, 0], 0.0)
        # the sum of magnitudes of a logit's products by the norms of its factors
        eps = xd.norm(dim=-1) * wd.norm(dim=-1).max() * 64 * 2.0 ** -23 + z.abs().amax(-1) * 2.0 ** -22
        _within(losses[s], want, 2.5 * eps + want.abs() * 2.0 ** -20 + 2.0 ** -21, "losses")
    assert ops.require().status(0) == 0


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_one_gradient_alone(cuda, reduction):
    """The gradient of the states under a frozen head, and of a head under frozen states, as of both together."""
    x, w, y = _inputs(cuda, 300, 136, 5000, 0.2, seed=23)
    up = torch.linspace(-1.0, 2.0, 300, device=cuda) if reduction == "none" else torch.tensor(1.0, device=cuda)

    def grads(*which):
        args = [x.detach(), w.detach()]
        for i in which:
            args[i].requires_grad_()
        loss = ops.linear_cross_entropy(*args, y, reduction=reduction)
        return torch.autograd.grad(loss, [args[i] for i in which], up)

    both = grads(0, 1)
    count = int((y != -100).sum())
    o = _oracle(x, w, y, 1.0, up if reduction == "none" else up.expand(300) / (count if reduction == "mean" else 1))
    for i, name in enumerate(("dx", "dw")):
        (alone,) = grads(i)
        _within(alone, o[name], o[name + "_err"], name)
        assert torch.equal(alone, both[i])


def test_gradients_of_infinite_logits(cuda):
    """Vocabulary rows of minus infinity have probability zero: their gradient is zero, the others' that of the rest of
    the vocabulary. The states' gradient is NaN: the product multiplies the zeros with the infinite rows, as the plain
    formula's does."""
    x, w, y = _inputs(cuda, 33, 64, 400, seed=7)
    x = x.abs()
    y = torch.where((y >= 5) & (y < 300), 0, y)
    keep = torch.cat([torch.arange(5), torch.arange(300, 400)]).to(cuda)
    g = torch.linspace(-1.0, 2.0, 33, device=cuda)
    o = _oracle(x, w[keep], torch.where(y < 5, y, y - 295), 1.0, g)
    w[5:300] = float("-inf")
    x.requires_grad_()
    w.requires_grad_()
    dx, dw = torch.autograd.grad(ops.linear_cross_entropy(x, w, y, reduction="none"), (x, w), g)
    assert (dw[5:300] == 0).all() and torch.isnan(dx).all()
    _within(dw[keep], o["dw"], o["dw_err"], "dw")


def test_gradients_of_large_logits(cuda):
    x, w, y = _inputs(cuda, 60, 256, 900, seed=8)
    x, w = (x * 40).requires_grad_(), (w * 40).requires_grad_()
    dx, dw = torch.autograd.grad(ops.linear_cross_entropy(x, w, y), (x, w))
    o = _oracle(x.detach(), w.detach(), y, 1.0, torch.full((60,), 1 / 60, device=cuda))
    _within(dx, o["dx"], o["dx_err"], "dx")
    _within(dw, o["dw"], o["dw_err"], "dw")


@pytest.mark.parametrize("upstream", [1 / 3, -0.7, 4.0])
def test_upstream_gradients(cuda, upstream):
    """The gradients of a mean are rounded before the upstream gradient is known: their product with it is rounded once
    more (a power of two leaves them as they are)."""
    x, w, y = _inputs(cuda, 90, 264, 1300, 0.2, seed=24)
    x.requires_grad_()
    w.requires_grad_()
    dx, dw = torch.autograd.grad(ops.linear_cross_entropy(x, w, y) * upstream, (x, w))
    count = int((y != -100).sum())
    o = _oracle(x.detach(), w.detach(), y, 1.0, torch.full((90,), upstream / count, device=cuda))
    again = 0.0 if upstream == 4.0 else 2.0 ** -8 * (1 + 2.0 ** -7)
    _within(dx, o["dx"], o["dx_err"] + again * (o["dx"].abs() + o["dx_err"]), "dx")
    _within(dw, o["dw"], o["dw_err"] + again * (o["dw"].abs() + o["dw_err"]), "dw")


@pytest.mark.parametrize("hidden", [512, 1000, 1032, 2560, 4096])
def test_long_sums_do_not_shrink(cuda, hidden):
    """The tensor cores cut off what an accumulator cannot hold, towards zero, at every 16 products: in one sum of 4096
    the logits, and so every loss, came out 4 millionths too small. A sum of 1024 products is cut 64 times, by half of its
    last place (2^-24 of itself) on average, while it grows to its full size: 64 2^-25 = 1.9e-6 of itself. Sums of sums
    are rounded, which has no direction. Read from the losses of a vocabulary of two, of which one logit is zero:
    nll = log(1 + exp z)."""
    rows = 40000
    g = torch.Generator(device=cuda).manual_seed(25)
    w = torch.zeros(2, hidden, device=cuda)
    w[1] = torch.randn(hidden, device=cuda, generator=g) * (1.28 / hidden ** 0.5)
    w = w.bfloat16()
    lean = (2 * torch.rand(rows, 1, device=cuda, generator=g) - 1) * 6.25
    x = (torch.randn(rows, hidden, device=cuda, generator=g) + lean * w[1].float() / w[1].float().norm()).bfloat16()
    z = x.double() @ w[1].double()
    nll = ops.linear_cross_entropy(x, w, torch.zeros(rows, device=cuda, dtype=torch.long), reduction="none").double()
    off = torch.log(torch.expm1(nll)) - z
    assert abs((off * z).sum() / z.square().sum()) <= 64 * 2.0 ** -25
