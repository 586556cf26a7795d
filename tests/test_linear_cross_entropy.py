"""The readout cross-entropy on the CPU path: the formula, masked rows, reductions, gradients by differences."""

import pytest
import torch
import torch.nn.functional as F

from economize_b200 import ops


def _inputs(rows=13, hidden=10, vocab=17, seed=0, dtype=torch.float64):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, hidden, generator=g, dtype=dtype)
    w = torch.randn(vocab, hidden, generator=g, dtype=dtype)
    y = torch.randint(0, vocab, (rows,), generator=g)
    y[2] = y[7] = -100
    return x, w, y


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_equals_cross_entropy_of_the_logits(reduction):
    x, w, y = _inputs()
    got = ops.linear_cross_entropy(x, w, y, reduction=reduction, logit_scale=0.3)
    want = F.cross_entropy(0.3 * x @ w.t(), y, reduction=reduction)
    torch.testing.assert_close(got, want, rtol=1e-12, atol=1e-12)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_gradients_by_differences(reduction):
    x, w, y = _inputs(rows=9, hidden=4, vocab=5, seed=1)
    x.requires_grad_()
    w.requires_grad_()
    assert torch.autograd.gradcheck(lambda a, b: ops.linear_cross_entropy(a, b, y, reduction=reduction), (x, w))


def test_masked_rows_hold_anything():
    x, w, y = _inputs(seed=2)
    dirty = x.clone()
    dirty[y == -100] = float("nan")
    dirty.requires_grad_()
    loss = ops.linear_cross_entropy(dirty, w, y)
    loss.backward()
    assert torch.equal(loss.detach(), ops.linear_cross_entropy(x, w, y))
    assert torch.isfinite(dirty.grad).all() and (dirty.grad[y == -100] == 0).all()


def test_no_row_has_a_target():
    x, w, y = _inputs(seed=3)
    y.fill_(-100)
    x.requires_grad_()
    loss = ops.linear_cross_entropy(x, w, y)
    loss.backward()
    assert loss == 0 and (x.grad == 0).all()
    assert (ops.linear_cross_entropy(x, w, y, reduction="none") == 0).all()


def test_leading_dimensions_and_refusals():
    x, w, y = _inputs(rows=12)
    losses = ops.linear_cross_entropy(x.view(3, 4, -1), w, y.view(3, 4), reduction="none")
    assert losses.shape == (3, 4)
    with pytest.raises(ValueError, match="reduction"):
        ops.linear_cross_entropy(x, w, y, reduction="max")
    with pytest.raises(ValueError, match="do not match"):
        ops.linear_cross_entropy(x, w[:, :3], y)
    with pytest.raises(ValueError, match="do not match"):
        ops.linear_cross_entropy(x, w, y[:3])


def test_forward_mode_and_second_derivatives():
    x, w, y = _inputs(rows=9, hidden=4, vocab=5, seed=4)
    x.requires_grad_()
    w.requires_grad_()
    loss = lambda a, b: ops.linear_cross_entropy(a, b, y)  # noqa: E731
    assert torch.autograd.gradcheck(loss, (x, w), check_forward_ad=True)
    assert torch.autograd.gradgradcheck(loss, (x, w))


@pytest.mark.parametrize("ignore", [-1, 3])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_only_ignore_index_is_ignored(ignore, reduction):
    """Any index may be the ignored one; another target outside the vocabulary is an error, -100 included."""
    x, w, y = _inputs(rows=12, seed=5)
    y[2] = y[7] = ignore
    got = ops.linear_cross_entropy(x, w, y, reduction=reduction, ignore_index=ignore)
    want = F.cross_entropy(x @ w.t(), y, reduction=reduction, ignore_index=ignore)
    torch.testing.assert_close(got, want, rtol=1e-12, atol=1e-12)
    for target in (-100, 17):
        bad = y.clone()
        bad[4] = target
        with pytest.raises(IndexError, match="out of bounds"):
            ops.linear_cross_entropy(x, w, bad, reduction=reduction, ignore_index=ignore)


def test_refuses_a_negative_chunk():
    x, w, y = _inputs()
    with pytest.raises(ValueError, match="chunk_rows"):
        ops.linear_cross_entropy(x, w, y, chunk_rows=-64)
