"""Packed causal attention on the CPU path: against attention over each sequence alone, gradients by differences."""

import pytest
import torch
import torch.nn.functional as F

from economize_b200 import ops


def _inputs(lens, heads=4, kv_heads=2, dim=6, pad=0, seed=0):
    g = torch.Generator().manual_seed(seed)
    t = sum(lens) + pad
    q, k, v = (torch.randn(t, h, dim, generator=g, dtype=torch.float64) for h in (heads, kv_heads, kv_heads))
    return q, k, v, torch.tensor([0, *lens]).cumsum(0).int()


@pytest.mark.parametrize("lens,pad", [([1], 0), ([5, 0, 3], 2), ([7, 2], 0)])
def test_each_sequence_alone(lens, pad):
    q, k, v, cu = _inputs(lens, pad=pad)
    out = ops.packed_attention(q, k, v, cu, 0.3)
    a = 0
    for n in lens:
        s = slice(a, a + n)
        if n:
            want = F.scaled_dot_product_attention(*(x[s].transpose(0, 1)[None] for x in (q, k, v)), is_causal=True,
                                                  scale=0.3, enable_gqa=True)[0].transpose(0, 1)
            torch.testing.assert_close(out[s], want, rtol=1e-12, atol=1e-12)
        a += n
    assert (out[a:] == 0).all()


def test_gradients_by_differences():
    q, k, v, cu = _inputs([3, 0, 4], heads=2, kv_heads=1, dim=3, pad=1)
    args = [x.requires_grad_() for x in (q, k, v)]
    assert torch.autograd.gradcheck(lambda *x: ops.packed_attention(*x, cu), args)


def test_refusals():
    q, k, v, cu = _inputs([4])
    with pytest.raises(ValueError, match="expects"):
        ops.packed_attention(q[:, :3], k, v, cu)
    with pytest.raises(ValueError, match="int32"):
        ops.packed_attention(q, k, v, cu.long())
    with pytest.raises(ValueError, match="offsets"):
        ops.packed_attention(q, k, v, torch.tensor([0, 3, 2]).int())
    with pytest.raises(ValueError, match="offsets"):
        ops.packed_attention(q, k, v, torch.tensor([0, 9]).int())


def test_forward_mode_and_second_derivatives():
    q, k, v, cu = _inputs([3, 0, 2], heads=2, kv_heads=1, dim=3, pad=1)
    args = [x.requires_grad_() for x in (q, k, v)]
    assert torch.autograd.gradcheck(lambda *x: ops.packed_attention(*x, cu), args, check_forward_ad=True)
    assert torch.autograd.gradgradcheck(lambda *x: ops.packed_attention(*x, cu), args)


@pytest.mark.parametrize("scale", [0.0, -1.0, float("inf"), float("nan")])
def test_refuses_a_scale_that_is_not_positive(scale):
    """As the kernels do."""
    q, k, v, cu = _inputs([4])
    with pytest.raises(ValueError, match="scale"):
        ops.packed_attention(q, k, v, cu, scale)
