"""Operators of training steps, with autograd: the readout cross-entropy, causal attention over packed documents, and
the norms around a block (which inference uses too).

On CUDA both directions are the hand-written kernels of ``csrc/readout.cu``, ``csrc/packed_attention.cu``,
``csrc/packed_attention_bwd.cu`` and ``csrc/block_norm.cu`` (autograd functions in ``csrc/bindings_train.cpp`` and
``csrc/bindings_block.cpp``); CPU tensors take the formulas of :mod:`.reference`, which autograd differentiates in either
mode and any number of times. The kernels have the first reverse-mode derivative: dual tensors and ``create_graph=True``
are refused on CUDA. There is no third path.
"""

from __future__ import annotations

import math

import torch

from . import reference
from ._ext import require
from .fp4 import FORMATS, FP4Tensor, _check_format
from .fp4 import quantize as fp4_quantize

__all__ = ["block_norm", "linear_cross_entropy", "packed_attention"]

_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


def _autocast(*tensors: torch.Tensor) -> tuple[torch.Tensor, ...]:
    """Under CUDA autocast to bfloat16, the operands in bfloat16 (their gradients return in their own type)."""
    if tensors[0].is_cuda and torch.is_autocast_enabled("cuda") and \
            torch.get_autocast_dtype("cuda") == torch.bfloat16:
        return tuple(t.to(torch.bfloat16) for t in tensors)
    return tensors


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, *,
                         ignore_index: int = -100, reduction: str = "mean", logit_scale: float = 1.0,
                         chunk_rows: int = 0) -> torch.Tensor:
    """Softmax cross-entropy of ``logit_scale * hidden @ weight.T`` against ``targets`` without keeping the logits,
    differentiable in ``hidden`` and ``weight``.

    Args:
        hidden: States ``[..., H]`` (bf16 on CUDA, ``H`` a multiple of 8; cast under bf16 autocast).
        weight: The vocabulary rows ``[V, H]``.
        targets: Target ids ``[...]`` (int64). Rows whose target is ``ignore_index`` cost nothing, add nothing to the
            loss and get zero gradients, whatever their states hold (NaN included). Any other target outside ``[0, V)``
            is ignored on CUDA and reported in the device status word, and raises on the CPU.
        reduction: ``"mean"`` over the rows with a target (0 when there is none), ``"sum"``, or ``"none"``:
            per-row losses ``[...]`` (0 for ignored rows), whose backward pass computes the logits again.
        chunk_rows: Rows processed at a time (0: as many as 1 GiB of 16-bit probabilities hold, more where a trained
            ``weight`` needs as much for the sum over several chunks).

    On CUDA a mean or sum computes the gradients of what requires them with the loss, three products instead of one: take
    a loss that is not differentiated under ``torch.no_grad()``. They are rounded to bf16 there, and once more in the
    backward pass where the upstream gradient is no power of two (a loss divided by three batches).
    """
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {tuple(_REDUCTIONS)}, got {reduction!r}")
    if hidden.dim() < 1 or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"hidden {tuple(hidden.shape)} and weight {tuple(weight.shape)} do not match")
    if targets.shape != hidden.shape[:-1]:
        raise ValueError(f"targets {tuple(targets.shape)} do not match hidden {tuple(hidden.shape)}")
    if chunk_rows < 0:
        raise ValueError(f"chunk_rows must be 0 or more, got {chunk_rows}")
    hidden, weight = _autocast(hidden, weight)
    shape = targets.shape
    if hidden.dim() != 2:
        hidden, targets = hidden.reshape(-1, hidden.shape[-1]), targets.reshape(-1)
    if hidden.is_cuda:
        loss = require().linear_cross_entropy(hidden, weight, targets, ignore_index, logit_scale,
                                              _REDUCTIONS[reduction], chunk_rows)
    else:
        loss = reference.linear_cross_entropy(hidden, weight, targets, ignore_index, reduction, logit_scale)
    return loss.reshape(shape) if reduction == "none" and len(shape) != 1 else loss


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor,
                     scale: float | None = None) -> torch.Tensor:
    """Causal attention of packed sequences with grouped heads, differentiable in ``q``, ``k`` and ``v``.

    Args:
        q: Queries ``[T, H, D]`` of all sequences one after another (bf16 on CUDA; cast under bf16 autocast). Views
            with 16-byte strides (parts of a fused projection) are read in place.
        k, v: Keys and values ``[T, H_kv, D]``; query head ``h`` reads head ``h // (H / H_kv)``.
        cu_seqlens: int32 ``[B + 1]``: sequence ``i`` holds tokens ``cu_seqlens[i]`` to ``cu_seqlens[i + 1]``. A token
            attends itself and those before it in its sequence; empty sequences are allowed. Tokens outside every
            sequence (a row's padding) may hold anything: their outputs and gradients are zero.
        scale: Of the scores (``D ** -0.5``); positive.

    Head dimensions 8 to 128 in steps of 8 on CUDA. Offsets that fall or lie outside ``[0, T]`` are clamped on CUDA and
    reported in the device status word.
    """
    scale = float(scale if scale is not None else q.shape[-1] ** -0.5)
    q, k, v = _autocast(q, k, v)
    if not q.is_cuda:
        return reference.packed_attention(q, k, v, cu_seqlens, scale)
    return require().packed_attention(q, k, v, cu_seqlens, scale)


def block_norm(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, *,
               post_weight: torch.Tensor | None = None, gate: torch.Tensor | None = None, scale: float = 1.0,
               eps: float = 1e-6, quantize: str | None = None) -> tuple[torch.Tensor | FP4Tensor, torch.Tensor]:
    """The norms on both sides of a block's end, its gate, residual scale and residual sum in one pass: ``(normed,
    stream)`` with ``stream = residual + scale * gate * rms(x) * post_weight`` and ``normed = rms(stream) * weight``, where
    ``rms(v) = v / sqrt(mean(v^2) + eps)`` over the last dimension. Differentiable in every tensor.

    Args:
        x: The block's output ``[..., H]`` (``H`` up to 16384; bf16, fp16 or fp32 on CUDA, rows may be strided).
        residual: The stream that enters the block, like ``x``; ``None``: nothing is added.
        weight: Of the norm before the next block, ``[H]``.
        post_weight: Of the norm behind the block, ``[H]``; ``None``: no such norm.
        gate: Per token ``[..., 1]`` or per element ``[..., H]``; ``None``: ungated.
        scale: Factor of what joins the residual.
        quantize: ``"nvfp4"`` or ``"mxfp4"``: ``normed`` comes in 4 bits, as an
            :class:`~economize_b200.ops.fp4.FP4Tensor` of the bf16 result (bf16 on CUDA, ``H`` a multiple of 32) without
            a gradient; ``stream`` keeps its own. (Where one is asked for, the norm and the quantisation are two kernels.)

    All operands have one type (under bf16 autocast they are cast, under fp16 autocast where their types differ). Sums and
    what lies between are fp32; ``stream`` and ``normed`` are rounded once each, so ``normed`` is the norm of the unrounded
    stream (unlike two calls of :func:`~economize_b200.ops.rmsnorm`, which round in between as Hugging Face's modules do).
    Gradients are taken from the unrounded stream, which the backward pass forms again from ``x`` and ``residual``; without
    ``post_weight`` and ``gate`` and with ``scale=1`` those of ``x`` and ``residual`` are one tensor. A call captured into a
    CUDA graph with its backward pass needs leaves that no living graph of the default stream holds; where an operand is
    such a leaf, or a view or a cast of one, the call is refused.
    """
    if x.is_cuda:  # the checks are the extension's, in C++
        if torch.is_autocast_enabled("cuda"):
            to, given = torch.get_autocast_dtype("cuda"), (x, residual, weight, post_weight, gate)
            if to == torch.bfloat16 or to == torch.float16 and quantize is None and \
                    any(t is not None and t.dtype != x.dtype for t in given):
                x, residual, weight, post_weight, gate = (None if t is None else t.to(to) for t in given)
        if quantize is None:
            return require().block_norm(x, residual, weight, post_weight, gate, scale, eps)
        _check_format(quantize)
        data, stream = require().block_norm_fp4(x, residual, weight, post_weight, gate, scale, eps, FORMATS[quantize])
        return FP4Tensor(data, quantize, x.shape), stream
    given = [t for t in (x, residual, weight, post_weight, gate) if t is not None]
    if x.dim() < 1 or weight.dim() != 1 or x.shape[-1] != weight.shape[0]:
        raise ValueError(f"x {tuple(x.shape)} and weight {tuple(weight.shape)} do not match")
    if post_weight is not None and post_weight.shape != weight.shape:
        raise ValueError(f"post_weight {tuple(post_weight.shape)} and weight {tuple(weight.shape)} do not match")
    if residual is not None and residual.shape != x.shape:
        raise ValueError(f"residual {tuple(residual.shape)} does not match x {tuple(x.shape)}")
    if gate is not None and gate.shape not in (x.shape, (*x.shape[:-1], 1)):
        raise ValueError(f"gate {tuple(gate.shape)} must be {(*x.shape[:-1], 1)} or {tuple(x.shape)}")
    if any(t.dtype != x.dtype or t.device != x.device for t in given):
        raise ValueError("all operands must have one type and device, got "
                         + ", ".join(f"{t.dtype} on {t.device}" for t in given))
    if not x.is_floating_point() or not math.isfinite(scale) or not 0.0 <= eps < math.inf:
        raise ValueError(f"block_norm takes floating point and a finite scale and eps >= 0, got {x.dtype}, {scale}, {eps}")
    if quantize is not None:
        _check_format(quantize)
    normed, stream = reference.block_norm(x, residual, weight, post_weight, gate, float(scale), float(eps))
    return (normed, stream) if quantize is None else (fp4_quantize(normed, quantize), stream)
