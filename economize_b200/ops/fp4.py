"""4-bit floating point operands (MXFP4 and NVFP4) and their products: activations and weights both in 4 bits.

:func:`quantize` turns bf16 rows into an :class:`FP4Tensor`; :class:`FP4Weight` holds a ``[N, K]`` weight in the same
form, and :func:`economize_b200.ops.linear` multiplies the two on the tensor cores' block-scaled 4-bit path
(``csrc/fp4.cu``, ``csrc/gemm_fp4.cu``). The CPU path quantises with the same rules and multiplies the dequantised
operands in fp32. (The weight-only formats of :mod:`.quant`, which keep bf16 activations, are another product.)

A value is an E2M1 code (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives; ties go to the even code) times scales:

* ``mxfp4``: one power of two per 32 columns, ``2^(E - 2)`` with ``E`` the exponent of the group's largest magnitude,
  twice that when its mantissa is 1.75 or more; kept between 2^-126 and 2^125.
* ``nvfp4``: one e4m3 scale per 16 columns, the group's largest magnitude over 6 (at least 2^-9), in units of a power of
  two per row: the smallest (from 2^-100 on) that is no less than the row's largest magnitude over 2688 = 6 x 448. The
  row's power of two takes the place of a calibrated scale per tensor, is found in the same pass, and is exact.

A group that holds an infinity or a NaN gets the scale format's NaN: its values, and the products that read them, are NaN.
Infinities do not raise the row's power of two.
"""

from __future__ import annotations

import torch
from torch import nn

from ..errors import ConfigError
from ._ext import require
from .quant import E2M1_VALUES, e2m1_round

__all__ = ["FORMATS", "FP4Tensor", "FP4Weight", "quantize"]

#: kernel format codes (``csrc/fp4_common.cuh``)
FORMATS = {"nvfp4": 1, "mxfp4": 2}
GROUPS = {"nvfp4": 16, "mxfp4": 32}
#: columns of one K block of the product; scales are padded to whole blocks
BLOCK_K = 256
_ROWS = 128  # rows of a tile of scales


def _check_format(fmt: str) -> None:
    if fmt not in FORMATS:
        raise ConfigError(f"unknown 4-bit format {fmt!r} (one of {', '.join(FORMATS)})")


def _tiles(columns: int, fmt: str) -> int:
    """Tiles of 4 groups along the columns, in whole K blocks."""
    return (columns + BLOCK_K - 1) // BLOCK_K * (BLOCK_K // (4 * GROUPS[fmt]))


def _tile_scales(scales: torch.Tensor, columns: int, fmt: str) -> torch.Tensor:
    """Scale bytes ``[rows, groups]`` in the kernels' order ``[rows / 128, tiles, 512]``: row ``r`` and group ``g`` of a
    tile at ``(r % 32) * 16 + (r // 32) * 4 + g``, zeros in the padding."""
    rows, groups = scales.shape
    tiles, high = _tiles(columns, fmt), (rows + _ROWS - 1) // _ROWS
    padded = scales.new_zeros(high * _ROWS, tiles * 4)
    padded[:rows, :groups] = scales
    return padded.view(high, 4, 32, tiles, 4).permute(0, 3, 2, 1, 4).reshape(high, tiles, 4 * _ROWS)


def _flat_scales(tiled: torch.Tensor, rows: int, columns: int, fmt: str) -> torch.Tensor:
    """Inverse of :func:`_tile_scales`."""
    high, tiles, _ = tiled.shape
    flat = tiled.view(high, tiles, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(high * _ROWS, tiles * 4)
    return flat[:rows, : columns // GROUPS[fmt]]


def _power(exponent: torch.Tensor) -> torch.Tensor:
    """``2^exponent`` in fp32, for whole exponents between -126 and 127."""
    return ((exponent.to(torch.int32) + 127) << 23).view(torch.float32)


def _powers_of_two(row: torch.Tensor) -> bool:
    """Whether ``row`` holds such scales alone (kernels multiply with them in 8 bits, and in an order that stays in range).
    Not looked at where that is not possible: without memory, or in a CUDA graph's capture."""
    if row.is_meta or row.numel() == 0 or row.is_cuda and torch.cuda.is_current_stream_capturing():
        return True
    mantissa, exponent = torch.frexp(row.detach().float())
    return bool(((mantissa == 0.5) & (exponent >= -99) & (exponent <= 121)).all())


def _reference_quantize(x: torch.Tensor, fmt: str) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Codes, tiled scales and row scales of ``x [M, K]`` in PyTorch, by the rules above."""
    rows, columns = x.shape
    g = x.float().reshape(rows, columns // GROUPS[fmt], GROUPS[fmt])
    finite = g.isfinite()
    bad = ~finite.all(-1)
    g = torch.where(finite, g, 0.0)
    top = g.abs().amax(-1)
    if fmt == "mxfp4":
        mantissa, exponent = torch.frexp(top)  # the mantissa in [0.5, 1)
        exponent = torch.where(top > 0, exponent - 3 + (mantissa >= 0.875), -126).clamp(-126, 125)
        unit = _power(exponent)
        scales = torch.where(bad, 255, exponent + 127).to(torch.uint8)
        row = x.new_zeros(0, dtype=torch.float32)
    else:
        mantissa, exponent = torch.frexp(top.amax(1) / 2688.0 if columns else top.new_zeros(rows))
        exponent = torch.where(mantissa > 0, exponent - (mantissa == 0.5).int(), 0).clamp(-100, 120)
        row = _power(exponent)
        g = g / row[:, None, None]
        scale = (top / row[:, None] / 6.0).clamp(min=2.0 ** -9).to(torch.float8_e4m3fn)
        unit = scale.float()
        scales = torch.where(bad, 0x7F, scale.view(torch.uint8).int()).to(torch.uint8)
    values = e2m1_round(g / unit[..., None])
    table = torch.tensor(E2M1_VALUES, dtype=torch.float32, device=x.device)
    index = torch.bucketize(values.abs(), table)
    codes = (index | ((values < 0) & (index > 0)).to(index.dtype) << 3).reshape(rows, columns // 2, 2)
    packed = (codes[..., 0] | codes[..., 1] << 4).to(torch.uint8)
    return packed, _tile_scales(scales, columns, fmt), row


def _reference_dequantize(codes: torch.Tensor, scales: torch.Tensor, row: torch.Tensor, fmt: str) -> torch.Tensor:
    rows, columns = codes.shape[0], codes.shape[1] * 2
    flat = _flat_scales(scales, rows, columns, fmt)
    if fmt == "mxfp4":
        unit = torch.where(flat == 255, float("nan"), torch.exp2(flat.float() - 127.0))
    else:
        unit = flat.contiguous().view(torch.float8_e4m3fn).float() * row[:, None]
    c = codes.to(torch.int64)
    c = torch.stack([c & 15, c >> 4], -1).reshape(rows, columns)
    table = torch.tensor(E2M1_VALUES, dtype=torch.float32, device=codes.device)
    values = torch.where(c >= 8, -table[c & 7], table[c & 7])
    return (values.view(rows, -1, GROUPS[fmt]) * unit[..., None]).reshape(rows, columns)


class FP4Tensor:
    """Rows of a tensor ``[..., K]`` in 4 bits, in one buffer of bytes.

    Attributes:
        data: The buffer (uint8): tiled scales, codes and row scales (:meth:`parts`), each from a multiple of 256 bytes on.
        fmt: ``"nvfp4"`` or ``"mxfp4"``.
        shape: Of the tensor the codes stand for.
    """

    __slots__ = ("data", "fmt", "shape")

    def __init__(self, data: torch.Tensor, fmt: str, shape: torch.Size) -> None:
        self.data, self.fmt, self.shape = data, fmt, shape

    @property
    def is_cuda(self) -> bool:
        return self.data.is_cuda

    @property
    def device(self) -> torch.device:
        return self.data.device

    @property
    def dtype(self) -> torch.dtype:
        return torch.bfloat16  # of the values, which bf16 holds exactly

    @property
    def rows(self) -> int:
        n = 1
        for d in self.shape[:-1]:
            n *= d
        return n

    @property
    def codes(self) -> torch.Tensor:
        """uint8 ``[M, K / 2]``, column ``2b`` in the low nibble of byte ``b``."""
        return self.parts()[0]

    @property
    def scales(self) -> torch.Tensor:
        """Scale bytes (e4m3 or E8M0) in tiles ``[M / 128, tiles, 512]`` as the tensor cores read them."""
        return self.parts()[1]

    @property
    def row_scale(self) -> torch.Tensor:
        """fp32 powers of two ``[M]`` (nvfp4), else empty."""
        return self.parts()[2]

    def parts(self) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """Views of the buffer: codes, scales, row scales."""
        rows, columns = self.rows, self.shape[-1]
        high = (rows + _ROWS - 1) // _ROWS
        tiles = _tiles(columns, self.fmt)
        at = high * tiles * 4 * _ROWS
        end = at + rows * columns // 2
        row = _round_up(end)
        return (self.data[at:end].view(rows, columns // 2), self.data[:at].view(high, tiles, 4 * _ROWS),
                self.data[row:row + (4 * rows if self.fmt == "nvfp4" else 0)].view(torch.float32))

    def nbytes(self) -> int:
        return self.data.numel()

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The values the codes stand for, exact in bf16 and fp32 (those beyond a type's range, which only rows near
        bf16's largest values have, become infinite)."""
        shape = self.shape
        if self.data.is_cuda:
            rows = shape[0] if len(shape) == 2 else self.rows
            out = require().fp4_values(self.data, rows, shape[-1], FORMATS[self.fmt])
        else:
            out = _reference_dequantize(*self.parts(), self.fmt)
        if out.dtype != dtype:
            out = out.to(dtype)
        return out if len(shape) == 2 else out.reshape(shape)

    def __repr__(self) -> str:
        return f"FP4Tensor({tuple(self.shape)}, fmt={self.fmt!r}, device={self.device})"


def _round_up(n: int) -> int:
    return (n + 255) // 256 * 256


def _buffer(codes: torch.Tensor, scales: torch.Tensor, row_scale: torch.Tensor) -> torch.Tensor:
    """The parts of an :class:`FP4Tensor` in one buffer."""
    pad = codes.new_zeros(_round_up(codes.numel()) - codes.numel())
    return torch.cat([scales.reshape(-1), codes.reshape(-1), pad, row_scale.contiguous().view(torch.uint8)])


def quantize(x: torch.Tensor, fmt: str = "nvfp4") -> FP4Tensor:
    """``x [..., K]`` in 4 bits (bf16 on CUDA, any float type on the CPU; ``K`` a multiple of 32, at most 65536). The
    result carries no gradient."""
    _check_format(fmt)
    shape = x.shape
    if len(shape) < 1 or shape[-1] < 32 or shape[-1] % 32 or shape[-1] > 65536:
        raise ConfigError(f"4-bit rows need a multiple of 32 columns, up to 65536, got {tuple(shape)}")
    if x.is_cuda:
        return FP4Tensor(require().fp4_quantize(x, FORMATS[fmt]), fmt, shape)
    if not x.is_floating_point():
        raise ConfigError(f"4-bit rows are quantised from floating point, got {x.dtype}")
    return FP4Tensor(_buffer(*_reference_quantize(x.detach().reshape(-1, shape[-1]), fmt)), fmt, shape)


class FP4Weight(nn.Module):
    """A ``[out_features, in_features]`` weight in 4 bits whose products quantise their activations too (W4A4).

    ``linear`` takes bf16 activations, which it quantises row by row, or an :class:`FP4Tensor` of the same format that
    another operator left (:func:`economize_b200.ops.block_norm`). It is made for inference: its result carries no
    gradient (training paths multiply with :meth:`dequantize`). A row's result does not depend on how many rows there
    are, up to 128.

    Args:
        codes: uint8 ``[out_features, in_features / 2]``, as in :meth:`FP4Tensor.parts`.
        scales: Tiled scale bytes.
        row_scale: nvfp4: a power of two per row, from 2^-100 to 2^120 as :func:`quantize` makes them (another number,
            such as one scale for a whole tensor, belongs into the group scales); mxfp4: empty.
        fmt: ``"nvfp4"`` or ``"mxfp4"``.
        dtype: Of :meth:`dequantize`.
    """

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, row_scale: torch.Tensor, fmt: str,
                 dtype: torch.dtype = torch.bfloat16) -> None:
        super().__init__()
        _check_format(fmt)
        self.fmt = fmt
        self.out_features, self.in_features = int(codes.shape[0]), 2 * int(codes.shape[1])
        if self.in_features < 32 or self.in_features % 32 or self.in_features > 65536:
            raise ConfigError(f"4-bit weights need a multiple of 32 input columns, up to 65536, got {self.in_features}")
        high = (self.out_features + _ROWS - 1) // _ROWS
        if tuple(scales.shape) != (high, _tiles(self.in_features, fmt), 4 * _ROWS) or \
                row_scale.numel() != (self.out_features if fmt == "nvfp4" else 0):
            raise ConfigError(f"scales {tuple(scales.shape)} and {tuple(row_scale.shape)} do not belong to {fmt} codes "
                              f"{tuple(codes.shape)}")
        if not _powers_of_two(row_scale):
            raise ConfigError("the row scales of nvfp4 are powers of two from 2^-100 to 2^120")
        self.compute_dtype = dtype
        # copies of their own, not views of an operator's buffer
        self.register_buffer("codes", codes.detach().clone(memory_format=torch.contiguous_format))
        self.register_buffer("scales", scales.detach().clone(memory_format=torch.contiguous_format))
        self.register_buffer("row_scale", row_scale.detach().float().clone(memory_format=torch.contiguous_format))

    def _apply(self, fn, recurse: bool = True):
        """Moves like any module's, but a cast leaves the powers of two of the rows as they are: fp32, from 2^-100 on."""
        row = self.row_scale
        super()._apply(fn, recurse)
        moved = self._buffers["row_scale"]
        if moved.dtype != torch.float32:
            self._buffers["row_scale"] = row.to(moved.device)
        return self

    @classmethod
    def from_weight(cls, w: torch.Tensor, fmt: str = "nvfp4") -> FP4Weight:
        """``w [N, K]`` rounded to nearest (on CUDA from its bf16 values)."""
        if w.dim() != 2:
            raise ConfigError(f"a 4-bit weight is made from [N, K], got {tuple(w.shape)}")
        q = quantize(w.detach().to(torch.bfloat16) if w.is_cuda else w.detach(), fmt)
        return cls(*q.parts(), fmt, w.dtype)

    @property
    def shape(self) -> torch.Size:
        return torch.Size((self.out_features, self.in_features))

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @property
    def dtype(self) -> torch.dtype:
        return self.compute_dtype

    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel() + 4 * self.row_scale.numel()

    def dequantize(self, dtype: torch.dtype | None = None) -> torch.Tensor:
        if self.codes.is_cuda:
            out = require().fp4_dequantize(self.codes, self.scales, self.row_scale, FORMATS[self.fmt])
        else:
            out = _reference_dequantize(self.codes, self.scales, self.row_scale, self.fmt)
        return out.to(dtype or self.compute_dtype)

    def linear(self, x: torch.Tensor | FP4Tensor) -> torch.Tensor:
        """``x @ w.T`` with both operands in 4 bits: fp32 sums, rounded to bf16 on CUDA, in ``x``'s type."""
        if x.shape[-1] != self.in_features:
            raise ConfigError(f"activations {tuple(x.shape)} do not match a weight of {self.in_features} columns")
        b = self._buffers  # looked up once: a module's own lookup takes longer than the launch
        codes, scales, row_scale = b["codes"], b["scales"], b["row_scale"]
        if isinstance(x, FP4Tensor):
            if x.fmt != self.fmt:
                raise ConfigError(f"{x.fmt} activations do not multiply with an {self.fmt} weight")
            if x.data.is_cuda:
                rows = x.shape[0] if len(x.shape) == 2 else x.rows
                y = require().fp4_matmul(x.data, rows, self.in_features, codes, scales, row_scale, FORMATS[self.fmt])
                return y if len(x.shape) == 2 else y.reshape(*x.shape[:-1], self.out_features)
        elif x.is_cuda:
            return require().linear_fp4(x, codes, scales, row_scale, FORMATS[self.fmt])
        if codes.is_cuda:
            raise ConfigError(f"activations on {x.device}, weight on {self.device}")
        with torch.no_grad():
            q = x if isinstance(x, FP4Tensor) else quantize(x, self.fmt)
            y = q.dequantize(torch.float32).reshape(-1, self.in_features) @ self.dequantize(torch.float32).t()
            return y.to(x.dtype).reshape(*x.shape[:-1], self.out_features)

    def extra_repr(self) -> str:
        return f"{self.out_features}x{self.in_features}, fmt={self.fmt}"
