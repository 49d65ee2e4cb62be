"""4-bit floating-point rows: quantisation, its inverse, the product, and a linear layer on them.

Two formats of e2m1 codes (two a byte, the even column in the low nibble) under block scales:
  * "nvfp4": blocks of 16 columns, e4m3 scales, one fp32 scale per row on top;
  * "mxfp4": blocks of 32 columns, e8m0 scales (powers of two).
Block scales are kept in the order in which the tensor core reads them, uint8 [ceil(rows / 128), ceil(blocks / 4),
32, 4, 4]: element [R, C, r, j, c] is the scale of row 128 R + 32 j + r, block 4 C + c; blocks past the row hold zeros
(``tile_scales`` brings a [rows, blocks] matrix into it). e4m3 scales are not negative. Widths are multiples of 32.
"""
from __future__ import annotations

import torch
from torch import nn

from . import _lib
from ._lib import check, ptr, stream_of

__all__ = ["quantize_rows_fp4", "dequantize_rows_fp4", "fp4_matmul", "tile_scales", "Fp4Linear"]

FORMATS = {"nvfp4": (_lib.LR_FP4_NV, 16), "mxfp4": (_lib.LR_FP4_MX, 32)}


def _format(name: str, format: str):
    if format not in FORMATS:
        raise ValueError(f"{name}: format must be one of {sorted(FORMATS)}, got {format!r}")
    return FORMATS[format]


def _scale_shape(rows: int, width: int, block: int):
    return (rows + 127) // 128, (width // block + 3) // 4, 32, 4, 4


def _check_packed(name: str, what: str, codes: torch.Tensor, scales: torch.Tensor, block: int):
    """(rows, width) of a packed matrix whose codes and scales fit each other."""
    if codes.dtype != torch.uint8 or codes.ndim != 2 or not codes.is_contiguous():
        raise ValueError(f"{name}: {what} codes must be a contiguous uint8 [rows, width / 2] tensor")
    rows, half = codes.shape
    shape = _scale_shape(rows, 2 * half, block)
    if scales.dtype != torch.uint8 or scales.shape != shape or not scales.is_contiguous() or scales.device != codes.device:
        raise ValueError(f"{name}: {what} scales must be contiguous uint8 {shape} on the codes' device, "
                         f"got {scales.dtype} {tuple(scales.shape)}")
    return rows, 2 * half


def _vector(name: str, what: str, t: torch.Tensor, count: int, dtype: torch.dtype, device):
    if t.dtype != dtype or t.numel() != count or t.device != device:
        raise ValueError(f"{name}: {what} must hold {count} {dtype} values on the codes' device")
    return t.contiguous()


def tile_scales(scales: torch.Tensor) -> torch.Tensor:
    """[rows, blocks] scale bytes (uint8, or any 1-byte type) -> the tiled order, zeros past the matrix."""
    if scales.ndim != 2 or scales.element_size() != 1:
        raise ValueError("tile_scales: expected a [rows, blocks] matrix of 1-byte scales")
    rows, blocks = scales.shape
    whole = torch.zeros(((rows + 127) // 128 * 128, (blocks + 3) // 4 * 4), dtype=torch.uint8, device=scales.device)
    whole[:rows, :blocks] = scales.view(torch.uint8)
    return whole.unflatten(0, (-1, 4, 32)).unflatten(3, (-1, 4)).permute(0, 3, 2, 1, 4).contiguous()


def quantize_rows_fp4(value: torch.Tensor, *, format: str = "nvfp4"):
    """bf16 [rows, width] -> (codes uint8 [rows, width / 2], tiled scales, row scales fp32 [rows, 1]; None for mxfp4).

    Rows may be strided (unit column stride). Nearest even, saturating; a row (nvfp4) or block (mxfp4) with an infinity
    or a NaN gets a NaN scale."""
    code, block = _format("quantize_rows_fp4", format)
    if value.dtype != torch.bfloat16 or value.ndim != 2:
        raise ValueError(f"quantize_rows_fp4: expected a bf16 [rows, width] tensor, got {value.dtype} {tuple(value.shape)}")
    rows, width = value.shape
    if width == 0 or width % 32:
        raise ValueError(f"quantize_rows_fp4: the width must be a positive multiple of 32, got {width}")
    stride, column_stride = value.stride()
    if column_stride != 1 or (rows > 1 and (stride % 8 or stride < width)) or value.data_ptr() % 16:
        value, stride = value.clone(memory_format=torch.contiguous_format), width
    device = value.device
    codes = torch.empty(rows, width // 2, dtype=torch.uint8, device=device)
    scales = torch.empty(*_scale_shape(rows, width, block), dtype=torch.uint8, device=device)
    row_scale = torch.empty(rows, 1, dtype=torch.float32, device=device) if block == 16 else None
    check(_lib.load().lr_fp4_quantize_rows(value.data_ptr(), rows, width, stride, code, codes.data_ptr(), scales.data_ptr(),
                                           ptr(row_scale), stream_of(value)), "quantize_rows_fp4")
    return codes, scales, row_scale


def dequantize_rows_fp4(codes: torch.Tensor, scales: torch.Tensor, row_scale: torch.Tensor | None = None, *,
                        format: str = "nvfp4") -> torch.Tensor:
    """The values of packed rows: bf16 [rows, width], code * (scale * row_scale) rounded once."""
    code, block = _format("dequantize_rows_fp4", format)
    rows, width = _check_packed("dequantize_rows_fp4", "the", codes, scales, block)
    if row_scale is not None:
        row_scale = _vector("dequantize_rows_fp4", "row_scale", row_scale, rows, torch.float32, codes.device)
    output = torch.empty(rows, width, dtype=torch.bfloat16, device=codes.device)
    check(_lib.load().lr_fp4_dequantize_rows(ptr(codes), ptr(scales), ptr(row_scale), rows, width, code, ptr(output),
                                             stream_of(codes)), "dequantize_rows_fp4")
    return output


def fp4_matmul(a_codes: torch.Tensor, a_scales: torch.Tensor, b_codes: torch.Tensor, b_scales: torch.Tensor,
               row_scale: torch.Tensor | None = None, column_scale: torch.Tensor | None = None,
               bias: torch.Tensor | None = None, *, format: str = "nvfp4") -> torch.Tensor:
    """bf16 [M, N] = (A B^T) * row_scale[m] * column_scale[n] + bias[n], accumulated in fp32 and rounded once.

    A: [M, K] packed rows (activations), B: [N, K] packed rows (a weight, one row per output); both of ``format``."""
    code, block = _format("fp4_matmul", format)
    m, k = _check_packed("fp4_matmul", "a", a_codes, a_scales, block)
    n, kb = _check_packed("fp4_matmul", "b", b_codes, b_scales, block)
    if k != kb or b_codes.device != a_codes.device:
        raise ValueError(f"fp4_matmul: operands of widths {k} and {kb} (and one device) are wanted to be alike")
    if n == 0 or k == 0:
        raise ValueError("fp4_matmul: empty weight")
    device = a_codes.device
    if row_scale is not None:
        row_scale = _vector("fp4_matmul", "row_scale", row_scale, m, torch.float32, device)
    if column_scale is not None:
        column_scale = _vector("fp4_matmul", "column_scale", column_scale, n, torch.float32, device)
    if bias is not None:
        bias = _vector("fp4_matmul", "bias", bias, n, torch.bfloat16, device)
    output = torch.empty(m, n, dtype=torch.bfloat16, device=device)
    check(_lib.load().lr_fp4_gemm(a_codes.data_ptr(), a_scales.data_ptr(), b_codes.data_ptr(), b_scales.data_ptr(), m, n, k,
                                  code, ptr(row_scale), ptr(column_scale), ptr(bias), output.data_ptr(), n,
                                  stream_of(a_codes)), "fp4_matmul")
    return output


class Fp4Linear(nn.Module):
    """A linear layer with a 4-bit weight whose inputs are quantised to 4 bits on the fly."""

    def __init__(self, linear: nn.Linear, *, format: str = "nvfp4"):
        super().__init__()
        weight = linear.weight.detach().to(torch.bfloat16)
        codes, scales, row_scale = quantize_rows_fp4(weight, format=format)
        self._assign(codes, scales, row_scale, None if linear.bias is None else linear.bias.detach(), format)

    @classmethod
    def from_packed(cls, codes, scales, weight_scale=None, bias=None, *, format: str = "nvfp4") -> "Fp4Linear":
        """From a packed weight [out_features, in_features]: codes, tiled scales, and fp32 scales per output (or None)."""
        layer = cls.__new__(cls)
        nn.Module.__init__(layer)
        layer._assign(codes, scales, weight_scale, bias, format)
        return layer

    def _assign(self, codes, scales, weight_scale, bias, format):
        _, block = _format("Fp4Linear", format)
        self.format = format
        self.out_features, self.in_features = _check_packed("Fp4Linear", "weight", codes, scales, block)
        self.register_buffer("weight_codes", codes)
        self.register_buffer("weight_scales", scales)
        self.register_buffer("weight_scale", None if weight_scale is None else weight_scale.reshape(-1).float())
        self.register_buffer("bias", None if bias is None else bias.to(torch.bfloat16))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        codes, scales, row_scale = quantize_rows_fp4(x.reshape(-1, x.shape[-1]), format=self.format)
        return self.forward_quantized(codes, scales, row_scale, x.shape[:-1])

    def forward_quantized(self, codes, scales, row_scale, shape) -> torch.Tensor:
        """The product for rows that are quantised already (one quantisation for several layers)."""
        y = fp4_matmul(codes, scales, self.weight_codes, self.weight_scales, row_scale, self.weight_scale, self.bias,
                       format=self.format)
        return y.reshape(*shape, self.out_features)
