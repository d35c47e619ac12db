"""Microscaled 4-bit values: 32 neighbouring values of a row share a power-of-two scale.  `quantise` writes them, `dequantise`
reads them back, `linear` multiplies two such matrices on the block-scaled matrix instructions and can leave its result in the same form.

The scale of a block is the smallest power of two that brings its largest magnitude to 6 or below, so nothing is cut off; a
value is then the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with its sign, ties to the even code.  A block that holds an infinity
or a NaN reads back as NaN.  For serving: there are no gradients.  `leaf_eval.Mx4ValueMLP` is a value network in this form.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from . import _lib

ACTIVATIONS = {"gelu": 0, "silu": 1, "none": 2}
_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
FEW_ROWS = 4  # up to so many rows are quantised by the product itself (p2b_mx4_few_rows)


@dataclass
class Mx4:
    """A matrix in 4 bits: `values` [rows, ceil(width/32)*16] bytes, two values a byte; `scales`, the blocks' exponents in the
    order in which the matrix instructions read them (include/poker2_b200.h); `shape` of what was quantised."""

    values: torch.Tensor
    scales: torch.Tensor
    shape: tuple
    _sound = None  # the arrays and shape that _check_layout has seen

    @property
    def device(self) -> torch.device:
        return self.values.device

    @property
    def rows(self) -> int:
        return self.values.shape[0]

    @property
    def width(self) -> int:
        return self.shape[-1]

    def dequantise(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values stood for, in bf16, fp16 or fp32 (exact but for what lies outside the type's range)."""
        kind, values = _TYPES.get(dtype), self.values
        if kind is None:
            raise ValueError("values are read back in bf16, fp16 or fp32")
        if values.get_device() < 0:
            _lib.require_cuda(values, "dequantise")
        _check_layout(self)
        out, width = values.new_empty(self.shape, dtype=dtype), self.shape[-1]
        _lib.call_on(values.get_device(), "p2b_mx4_dequantise", values.data_ptr(), self.scales.data_ptr(), values.shape[0], width, kind,
                     out.data_ptr(), width)
        return out


def _check_layout(m: Mx4) -> None:
    """The arrays hold what `shape` says (a kernel reads as far as that goes); looked at once for a matrix, 1 us."""
    values, scales, shape, seen = m.values, m.scales, m.shape, m._sound
    if seen is not None and seen[0] is values and seen[1] is scales and seen[2] is shape:
        return
    width, rows = shape[-1], shape[0] if len(shape) == 2 else math.prod(shape[:-1])
    if (values.nbytes != rows * ((width + 31) // 32 * 16) or scales.nbytes != (rows + 127) // 128 * ((width + 255) // 256) * 1024
            or values.shape[0] != rows or not values.is_contiguous() or not scales.is_contiguous() or scales.get_device() != values.get_device()):
        raise ValueError("the values and scales of a quantised matrix are packed, lie on one device and are as many as its shape says")
    m._sound = (values, scales, shape)


def _made(values: torch.Tensor, scales: torch.Tensor, shape: tuple) -> Mx4:
    m = Mx4(values, scales, shape)
    m._sound = (values, scales, shape)
    return m


def quantise(x: torch.Tensor) -> Mx4:
    """x [..., width], bf16, fp16 or fp32, any strides; the blocks lie along the last dimension, the last one may be short."""
    kind, shape, device = _TYPES.get(x.dtype), x.shape, x.get_device()
    _lib.refuse_tangents("quantise", x)
    if device < 0:
        _lib.require_cuda(x, "quantise")
    if kind is None:
        raise ValueError("quantise takes bf16, fp16 or fp32 tensors")
    if len(shape) < 1 or shape[-1] == 0:
        raise ValueError("quantise wants rows of at least one value")
    width = shape[-1]
    flat = x if len(shape) == 2 else x.detach().reshape(-1, width)
    rows = flat.shape[0]
    if width > 1 and flat.stride(1) != 1:
        flat = flat.detach().contiguous()
    bytes_ = (width + 31) // 32 * 16
    values = flat.new_empty((rows, bytes_), dtype=torch.uint8)
    scales = flat.new_empty(((rows + 127) // 128 * ((width + 255) // 256) * 1024,), dtype=torch.uint8)
    _lib.call_on(device, "p2b_mx4_quantise", flat.data_ptr(), flat.stride(0), rows, width, kind, values.data_ptr(), scales.data_ptr())
    return _made(values, scales, tuple(shape))


def linear(x: torch.Tensor | Mx4, weight: Mx4, bias: torch.Tensor | None = None, *, activation: str = "none",
           dtype: torch.dtype | None = None, quantised: bool = False) -> torch.Tensor | Mx4:
    """act(q(x) weight^T + bias) [..., columns]: x [..., width] as a tensor (quantised here) or quantised already, weight a quantised
    [columns, width] matrix, bias [columns] in the type of the result, which is x's (bf16 where x is fp32 or quantised)
    unless `dtype` says bf16 or fp16.  `activation`: "none", "gelu" (with erf) or "silu".  Sums are fp32, one rounding at the end.
    `quantised`: the result as `quantise` would make of it, without its way through memory, for the next such layer."""
    if not isinstance(weight, Mx4) or len(weight.shape) != 2:
        raise ValueError("the weight is a quantised matrix [columns, width]")
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"unknown activation {activation!r}: one of {', '.join(ACTIVATIONS)}")
    tensor = isinstance(x, torch.Tensor)
    if torch.is_grad_enabled() and (tensor and x.requires_grad or bias is not None and bias.requires_grad):
        raise RuntimeError("mx4.linear has no gradient: call it under torch.no_grad(), or train the layer that was quantised")
    _lib.refuse_tangents("mx4.linear", x if tensor else None, bias)
    if dtype is None:
        dtype = torch.float16 if tensor and x.dtype == torch.float16 else torch.bfloat16
    elif dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("the result is bf16 or fp16")
    columns, width = weight.shape
    device = weight.values.get_device()
    if device < 0:
        _lib.require_cuda(weight.values, "mx4.linear")
    if len(x.shape) < 1 or x.shape[-1] != width or (x if tensor else x.values).get_device() != device:
        raise ValueError("x must have the weight's width and device")
    if columns == 0:
        raise ValueError("the weight has no row")
    _check_layout(weight)
    if not tensor:
        _check_layout(x)
    if bias is not None:
        if bias.dim() != 1 or bias.shape[0] != columns or bias.dtype != dtype or bias.get_device() != device:
            raise ValueError("the bias has one entry for each output, in the type of the result and on its device")
        bias = bias.contiguous()
    if tensor and not quantised and x.dtype in _TYPES:
        flat = x if x.dim() == 2 else x.reshape(-1, width)
        if width > 1 and flat.stride(1) != 1:
            flat = flat.contiguous()
        rows = flat.shape[0]
        out, scratch, size = x.new_empty((rows, columns), dtype=dtype), None, 0
        if rows > FEW_ROWS:
            size = (rows + 127) // 128 * ((width + 255) // 256) * 1024 + rows * ((width + 31) // 32 * 16)
            scratch = x.new_empty((size,), dtype=torch.uint8)
        _lib.call_on(device, "p2b_mx4_linear_rows", flat.data_ptr(), flat.stride(0), _TYPES[x.dtype], rows, weight.values.data_ptr(),
                     weight.scales.data_ptr(), columns, width, None if bias is None else bias.data_ptr(), _TYPES[dtype], act, out.data_ptr(), columns,
                     None if scratch is None else scratch.data_ptr(), size)
        return out if x.dim() == 2 else out.view(*x.shape[:-1], columns)
    a = quantise(x) if tensor else x
    if quantised:
        rows, v = a.values.shape[0], a.values
        values = v.new_empty((rows, (columns + 31) // 32 * 16))
        scales = v.new_empty(((rows + 127) // 128 * ((columns + 255) // 256) * 1024,))
        _lib.call_on(device, "p2b_mx4_linear_mx4", v.data_ptr(), a.scales.data_ptr(), rows, weight.values.data_ptr(), weight.scales.data_ptr(), columns,
                     width, None if bias is None else bias.data_ptr(), _TYPES[dtype], act, values.data_ptr(), scales.data_ptr())
        return _made(values, scales, (*a.shape[:-1], columns))
    out = a.values.new_empty((*a.shape[:-1], columns), dtype=dtype)
    _lib.call_on(device, "p2b_mx4_linear", a.values.data_ptr(), a.scales.data_ptr(), a.values.shape[0], weight.values.data_ptr(),
                 weight.scales.data_ptr(), columns, width, None if bias is None else bias.data_ptr(), _TYPES[dtype], act, out.data_ptr(), columns)
    return out
