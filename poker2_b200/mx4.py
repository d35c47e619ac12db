"""Microscaled 4-bit values: 32 neighbouring values of a row share a power-of-two scale.  `quantise` writes them, `dequantise`
reads them back, `linear` multiplies two such matrices on the block-scaled matrix instructions.

The scale of a block is the smallest power of two that brings its largest magnitude to 6 or below, so nothing is cut off; a
value is then the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with its sign, ties to the even code.  A block that holds an infinity
or a NaN reads back as NaN.  For serving: there are no gradients.  `leaf_eval.Mx4ValueMLP` is a value network in this form.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _lib

ACTIVATIONS = {"gelu": 0, "silu": 1, "none": 2}
_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


@dataclass(frozen=True)
class Mx4:
    """A matrix in 4 bits: `values` [rows, ceil(width/32)*16] bytes, two values a byte; `scales`, the blocks' exponents in the
    order in which the matrix instructions read them (include/poker2_b200.h); `shape` of what was quantised."""

    values: torch.Tensor
    scales: torch.Tensor
    shape: tuple

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
        if dtype not in _TYPES:
            raise ValueError("values are read back in bf16, fp16 or fp32")
        out = torch.empty(self.shape, dtype=dtype, device=self.device)
        with _lib.on(self.device):
            _lib.call("p2b_mx4_dequantise", _lib.ptr(self.values), _lib.ptr(self.scales), self.rows, self.width, _TYPES[dtype], _lib.ptr(out),
                      self.width, _lib.stream_ptr(self.device))
        return out


def quantise(x: torch.Tensor) -> Mx4:
    """x [..., width], bf16, fp16 or fp32, any strides; the blocks lie along the last dimension, the last one may be short."""
    _lib.require_cuda(x, "quantise")
    if x.dtype not in _TYPES:
        raise ValueError("quantise takes bf16, fp16 or fp32 tensors")
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError("quantise wants rows of at least one value")
    width = x.shape[-1]
    flat = x.detach().reshape(-1, width)
    flat = flat if flat.stride(1) == 1 else flat.contiguous()
    rows = flat.shape[0]
    values = torch.empty(rows, (width + 31) // 32 * 16, dtype=torch.uint8, device=x.device)
    scales = torch.empty((rows + 127) // 128 * ((width + 255) // 256) * 1024, dtype=torch.uint8, device=x.device)
    with _lib.on(x.device):
        _lib.call("p2b_mx4_quantise", _lib.ptr(flat), flat.stride(0), rows, width, _TYPES[x.dtype], _lib.ptr(values), _lib.ptr(scales),
                  _lib.stream_ptr(x.device))
    return Mx4(values, scales, tuple(x.shape))


def linear(x: torch.Tensor | Mx4, weight: Mx4, bias: torch.Tensor | None = None, *, activation: str = "none",
           dtype: torch.dtype | None = None) -> torch.Tensor:
    """act(q(x) weight^T + bias) [..., columns]: x [..., width] as a tensor (quantised here) or quantised already, weight a quantised
    [columns, width] matrix, bias [columns] in the type of the result, which is x's (bf16 where x is fp32 or quantised)
    unless `dtype` says bf16 or fp16.  `activation`: "none", "gelu" (with erf) or "silu".  Sums are fp32, one rounding at the end."""
    if not isinstance(weight, Mx4) or len(weight.shape) != 2:
        raise ValueError("the weight is a quantised matrix [columns, width]")
    if activation not in ACTIVATIONS:
        raise ValueError(f"unknown activation {activation!r}: one of {', '.join(ACTIVATIONS)}")
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in (x, bias)):
        raise RuntimeError("mx4.linear has no gradient: call it under torch.no_grad(), or train the layer that was quantised")
    if dtype is None:
        dtype = x.dtype if isinstance(x, torch.Tensor) and x.dtype == torch.float16 else torch.bfloat16
    if dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("the result is bf16 or fp16")
    if len(x.shape) < 1 or x.shape[-1] != weight.width or x.device != weight.device:
        raise ValueError("x must have the weight's width and device")
    columns = weight.shape[0]
    if columns == 0:
        raise ValueError("the weight has no row")
    if bias is not None and (tuple(bias.shape) != (columns,) or bias.dtype != dtype or bias.device != weight.device):
        raise ValueError("the bias has one entry for each output, in the type of the result and on its device")
    a = x if isinstance(x, Mx4) else quantise(x)
    out = torch.empty(*a.shape[:-1], columns, dtype=dtype, device=weight.device)
    bias = None if bias is None else bias.contiguous()
    p = _lib.ptr
    with _lib.on(weight.device):
        _lib.call("p2b_mx4_linear", p(a.values), p(a.scales), a.rows, p(weight.values), p(weight.scales), columns, weight.width, p(bias),
                  _TYPES[dtype], ACTIVATIONS[activation], p(out), columns, _lib.stream_ptr(weight.device))
    return out
