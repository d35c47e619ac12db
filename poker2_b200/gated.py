"""The gated hidden layer of a value or policy network, h = act(x Wg^T + bg) * (x Wu^T + bu), on the tensor cores.

`gated_linear` is the layer, with gradients through autograd; `gated_linear_backward` gives the gradients by themselves, for
callers that keep their own tape or capture a training step in a CUDA graph.  Both projections, the activation and the
product are one kernel; the backward pass takes the projections anew or, in large layers where that takes longer, finds gate and up
as autograd's forward pass kept them: the same bits either way.  What is kept takes 8 bytes a hidden value (of `hidden` rounded up to 128,
so up to 16; narrower layers keep nothing), four times h, from forward to backward; `keep=False`, or no memory for it, takes them anew.
`leaf_eval.GatedValueMLP` is a value network made of such layers.
"""
from __future__ import annotations

import torch

from . import _lib

ACTIVATIONS = {"gelu": 0, "silu": 1}
_TYPES = {torch.bfloat16: 0, torch.float16: 1}
KEPT_PRODUCTS = 1 << 33  # rows * width * hidden from which on the forward pass may keep gate and up (p2b_gated_kept_bytes)
FEW_ROWS = 4  # up to so many rows the forward pass reads operands of any alignment (p2b_gated_few_rows)


def gated_linear(x: torch.Tensor, gate_weight: torch.Tensor, up_weight: torch.Tensor, gate_bias: torch.Tensor | None = None,
                 up_bias: torch.Tensor | None = None, *, activation: str = "gelu", keep: bool = True) -> torch.Tensor:
    """x [..., width], gate_weight and up_weight [hidden, width], biases [hidden] or None, all bf16 or all fp16 on one GPU
    -> act(x Wg^T + bg) * (x Wu^T + bu) [..., hidden].  Sums are fp32 and the result is rounded once.  `activation` is
    "gelu" (with erf) or "silu".  Any strides; rows that start on 16-byte boundaries (and weights likewise) are read in place.
    `keep`: large training steps may hold gate and up for the backward pass, 8 to 16 bytes a hidden value.
    With gradients wanted the call is refused while a CUDA graph is being captured: use `gated_linear_backward` there."""
    act = _check(x, gate_weight, up_weight, gate_bias, up_bias, activation)
    _lib.refuse_tangents("gated_linear", x, gate_weight, up_weight, gate_bias, up_bias)
    if torch.is_grad_enabled() and (x.requires_grad or gate_weight.requires_grad or up_weight.requires_grad
                                    or gate_bias is not None and gate_bias.requires_grad or up_bias is not None and up_bias.requires_grad):
        _refuse_capture("gated_linear")
        return _Gated.apply(x, gate_weight, up_weight, gate_bias, up_bias, act, keep)
    return _forward(x, gate_weight, up_weight, gate_bias, up_bias, act)


def gated_linear_backward(grad_h: torch.Tensor, x: torch.Tensor, gate_weight: torch.Tensor, up_weight: torch.Tensor,
                          gate_bias: torch.Tensor | None = None, up_bias: torch.Tensor | None = None, *, activation: str = "gelu",
                          needs: tuple = (True, True, True, True, True)):
    """Gradients of sum(grad_h * gated_linear(x, ...)) for (x, gate_weight, up_weight, gate_bias, up_bias); None where `needs` says
    so or the bias is None.  The same inputs give the same bits.  Like the layer's own intermediate values in fp16, those of the
    gradients (grad_h times gate or up) end at 65504 and lose bits below 6e-5: scale an fp16 loss as for any other layer."""
    act = _check(x, gate_weight, up_weight, gate_bias, up_bias, activation)
    if grad_h.shape != (*x.shape[:-1], gate_weight.shape[0]) or grad_h.dtype != x.dtype or grad_h.get_device() != x.get_device():
        raise ValueError("the gradient of the hidden layer must have its shape, type and device")
    _lib.refuse_tangents("gated_linear_backward", grad_h, x, gate_weight, up_weight, gate_bias, up_bias)
    with torch.no_grad():
        return _backward(grad_h, x, gate_weight, up_weight, gate_bias, up_bias, None, act, needs)


def _forward(x, gate_weight, up_weight, gate_bias, up_bias, act, kept=None):
    shape, hidden = x.shape, gate_weight.shape[0]
    width = shape[-1]
    xr = x if len(shape) == 2 else x.reshape(-1, width)
    rows = xr.shape[0]
    h = x.new_empty((rows, hidden))
    xr, gw, uw = _lib.plain_rows(xr), _lib.plain_rows(gate_weight), _lib.plain_rows(up_weight)
    size = 0 if rows <= FEW_ROWS else _align_bytes(xr, gw, uw)
    scratch = x.new_empty((size // 2,)) if size else None
    gb = None if gate_bias is None else gate_bias.contiguous()
    ub = None if up_bias is None else up_bias.contiguous()
    _lib.call_on(x.get_device(), "p2b_gated_forward", xr.data_ptr(), xr.stride(0), gw.data_ptr(), gw.stride(0), uw.data_ptr(), uw.stride(0),
                 None if gb is None else gb.data_ptr(), None if ub is None else ub.data_ptr(), rows, width, hidden, _TYPES[x.dtype], act,
                 h.data_ptr(), hidden, None if kept is None else kept.data_ptr(), None if scratch is None else scratch.data_ptr(), size)
    return h if len(shape) == 2 else h.view(*shape[:-1], hidden)


def _backward(grad_h, x, gate_weight, up_weight, gate_bias, up_bias, kept, act, needs):
    shape, hidden, p = x.shape, gate_weight.shape[0], _lib.ptr
    width = shape[-1]
    xr, gh = (x, grad_h) if len(shape) == 2 else (x.reshape(-1, width), grad_h.reshape(-1, hidden))
    rows = xr.shape[0]
    dx = _packed_like(xr) if needs[0] else None
    dwg = _packed_like(gate_weight) if needs[1] else None
    dwu = _packed_like(up_weight) if needs[2] else None
    dbg = _packed_like(gate_bias) if needs[3] and gate_bias is not None else None
    dbu = _packed_like(up_bias) if needs[4] and up_bias is not None else None
    xr, gw, uw, gh = _lib.plain_rows(xr), _lib.plain_rows(gate_weight), _lib.plain_rows(up_weight), _lib.plain_rows(gh)
    gb = None if gate_bias is None else gate_bias.contiguous()
    ub = None if up_bias is None else up_bias.contiguous()
    size = _lib.lib().p2b_gated_backward_scratch_bytes(rows, width, hidden) + _align_bytes(xr, gw, uw)
    scratch = x.new_empty((max(size, 16) // 2,))
    _lib.call_on(x.get_device(), "p2b_gated_backward", gh.data_ptr(), gh.stride(0), xr.data_ptr(), xr.stride(0), gw.data_ptr(), gw.stride(0),
                 uw.data_ptr(), uw.stride(0), p(gb), p(ub), rows, width, hidden, _TYPES[x.dtype], act, p(dx), width, p(dwg), p(dwu), p(dbg),
                 p(dbu), p(kept), scratch.data_ptr(), size)
    return dx if dx is None or len(shape) == 2 else dx.view(shape), dwg, dwu, dbg, dbu


def _packed_like(t: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)  # (the first takes 1.3 us, the other 1.8)


def _align_bytes(*matrices) -> int:
    """Bytes for copies whose rows start on 16-byte boundaries; 0 where all do already."""
    for t in matrices:
        if t.data_ptr() % 16 or t.stride(0) % 8 and t.shape[0] > 1:
            x, weight, _ = matrices
            return _lib.lib().p2b_gated_align_bytes(x.shape[0], x.shape[1], weight.shape[0])
    return 0


def _kept_area(x: torch.Tensor, weight: torch.Tensor) -> torch.Tensor | None:
    """Where the forward pass keeps gate and up; None where it does not, where most of it would be what `hidden` is rounded up by, and
    where there is no room."""
    hidden, width = weight.shape
    rows = x.numel() // width
    size = _lib.lib().p2b_gated_kept_bytes(rows, width, hidden)
    if not 0 < size <= 16 * rows * hidden:
        return None
    try:
        return x.new_empty((size // 2,))
    except torch.cuda.OutOfMemoryError:
        return None


class _Gated(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate_weight, up_weight, gate_bias, up_bias, act, keep):
        kept = _kept_area(x, gate_weight) if keep and x.numel() * gate_weight.shape[0] >= KEPT_PRODUCTS else None
        ctx.save_for_backward(x, gate_weight, up_weight, gate_bias, up_bias, kept)
        ctx.act = act
        return _forward(x, gate_weight, up_weight, gate_bias, up_bias, act, kept)

    @staticmethod
    def backward(ctx, grad_h):
        _refuse_capture("the backward pass of gated_linear")
        if torch.is_grad_enabled():
            raise RuntimeError("gated_linear has no second derivatives (create_graph=True)")
        _lib.refuse_tangents("the backward pass of gated_linear", grad_h)
        return (*_backward(grad_h, *ctx.saved_tensors, ctx.act, ctx.needs_input_grad), None, None)


def _refuse_capture(what: str) -> None:
    """Autograd joins a leaf's gradient on the stream that the leaf was first used on; with an eager graph of the same leaves alive that
    stream lies outside the capture, and the process ends in the engine's thread."""
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{what} cannot be captured into a CUDA graph through autograd; call gated_linear_backward, which can.")


def _check(x, gate_weight, up_weight, gate_bias, up_bias, activation) -> int:
    """The activation's number; ValueError where the arguments do not fit (asked once a call: the smallest calls last as long as the
    host takes to make them)."""
    device, dtype, shape = x.get_device(), x.dtype, gate_weight.shape
    if device < 0:
        _lib.require_cuda(x, "gated_linear")
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"unknown activation {activation!r}: one of {', '.join(ACTIVATIONS)}")
    if dtype not in _TYPES:
        raise ValueError("gated_linear takes bf16 or fp16 tensors")
    if len(shape) != 2 or up_weight.shape != shape or x.dim() < 1 or x.shape[-1] != shape[1]:
        raise ValueError("x [..., width] and two weights [hidden, width] are wanted")
    if shape[0] == 0 or shape[1] == 0:
        raise ValueError("width and hidden must not be zero")
    if gate_weight.dtype != dtype or up_weight.dtype != dtype or gate_weight.get_device() != device or up_weight.get_device() != device:
        raise ValueError("x, weights and biases must have one type and lie on one device")
    for b in (gate_bias, up_bias):
        if b is not None:
            if b.dtype != dtype or b.get_device() != device:
                raise ValueError("x, weights and biases must have one type and lie on one device")
            if b.dim() != 1 or b.shape[0] != shape[0]:
                raise ValueError("a bias has one entry for each hidden unit")
    return act
