"""The gated hidden layer of a value or policy network, h = act(x Wg^T + bg) * (x Wu^T + bu), on the tensor cores.

`gated_linear` is the layer, with gradients through autograd; `gated_linear_backward` gives the gradients by themselves, for
callers that keep their own tape or capture a training step in a CUDA graph.  Both projections, the activation and the
product are one kernel; the backward pass takes the projections anew, so nothing but the inputs is kept for it.
`leaf_eval.GatedValueMLP` is a value network made of such layers.
"""
from __future__ import annotations

import torch

from . import _lib

ACTIVATIONS = {"gelu": 0, "silu": 1}
_TYPES = {torch.bfloat16: 0, torch.float16: 1}


def gated_linear(x: torch.Tensor, gate_weight: torch.Tensor, up_weight: torch.Tensor, gate_bias: torch.Tensor | None = None,
                 up_bias: torch.Tensor | None = None, *, activation: str = "gelu") -> torch.Tensor:
    """x [..., width], gate_weight and up_weight [hidden, width], biases [hidden] or None, all bf16 or all fp16 on one GPU
    -> act(x Wg^T + bg) * (x Wu^T + bu) [..., hidden].  Sums are fp32 and the result is rounded once.  `activation` is
    "gelu" (with erf) or "silu".  Any strides; rows that start on 16-byte boundaries (and weights likewise) are read in place.
    With gradients wanted the call is refused while a CUDA graph is being captured: use `gated_linear_backward` there."""
    _check(x, gate_weight, up_weight, gate_bias, up_bias, activation)
    wanted = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, gate_weight, up_weight, gate_bias, up_bias))
    if not wanted:
        return _forward(x, gate_weight, up_weight, gate_bias, up_bias, activation)
    _refuse_capture("gated_linear", "gated_linear_backward")
    return _Gated.apply(x, gate_weight, up_weight, gate_bias, up_bias, activation)


def gated_linear_backward(grad_h: torch.Tensor, x: torch.Tensor, gate_weight: torch.Tensor, up_weight: torch.Tensor,
                          gate_bias: torch.Tensor | None = None, up_bias: torch.Tensor | None = None, *, activation: str = "gelu",
                          needs: tuple = (True, True, True, True, True)):
    """Gradients of sum(grad_h * gated_linear(x, ...)) for (x, gate_weight, up_weight, gate_bias, up_bias); None where `needs` says
    so or the bias is None.  The same inputs give the same bits."""
    _check(x, gate_weight, up_weight, gate_bias, up_bias, activation)
    width, hidden = x.shape[-1], gate_weight.shape[0]
    if tuple(grad_h.shape) != (*x.shape[:-1], hidden) or grad_h.dtype != x.dtype or grad_h.device != x.device:
        raise ValueError("the gradient of the hidden layer must have its shape, type and device")
    with torch.no_grad():
        rows_of = x.reshape(-1, width)
        rows = rows_of.shape[0]
        new = lambda wanted, *shape: torch.empty(*shape, dtype=x.dtype, device=x.device) if wanted else None  # noqa: E731
        dx = new(needs[0], rows, width)
        dwg, dwu = new(needs[1], hidden, width), new(needs[2], hidden, width)
        dbg, dbu = new(needs[3] and gate_bias is not None, hidden), new(needs[4] and up_bias is not None, hidden)
        xr, gw, uw = _lib.wide_rows(rows_of), _lib.wide_rows(gate_weight), _lib.wide_rows(up_weight)
        gh = grad_h.reshape(-1, hidden)
        gh = gh if gh.stride(1) == 1 and (rows <= 1 or gh.stride(0) >= hidden) else gh.contiguous()
        gb, ub = _packed(gate_bias), _packed(up_bias)
        p = _lib.ptr
        with _lib.on(x.device):
            size = _lib.lib().p2b_gated_backward_scratch_bytes(rows, hidden)
            scratch = torch.empty(max(size, 16), dtype=torch.uint8, device=x.device)
            _lib.call("p2b_gated_backward", p(gh), gh.stride(0), p(xr), xr.stride(0), p(gw), gw.stride(0), p(uw), uw.stride(0), p(gb), p(ub),
                      rows, width, hidden, _TYPES[x.dtype], ACTIVATIONS[activation], p(dx), width, p(dwg), p(dwu), p(dbg), p(dbu), p(scratch),
                      scratch.numel(), _lib.stream_ptr(x.device))
    return dx if dx is None else dx.view(x.shape), dwg, dwu, dbg, dbu


def _forward(x, gate_weight, up_weight, gate_bias, up_bias, activation):
    width, hidden = x.shape[-1], gate_weight.shape[0]
    with torch.no_grad():
        h = torch.empty(*x.shape[:-1], hidden, dtype=x.dtype, device=x.device)
        xr, gw, uw = x.reshape(-1, width), gate_weight, up_weight
        rows = xr.shape[0]
        whole = _lib.wide_rows if rows > _lib.lib().p2b_gated_few_rows() else _lib.plain_rows
        xr, gw, uw = whole(xr), whole(gw), whole(uw)
        gb, ub = _packed(gate_bias), _packed(up_bias)
        p = _lib.ptr
        with _lib.on(x.device):
            _lib.call("p2b_gated_forward", p(xr), xr.stride(0), p(gw), gw.stride(0), p(uw), uw.stride(0), p(gb), p(ub), rows, width, hidden,
                      _TYPES[x.dtype], ACTIVATIONS[activation], p(h), hidden, _lib.stream_ptr(x.device))
    return h


class _Gated(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate_weight, up_weight, gate_bias, up_bias, activation):
        ctx.save_for_backward(x, gate_weight, up_weight, gate_bias, up_bias)
        ctx.activation = activation
        return _forward(x, gate_weight, up_weight, gate_bias, up_bias, activation)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_h):
        _refuse_capture("the backward pass of gated_linear", "gated_linear_backward")
        return (*gated_linear_backward(grad_h, *ctx.saved_tensors, activation=ctx.activation, needs=ctx.needs_input_grad[:5]), None)


def _refuse_capture(what: str, instead: str) -> None:
    """Autograd joins a leaf's gradient on the stream that the leaf was first used on; with an eager graph of the same leaves alive that
    stream lies outside the capture, and the process ends in the engine's thread."""
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{what} cannot be captured into a CUDA graph through autograd; call {instead}, which can.")


def _packed(bias):
    return None if bias is None else bias.contiguous()


def _check(x, gate_weight, up_weight, gate_bias, up_bias, activation) -> None:
    _lib.require_cuda(x, "gated_linear")
    if activation not in ACTIVATIONS:
        raise ValueError(f"unknown activation {activation!r}: one of {', '.join(ACTIVATIONS)}")
    if x.dtype not in _TYPES:
        raise ValueError("gated_linear takes bf16 or fp16 tensors")
    if x.dim() < 1 or gate_weight.dim() != 2 or gate_weight.shape != up_weight.shape or gate_weight.shape[1] != x.shape[-1]:
        raise ValueError("x [..., width] and two weights [hidden, width] are wanted")
    if gate_weight.numel() == 0:
        raise ValueError("width and hidden must not be zero")
    for t in (gate_weight, up_weight, gate_bias, up_bias):
        if t is not None and (t.dtype != x.dtype or t.device != x.device):
            raise ValueError("x, weights and biases must have one type and lie on one device")
    for b in (gate_bias, up_bias):
        if b is not None and tuple(b.shape) != (gate_weight.shape[0],):
            raise ValueError("a bias has one entry for each hidden unit")
