"""The loss that trains a policy head on what a search returned, with its gradient: a clipped policy term and the KL divergence to a
target policy, over all 1326 hands (or any number) of a batch of states and their legal actions.

Per state and hand, with p = softmax(logits) over the legal actions, q the old policy and t the target,

    l = -sum_a min(p_a A_a, clip(p_a, (1-clip) q_a, (1+clip) q_a) A_a) + kl * sum_a t_a (log t_a - log p_a)

is the clipped surrogate of the ratio p/q summed over the actions (a search gives every action's advantage, none is sampled)
plus the divergence from the target.  The loss is the mean over the hands by their weights.  `RebelBatchLike.policy_loss` calls it
on a minibatch of the replay ring.
"""
from __future__ import annotations

import torch

from . import _lib

NUM_HANDS = _lib.NUM_HANDS
MAX_ACTIONS = 16
_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def clipped_policy_loss(logits: torch.Tensor, old_policy: torch.Tensor | None, advantages: torch.Tensor | None, target: torch.Tensor,
                        legal: torch.Tensor, weights: torch.Tensor | None = None, *, clip: float = 0.2, kl: float = 1.0) -> torch.Tensor:
    """logits [states, hands, actions] bf16, fp16 or fp32; old_policy and advantages (both None: the KL term alone) and target of that
    shape in fp32; legal [states, actions] bool; weights [states, hands] fp32, none negative (None: 1) -> the loss, an fp32 scalar
    that differentiates to the logits.

    Illegal actions, hands of weight 0, states without a legal action and hands whose legal logits are all -inf add nothing
    and get a zero gradient, whatever their entries hold; a NaN or +inf among the legal logits of a hand that counts makes the loss and the
    hand's gradient NaN, a NaN among the weights (of states with a legal action) the loss and the gradients of all hands.

    With gradients wanted the gradient is computed in the same pass and the call is refused while a CUDA graph is being captured: use
    `clipped_policy_loss_and_grad` there.  bf16 and fp32 logits: it is rounded to their type, and once more with the factor that the
    backward pass brings.  fp16 logits: it stays in fp32 until that factor is known, so that a gradient scaler's reaches entries of the
    size 1 / (states * hands), which fp16 has no room for (factors up to 2, which raise nothing into its range, multiply the rounded
    gradient)."""
    _check(logits, old_policy, advantages, target, legal, weights, clip, kl)
    if not (torch.is_grad_enabled() and logits.requires_grad):
        return _run(logits, old_policy, advantages, target, legal, weights, clip, kl, False)[0]
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("clipped_policy_loss cannot be captured into a CUDA graph through autograd; call clipped_policy_loss_and_grad, which can.")
    return _Loss.apply(logits, old_policy, advantages, target, legal, weights, clip, kl)


def clipped_policy_loss_and_grad(logits: torch.Tensor, old_policy: torch.Tensor | None, advantages: torch.Tensor | None, target: torch.Tensor,
                                 legal: torch.Tensor, weights: torch.Tensor | None = None, *, clip: float = 0.2, kl: float = 1.0,
                                 scale: float | torch.Tensor = 1.0):
    """(loss, its gradient to the logits in their type) of `clipped_policy_loss`, in one pass and without autograd: hand the gradient
    to `logits.backward(grad)`.  `scale`, a number or an fp32 tensor of one element on the logits' device, multiplies the gradient (the
    loss stays as it is) before it is rounded: what a gradient scaler brings, without which entries of the size 1 / (states * hands)
    are lost in fp16."""
    _check(logits, old_policy, advantages, target, legal, weights, clip, kl)
    at = None
    if type(scale) is not float and isinstance(scale, torch.Tensor):
        if scale.numel() != 1 or scale.dtype != torch.float32 or scale.get_device() != logits.get_device():
            raise ValueError("the scale is a number, or an fp32 tensor of one element on the logits' device")
        scale, at = 1.0, scale.data_ptr()
    elif not abs(scale) <= 3.4028234e38:
        raise ValueError("the scale is finite")
    return _run(logits, old_policy, advantages, target, legal, weights, clip, kl, True, scale, at)


def hand_weights(beliefs: torch.Tensor, to_act: torch.Tensor, board: torch.Tensor) -> torch.Tensor:
    """[n, 1326] fp32: the chance that the player to act holds a hand, times the chance that the other player's range leaves it
    open; 0 for hands with a card on the board.  beliefs [n, 2*1326], to_act [n], board [n, L] with -1 for cards not dealt.  A state
    whose player is neither 0 nor 1, or with a card above 51, has NaN for all its weights."""
    from .fused_cfr import unblocked_mass_triton

    _lib.require_cuda(beliefs, "hand_weights")
    if torch.is_grad_enabled() and beliefs.requires_grad:
        raise RuntimeError("hand_weights has no gradient: detach the beliefs")  # (half of the product's would be lost in the kernel)
    _lib.refuse_tangents("hand_weights", beliefs)
    n = beliefs.shape[0]
    if tuple(beliefs.shape) != (n, 2 * NUM_HANDS) or tuple(to_act.shape) != (n,) or board.dim() != 2 or board.shape[0] != n:
        raise ValueError("beliefs [n, 2652], to_act [n] and board [n, L] are wanted")
    device = beliefs.device
    ranges = beliefs.to(torch.float32).view(n, 2, NUM_HANDS)
    player, rows = to_act.to(device=device, dtype=torch.int64), torch.arange(n, device=device)
    actor = player.clamp(0, 1)  # (an index outside would end the process's use of the device)
    held = ranges[rows, actor] * unblocked_mass_triton(ranges[rows, 1 - actor].contiguous()).clamp(min=0.0)
    c1, c2 = torch.triu_indices(52, 52, 1, device=device)
    board = board.to(device=device, dtype=torch.int64)
    dealt = torch.zeros(n, 53, dtype=torch.bool, device=device).scatter_(1, torch.where(board >= 0, board.clamp(max=52), 52), True)
    undefined = ((player != actor) | (board > 51).any(dim=1))[:, None]
    dealt |= undefined
    return torch.where(dealt[:, c1] | dealt[:, c2], torch.where(undefined, float("nan"), 0.0), held)


class _Loss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, old_policy, advantages, target, legal, weights, clip, kl):
        ctx.wide = logits.dtype is torch.float16
        loss, grad = _run(logits, old_policy, advantages, target, legal, weights, clip, kl, True, wide=ctx.wide)
        ctx.save_for_backward(grad)
        return loss

    @staticmethod
    def backward(ctx, factor):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the backward pass of clipped_policy_loss cannot be captured into a CUDA graph; call clipped_policy_loss_and_grad, which can.")
        if torch.is_grad_enabled():
            raise RuntimeError("clipped_policy_loss has no second derivatives (create_graph=True)")
        _lib.refuse_tangents("the backward pass of clipped_policy_loss", factor)
        grad, = ctx.saved_tensors
        if ctx.wide:
            out = torch.empty_like(grad, dtype=torch.float16)
            _lib.call_on(grad.get_device(), "p2b_policy_loss_scale_fp32", grad.data_ptr(), factor.data_ptr(), grad.numel(), out.data_ptr())
        else:
            out = torch.empty_like(grad)
            _lib.call_on(grad.get_device(), "p2b_policy_loss_scale", grad.data_ptr(), factor.data_ptr(), grad.numel(), _TYPES[grad.dtype], out.data_ptr())
        return out, None, None, None, None, None, None, None


def _packed(t):
    return t if t is None or t.is_contiguous() else t.detach().contiguous()


def _run(logits, old_policy, advantages, target, legal, weights, clip, kl, with_grad, scale=1.0, scale_at=None, wide=False):
    """(loss, the gradient times scale and *scale_at, of the logits' type or fp32 where `wide`; None where it is not wanted)."""
    states, hands, actions = logits.shape
    logits, target, legal = _packed(logits), _packed(target), _packed(legal)
    old_policy, advantages, weights = _packed(old_policy), _packed(advantages), _packed(weights)
    loss = target.new_empty(())
    grad = None if not with_grad else target.new_empty((states, hands, actions)) if wide else logits.new_empty((states, hands, actions))
    size = _lib.lib().p2b_policy_loss_scratch_bytes(states, hands)
    scratch = target.new_empty((size // 4,)) if size else None
    kind = _TYPES[logits.dtype]
    scaled = (2 if wide else kind, scale, scale_at) if wide or scale != 1.0 or scale_at else ()
    _lib.call_on(logits.get_device(), "p2b_policy_loss_scaled" if scaled else "p2b_policy_loss", logits.data_ptr(), None if old_policy is None else old_policy.data_ptr(),
                 None if advantages is None else advantages.data_ptr(), target.data_ptr(), legal.data_ptr(),
                 None if weights is None else weights.data_ptr(), states, hands, actions, kind, clip, kl, loss.data_ptr(),
                 None if grad is None else grad.data_ptr(), *scaled, None if scratch is None else scratch.data_ptr(), size)
    return loss, grad


def _check(logits, old_policy, advantages, target, legal, weights, clip, kl) -> None:
    device, shape, f32 = logits.get_device(), logits.shape, torch.float32
    if device < 0:
        _lib.require_cuda(logits, "clipped_policy_loss")
    if logits.dtype not in _TYPES or len(shape) != 3 or shape[1] < 1 or not 1 <= shape[2] <= MAX_ACTIONS:
        raise ValueError(f"logits [states, hands, actions] in bf16, fp16 or fp32 with 1 to {MAX_ACTIONS} actions are wanted")
    if (old_policy is None) != (advantages is None):
        raise ValueError("the old policy and the advantages come together")
    for t in (target, old_policy, advantages):
        if t is not None and (t.shape != shape or t.dtype != f32 or t.get_device() != device):
            raise ValueError("old policy, advantages and target have the logits' shape and device, in fp32")
    if legal.shape != (shape[0], shape[2]) or legal.dtype != torch.bool or legal.get_device() != device:
        raise ValueError("legal [states, actions] bool on the logits' device is wanted")
    if weights is not None and (weights.shape != shape[:2] or weights.dtype != f32 or weights.get_device() != device):
        raise ValueError("weights [states, hands] fp32 on the logits' device are wanted")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (old_policy, advantages, target, weights)):
        raise RuntimeError("the loss differentiates to the logits alone: detach the policies, advantages and weights")
    _lib.refuse_tangents("the policy loss", logits, old_policy, advantages, target, weights)
    if not 0.0 <= clip < 1.0 or not 0.0 <= kl < float("inf"):
        raise ValueError("clip lies in [0, 1), kl is not negative")
