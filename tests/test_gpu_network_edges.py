"""Edges of the network operators: values that are not finite, types at the end of their range, networks that are saved and moved."""
import pytest
import torch

import network_refs as refs
from poker2_b200 import _lib, gated, leaf_eval, mx4, policy_loss as pl

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("activation", ["none", "gelu"])
# one tile and a last one of up to 64 columns behind it, an odd piece behind the last tile, blocks that end short; pairs of tiles
@pytest.mark.parametrize("rows,width,columns", [(40, 96, 160), (130, 96, 192), (300, 64, 300), (129, 300, 257), (200, 96, 1), (33, 64, 128), (60, 64, 417), (300, 64, 97),
                                                (5000, 64, 700), (2400, 96, 1537), (4000, 64, 1409), (3000, 64, 1300)])
def test_rows_that_are_not_finite_stay_quantised(cuda_device, rows, width, columns, activation, dtype):
    """To the bit what quantising the result gives: behind the last column values of 0 and scales of 0, whatever the row holds."""
    g = torch.Generator(device=cuda_device).manual_seed(rows + columns)
    x = torch.randn(rows, width, device=cuda_device, generator=g)
    x[0, 3], x[7, width - 1], x[rows - 1, 40], x[31] = float("nan"), float("inf"), float("-inf"), float("nan")
    w = mx4.quantise(torch.randn(columns, width, device=cuda_device, generator=g) / width ** 0.5)
    bias = torch.randn(columns, device=cuda_device, generator=g).to(dtype)
    a = mx4.quantise(x)
    y = mx4.linear(a, w, bias, activation=activation, dtype=dtype)
    assert torch.isnan(y[[0, 7, 31, rows - 1]]).all() and torch.isfinite(y[1:7]).all()
    want = mx4.quantise(y)
    torch.full((rows * (columns + 300) * 2,), 255, dtype=torch.uint8, device=cuda_device)
    for _ in range(3):
        got = mx4.linear(a, w, bias, activation=activation, dtype=dtype, quantised=True)
        assert torch.equal(got.values, want.values) and torch.equal(got.scales, want.scales)
    again = mx4.linear(got, mx4.quantise(torch.ones(3, columns, device=cuda_device)))
    assert torch.isnan(again[[0, 7, 31, rows - 1]]).all() and torch.isfinite(again[1:7]).all()


def _loss_batch(states, hands, actions, dtype, device, seed=0):
    g = torch.Generator(device=device).manual_seed(seed + states + hands + actions)
    new = lambda *s: torch.randn(*s, device=device, generator=g)  # noqa: E731
    logits = new(states, hands, actions).to(dtype)
    legal = torch.rand(states, actions, device=device, generator=g) < 0.8
    legal[:, min(1, actions - 1)] = True
    old = torch.softmax(logits.float() + 0.3 * new(states, hands, actions), -1)
    target = (new(states, hands, actions) + 0.3).clamp(min=0.0)
    target = target / target.sum(-1, keepdim=True).clamp(min=1e-6)
    return logits, old, 0.1 * new(states, hands, actions), target, legal, torch.rand(states, hands, device=device, generator=g)


@pytest.mark.parametrize("factor", [65536.0, 1000.0, 3.0])
@pytest.mark.parametrize("states,hands,actions", [(4096, 1326, 5), (513, 1326, 8), (2, 255, 3), (77, 300, 4)])
def test_a_loss_scale_reaches_gradients_that_fp16_has_no_room_for(cuda_device, states, hands, actions, factor):
    """The factor of a gradient scaler times the 64-bit gradient, rounded once: entries of the size 1/(states*hands) survive in fp16."""
    batch = _loss_batch(states, hands, actions, torch.float16, cuda_device)
    _, _, grad, bound = refs.policy_loss(*batch, 0.2, 0.5, torch.float32)
    leaf = batch[0].clone().requires_grad_(True)
    got, = torch.autograd.grad(factor * pl.clipped_policy_loss(leaf, *batch[1:], clip=0.2, kl=0.5), leaf)
    # the fp32 gradient (its bound holds a rounding to fp32), the product's own step, the rounding to fp16
    value, err = factor * grad, factor * (bound + grad.abs() * 2.0 ** -24)
    refs.assert_within(got, value, err + refs.rounded(value.abs() + err, torch.float16))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("states,hands,actions", [(1, 1326, 5), (700, 1326, 5), (33, 256, 16), (3, 77, 3), (520, 511, 8), (2, 1, 1)])
def test_a_scale_is_taken_in_before_the_gradient_is_rounded(cuda_device, states, hands, actions, dtype):
    """The explicit form with a scale, on the host or on the device, in a captured graph too; without the policy term as well."""
    batch = _loss_batch(states, hands, actions, dtype, cuda_device, seed=5)
    plain = pl.clipped_policy_loss_and_grad(*batch)
    assert all(torch.equal(a, b) for a, b in zip(plain, pl.clipped_policy_loss_and_grad(*batch, scale=1.0)))
    for scale in (4096.0, 300.0, -0.7):
        for args in (batch, (batch[0], None, None, *batch[3:])):
            _, _, grad, bound = refs.policy_loss(*args, 0.2, 1.0, torch.float32)
            loss, got = pl.clipped_policy_loss_and_grad(*args, scale=scale)
            assert torch.equal(loss, pl.clipped_policy_loss(*args)) and got.dtype == dtype
            value, err = scale * grad, abs(scale) * (bound + grad.abs() * 2.0 ** -23)  # (two products in fp32)
            refs.assert_within(got, value, err + refs.rounded(value.abs() + err, dtype))
        held = torch.tensor([[scale]], device=cuda_device)
        assert torch.equal(pl.clipped_policy_loss_and_grad(*args, scale=held)[1], got)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            _, later = pl.clipped_policy_loss_and_grad(*args, scale=held)
        held.mul_(2.0)
        graph.replay()
        assert torch.equal(later, pl.clipped_policy_loss_and_grad(*args, scale=2.0 * scale)[1])
        # arrays off 16-byte boundaries take the other way into shared memory
        shifted = [t if t is None else torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape).copy_(t) for t in args]
        assert torch.equal(pl.clipped_policy_loss_and_grad(*shifted, scale=scale)[1], got)


def test_small_factors_multiply_the_rounded_fp16_gradient(cuda_device):
    batch = _loss_batch(600, 1326, 4, torch.float16, cuda_device)
    leaf = batch[0].clone().requires_grad_(True)
    loss, (_, _, grad, bound) = pl.clipped_policy_loss(leaf, *batch[1:]), refs.policy_loss(*batch, 0.2, 1.0, torch.float32)
    _, once = pl.clipped_policy_loss_and_grad(*batch)
    for factor in (1.0, 2.0, -2.0, 0.3, 0.0, 2.25, float("inf"), float("nan")):
        got, = torch.autograd.grad(loss, leaf, torch.tensor(factor, device=cuda_device), retain_graph=True)
        if abs(factor) <= 2.0:
            assert torch.equal(got, (once.float() * factor).half())
            value, err = factor * grad, abs(factor) * (bound + grad.abs() * 2.0 ** -24 + refs.rounded(grad.abs() + bound, torch.float16))
        elif factor == 2.25:
            value, err = factor * grad, factor * (bound + grad.abs() * 2.0 ** -24)
        else:
            assert not torch.isfinite(got[grad != 0]).any()
            continue
        refs.assert_within(got, value, err + refs.rounded(value.abs() + err, torch.float16))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("states,hands,actions", [(3, 40, 5), (300, 256, 5), (40, 77, 8), (6, 256, 1)])
def test_undefined_logits_are_not_taken_for_hands_without_actions(cuda_device, states, hands, actions, dtype):
    """NaN (or +inf, whose softmax is undefined) at a legal action of a hand that counts: the loss and that hand's legal gradients are
    NaN, all others what they were; at hands that do not count it is nothing."""
    nan = float("nan")
    logits, old, adv, target, legal, weights = _loss_batch(states, hands, actions, dtype, cuda_device)
    legal[2] = False
    legal[1, -1] = actions == 1  # (an illegal action beside the undefined ones)
    weights[0, 7] = 0.0
    weights[1:, :] += 0.01
    where = torch.zeros(states, hands, dtype=torch.bool, device=cuda_device)
    where[1, 5] = True
    undefined = where[:, :, None] & legal[:, None, :]
    for policies in ((old, adv), (None, None)):
        for kl in (0.0, 0.7):
            rest = (*policies, target, legal, weights)
            loss, grad = pl.clipped_policy_loss_and_grad(logits, *rest, kl=kl)
            for fill in ("all", "one", "one and -inf", "inf"):
                bad = logits.clone()
                if fill == "all":
                    bad[1, 5] = nan
                elif fill == "one":
                    bad[1, 5, 0] = nan
                    legal_target = target.clone()
                    legal_target[1, 5, 0] = 0.0  # (nothing of the KL term hangs on the undefined logit itself)
                    rest = (*policies, legal_target, legal, weights)
                    if not legal[1, 0]:
                        continue
                elif fill == "one and -inf":
                    bad[1, 5] = float("-inf")
                    bad[1, 5, 0] = nan
                    if not legal[1, 0]:
                        continue
                else:
                    bad[1, 5, 0] = float("inf")
                    if not legal[1, 0]:
                        continue
                got_loss, got = pl.clipped_policy_loss_and_grad(bad, *rest, kl=kl)
                assert torch.isnan(got_loss) and torch.isnan(pl.clipped_policy_loss(bad, *rest, kl=kl)), fill
                assert torch.isnan(got[undefined]).all(), fill
                assert torch.equal(got[~undefined], grad[~undefined]), fill
            quiet = logits.clone()
            quiet[0, 7] = quiet[2] = nan
            again = pl.clipped_policy_loss_and_grad(quiet, *policies, target, legal, weights, kl=kl)
            assert torch.equal(again[0], loss) and torch.equal(again[1], grad)
    everywhere = pl.clipped_policy_loss_and_grad(torch.full_like(logits, nan), old, adv, target, legal, weights)
    assert torch.isnan(everywhere[0]) and torch.isnan(everywhere[1][(weights != 0)[:, :, None] & legal[:, None, :]]).all()
    assert not everywhere[1][~legal[:, None, :].expand_as(logits)].any()
    leaf = torch.full_like(logits, nan).requires_grad_(True)
    value = pl.clipped_policy_loss(leaf, old, adv, target, legal, weights)
    assert torch.isnan(value) and torch.isnan(torch.autograd.grad(value, leaf)[0][1:2][legal[1:2, None, :].expand(1, hands, actions)]).all()


@pytest.mark.parametrize("states,hands,actions", [(3, 40, 5), (300, 256, 5), (40, 77, 8)])
def test_undefined_weights_are_no_batch_without_weight(cuda_device, states, hands, actions):
    nan = float("nan")
    logits, old, adv, target, legal, weights = _loss_batch(states, hands, actions, torch.float32, cuda_device)
    legal[2] = False
    weights[:, 3] = 0.0
    loss, grad = pl.clipped_policy_loss_and_grad(logits, old, adv, target, legal, weights)
    bad = weights.clone()
    bad[2] = nan  # a state that does not count
    got = pl.clipped_policy_loss_and_grad(logits, old, adv, target, legal, bad)
    assert torch.equal(got[0], loss) and torch.equal(got[1], grad)
    bad[1, 7] = nan
    counts = (bad != 0)[:, :, None] & legal[:, None, :]
    for policies in ((old, adv), (None, None)):
        for scale in (1.0, 1024.0):
            got = pl.clipped_policy_loss_and_grad(logits, *policies, target, legal, bad, scale=scale)
            assert torch.isnan(got[0]) and torch.isnan(got[1][counts]).all() and not got[1][~counts].any()
    leaf = logits.clone().requires_grad_(True)
    value = pl.clipped_policy_loss(leaf, old, adv, target, legal, bad)
    assert torch.isnan(value) and torch.isnan(torch.autograd.grad(value, leaf)[0][counts]).all()
    endless = weights.clone()
    endless[1, 7] = float("inf")
    got = pl.clipped_policy_loss_and_grad(logits, old, adv, target, legal, endless)
    assert torch.isnan(got[0]) and torch.isnan(got[1][1, 7][legal[1]]).all() and not got[1][~legal[:, None, :].expand_as(logits)].any()


def test_hand_weights_hand_an_undefined_player_on(cuda_device):
    """From a player that does not exist to the loss of a minibatch."""
    beliefs, to_act = torch.rand(4, 2 * 1326, device=cuda_device), torch.tensor([0, 1, 2, 1], device=cuda_device)
    board = torch.full((4, 5), -1, device=cuda_device)
    weights = pl.hand_weights(beliefs, to_act, board)
    assert torch.isnan(weights[2]).all() and torch.isfinite(weights[[0, 1, 3]]).all()
    logits, target = torch.randn(4, 1326, 3, device=cuda_device), torch.full((4, 1326, 3), 1 / 3, device=cuda_device)
    legal = torch.ones(4, 3, dtype=torch.bool, device=cuda_device)
    assert torch.isnan(pl.clipped_policy_loss(logits, None, None, target, legal, weights))
    board[1, 0] = 52
    assert torch.isnan(pl.hand_weights(beliefs, to_act, board)[[1, 2]]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("size", [1e-44, 1e-42, 1e-39, 1e-30, 1e30, 1e36, 3e38])
def test_weights_at_both_ends_of_fp32(cuda_device, size, dtype):
    """Their size falls out of loss and gradient, also where the reciprocal of their sum lies outside fp32."""
    for states, hands, actions in ((2, 60, 4), (40, 77, 3)):
        logits, old, adv, target, legal, weights = _loss_batch(states, hands, actions, dtype, cuda_device)
        weights = weights.clamp(min=0.1) * size
        loss, grad = pl.clipped_policy_loss_and_grad(logits, old, adv, target, legal, weights)
        want = refs.policy_loss(logits, old, adv, target, legal, weights, 0.2, 1.0, dtype)
        refs.assert_within(loss, want[0], want[1])
        refs.assert_within(grad, want[2], want[3])


def test_a_4_bit_network_saved_loaded_copied_and_moved(cuda_device, tmp_path):
    import copy

    one, two = (leaf_eval.Mx4ValueMLP(leaf_eval.ValueMLP(96, 2, seed=seed).to(cuda_device)) for seed in (1, 2))
    x = torch.randn(40, one.IN_PADDED, device=cuda_device).bfloat16()
    want, other = one.net(x), two.net(x)
    assert not torch.equal(want, other)
    torch.save(one.state_dict(), tmp_path / "net.pt")
    two.load_state_dict(torch.load(tmp_path / "net.pt", weights_only=True))
    assert torch.equal(two.net(x), want)
    torch.save(one, tmp_path / "whole.pt")
    assert torch.equal(torch.load(tmp_path / "whole.pt", weights_only=False).net(x), want)
    assert torch.equal(copy.deepcopy(one).net(x), want)
    home = two.cpu()
    assert all(m.values.device.type == m.scales.device.type == m.bias.device.type == "cpu" for m in home.net)
    for rows in (x[:2], x):
        with pytest.raises(ValueError):
            home.net(rows)
        with pytest.raises(ValueError, match="CUDA"):
            home.net(rows.cpu())
    assert torch.equal(home.to(cuda_device).net(x), want) and torch.equal(home.net(x[:1]), one.net(x[:1]))
    with pytest.raises(ValueError, match="type"):
        one.half()
    assert torch.equal(one.net(x), want)


def _gated_layer(rows, width, hidden, device):
    g = torch.Generator(device=device).manual_seed(rows + width + hidden)
    new = lambda *s: torch.randn(*s, device=device, generator=g)  # noqa: E731
    return [t.bfloat16() for t in (new(rows, width), new(hidden, width) / width ** 0.5, new(hidden, width) / width ** 0.5, new(hidden), new(hidden), new(rows, hidden))]


def _training_step(inputs, dh, **options):
    """Gradients of a step, and the bytes that were held between its passes."""
    leaves = [t.clone().requires_grad_(True) for t in inputs]
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    h = gated.gated_linear(*leaves, **options)
    held = torch.cuda.memory_allocated() - before
    return torch.autograd.grad(h, leaves, dh), held


@pytest.mark.parametrize("rows,width,hidden,keeps", [(131080, 1024, 64, True), (131080, 1024, 63, False), (840000, 2048, 5, False), (8200, 1536, 1024, True), (50000, 1024, 193, True)])
def test_what_a_training_step_holds_is_bounded(cuda_device, rows, width, hidden, keeps, monkeypatch):
    """At most 16 bytes a hidden value beside h; nothing with keep=False or without the memory; the same gradients in every way."""
    *inputs, dh = _gated_layer(rows, width, hidden, cuda_device)
    output, whole = 2 * rows * hidden, 8 * rows * ((hidden + 127) // 128 * 128)
    got, held = _training_step(inputs, dh)
    slack = 1 << 21  # (the allocator's rounding)
    assert held <= output + 16 * rows * hidden + slack and (held >= output + whole) == keeps
    apart = gated.gated_linear_backward(dh, *inputs)
    none, held = _training_step(inputs, dh, keep=False)
    assert held <= output + slack

    def full(*args, **kwargs):
        raise torch.cuda.OutOfMemoryError("no room")

    real = torch.Tensor.new_empty
    monkeypatch.setattr(torch.Tensor, "new_empty", lambda t, size, **k: full() if len(size) == 1 and size[0] == whole // 2 else real(t, size, **k))
    short, held = _training_step(inputs, dh)
    assert held <= output + slack
    for a, b, c, d in zip(got, apart, none, short):
        assert torch.equal(a, b) and torch.equal(c, b) and torch.equal(d, b)


def test_kept_values_of_more_rows_than_one_launch_takes(cuda_device):
    rows, width, hidden = 65535 * 32 + 45, 1024, 5
    *inputs, dh = _gated_layer(rows, width, hidden, cuda_device)
    size = _lib.lib().p2b_gated_kept_bytes(rows, width, hidden)
    kept = torch.empty(size // 2, dtype=torch.bfloat16, device=cuda_device)
    gated._forward(*inputs, 0, kept)
    needs = (False, True, True, True, True)
    for a, b in zip(gated._backward(dh, *inputs, kept, 0, needs)[1:], gated.gated_linear_backward(dh, *inputs, needs=needs)[1:]):
        assert torch.equal(a, b)


def test_networks_take_the_switch(cuda_device):
    kept, anew = (leaf_eval.GatedValueMLP(1024, 2, hidden=1024, keep=keep, seed=3).to(cuda_device) for keep in (True, False))
    x = torch.randn(8200, 1024, device=cuda_device).bfloat16()
    grads = [torch.autograd.grad(net.net[2](x).float().sum(), net.net[2].gate_weight)[0] for net in (kept, anew)]
    assert kept.net[2].keep and not anew.net[2].keep and torch.equal(*grads)


def _leaves(device, leaves=70, seed=1):
    g = torch.Generator(device=device).manual_seed(seed)
    boards = torch.rand(leaves, 48, device=device, generator=g).argsort(dim=1)[:, :5] + 4  # none of cards 0 to 3
    boards[:, 4] = -1
    beliefs = torch.zeros(leaves, 2, 1344, device=device)
    beliefs[..., :1326] = torch.rand(leaves, 2, 1326, device=device, generator=g)
    beliefs /= beliefs.sum(-1, keepdim=True)
    return boards, beliefs, torch.rand(leaves, 3, device=device, generator=g)


def test_a_first_layer_in_16_bits_sees_what_a_shared_scale_hides(cuda_device):
    """A one-hot card of 1 in a block leaves nothing of range entries below 1/16 beside it; in 16 bits it does."""
    source = leaf_eval.ValueMLP(96, 2, seed=5).to(cuda_device)
    with torch.no_grad():
        source.net[0].weight[:, 2624:2652] *= 30.0
    whole, mixed = leaf_eval.Mx4ValueMLP(source), leaf_eval.Mx4ValueMLP(source, quantise_first=False)
    boards, beliefs, context = _leaves(cuda_device)
    other = beliefs.clone()
    other[:, 1, 1298:1326] *= 20.0  # columns 2624 to 2651
    assert other[:, 1, 1298:1326].max() < 1 / 16
    for card, hidden in ((3, True), (4, False)):
        boards[:, 0] = card
        same = [torch.equal(net(beliefs[..., :1326], boards, context), net(other[..., :1326], boards, context)) for net in (whole, mixed)]
        assert same == [hidden, False]
    x = torch.randn(50, 2720, device=cuda_device).bfloat16()
    with torch.no_grad():
        y = torch.nn.functional.gelu(source.net[0](x))
        for layer, last in zip(list(mixed.net)[2:], (False, True)):
            y = mx4.linear(y, layer.weight, layer.bias, activation="none" if last else "gelu")
    assert torch.equal(mixed.net(x), y) and torch.equal(mixed.layers(x), y)
    direct = leaf_eval.DirectLeafEvaluator(mixed, boards, context, cuda_device)
    assert direct._direct() and torch.equal(direct(beliefs), mixed(beliefs[..., :1326], boards, context))


@pytest.mark.parametrize("kind", [leaf_eval.DirectLeafEvaluator, leaf_eval.ChanceLeafEvaluator])
def test_evaluators_read_a_4_bit_network_in_its_type(cuda_device, kind):
    source = leaf_eval.ValueMLP(96, 2, seed=6).to(cuda_device)
    half = leaf_eval.Mx4ValueMLP(leaf_eval.ValueMLP(96, 2, seed=6).to(cuda_device).half())
    boards, beliefs, context = _leaves(cuda_device, leaves=9)
    got, want = (kind(net, boards, context, cuda_device)(beliefs) for net in (half, leaf_eval.Mx4ValueMLP(source)))
    # (of one network in two types: roundings to 8 bits and the 4-bit steps that these change)
    assert torch.isfinite(got).all() and (got[..., :1326] - want[..., :1326]).norm() < 0.5 * want.norm()
    if kind is leaf_eval.DirectLeafEvaluator:  # another network put in place of the one it was made for
        short = kind(leaf_eval.Mx4ValueMLP(source), boards, context, cuda_device)
        assert short._direct()
        short.model = half
        assert not short._direct() and torch.equal(short(beliefs), got)
