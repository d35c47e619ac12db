"""Calls of the network operators that must not reach a kernel: refused on the host, no GPU needed.  `_lib.call` is replaced by one that
keeps what would have been called."""
import contextlib

import pytest
import torch

from poker2_b200 import _lib, mx4


@pytest.fixture
def launches(monkeypatch):
    seen = []
    monkeypatch.setattr(_lib, "call", lambda name, *args: seen.append(name))
    monkeypatch.setattr(_lib, "_get_device", lambda: 0)
    monkeypatch.setattr(_lib, "_raw_stream", lambda device: 0)
    # as with a GPU there: no device -1, so the current one
    monkeypatch.setattr(torch.cuda, "device", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: type("Stream", (), {"cuda_stream": 0}))
    return seen


def _quantised(rows, width, scales=None):
    scales = (rows + 127) // 128 * ((width + 255) // 256) * 1024 if scales is None else scales
    return mx4.Mx4(torch.zeros(rows, (width + 31) // 32 * 16, dtype=torch.uint8), torch.zeros(scales, dtype=torch.uint8), (rows, width))


@pytest.mark.parametrize("call", [
    lambda w: mx4.linear(torch.zeros(2, 32, dtype=torch.bfloat16), w), lambda w: mx4.linear(torch.zeros(40, 32), w), lambda w: mx4.linear(w, w),
    lambda w: mx4.linear(w, w, quantised=True), lambda w: w.dequantise(),
])
def test_matrices_in_host_memory_are_refused(launches, call):
    with pytest.raises(ValueError, match="CUDA"):
        call(_quantised(4, 32))
    assert not launches


def test_calls_without_a_device_are_refused(launches):
    with pytest.raises(ValueError, match="CUDA"):
        _lib.call_on(-1, "p2b_mx4_quantise")
    assert not launches


class _Elsewhere(torch.Tensor):
    """A CPU tensor that says it lies on a GPU."""

    def get_device(self):
        return 0


def _there(m):
    return mx4.Mx4(m.values.as_subclass(_Elsewhere), m.scales.as_subclass(_Elsewhere), m.shape)


def test_matrices_smaller_than_they_say_are_refused(launches):
    good = _there(_quantised(40, 300))
    mx4.linear(good, good)
    mx4.linear(good, good, quantised=True)
    good.dequantise()
    row = _there(_quantised(1, 300))
    row.shape = (300,)
    assert row.dequantise().shape == (300,)
    assert launches == ["p2b_mx4_linear", "p2b_mx4_linear_mx4", "p2b_mx4_dequantise", "p2b_mx4_dequantise"]
    launches.clear()
    v, s = good.values, good.scales
    for values, scales, shape in ((v[:39], s, (40, 300)), (v, s[:-1], (40, 300)), (v, s, (41, 300)), (v, s, (2, 21, 300)), (v, s, (40, 321)), (v, s, (40, 513)),
                                  (torch.zeros(40, 320, dtype=torch.uint8).as_subclass(_Elsewhere)[:, ::2], s, (40, 300)),
                                  (v, torch.zeros(4096, dtype=torch.uint8).as_subclass(_Elsewhere)[::2], (40, 300)), (v, torch.zeros(2048, dtype=torch.uint8), (40, 300)),
                                  (v.view(80, 80), s, (40, 300))):
        bad, width = mx4.Mx4(values, scales, shape), shape[-1]
        with pytest.raises(ValueError, match="shape says"):
            bad.dequantise()
        other = _there(_quantised(40, width))
        for call in (lambda: mx4.linear(bad, other), lambda: mx4.linear(bad, other, quantised=True)):
            with pytest.raises(ValueError, match="shape says"):
                call()
        if len(shape) == 2:
            with pytest.raises(ValueError, match="shape says"):
                mx4.linear(other, bad)
    assert not launches


def test_hand_weights_of_players_and_cards_that_do_not_exist(monkeypatch):
    """An index outside its range is an error on the CPU and the end of the context on a GPU: such states' weights are NaN instead."""
    from poker2_b200 import fused_cfr, policy_loss

    c1, c2 = torch.triu_indices(52, 52, 1)
    apart = ((c1[:, None] != c1) & (c1[:, None] != c2) & (c2[:, None] != c1) & (c2[:, None] != c2)).float()
    monkeypatch.setattr(_lib, "require_cuda", lambda t, what: None)
    monkeypatch.setattr(fused_cfr, "unblocked_mass_triton", lambda ranges: ranges @ apart)
    beliefs = torch.rand(8, 2 * 1326)
    to_act = torch.tensor([0, 1, 2, -1, 0, 1, 0, 7])
    board = torch.tensor([[3, 9, 20, -1, -1]] * 8)
    board[4, 1], board[5, 4], board[6, 3] = 52, 1 << 40, -7
    got = policy_loss.hand_weights(beliefs, to_act, board)
    wrong = torch.tensor([False, False, True, True, True, True, False, True])
    assert got.dtype == torch.float32 and torch.isnan(got[wrong]).all()
    assert torch.equal(got[~wrong], policy_loss.hand_weights(beliefs[~wrong], to_act[~wrong], board[~wrong]))
    ranges = beliefs.view(8, 2, 1326)
    for row in (0, 1, 6):
        blocked = torch.zeros(1326, dtype=torch.bool)
        for card in board[row].tolist():
            blocked |= (c1 == card) | (c2 == card)
        want = torch.where(blocked, 0.0, ranges[row, to_act[row]].double() * (ranges[row, 1 - to_act[row]].double() @ apart.double()))
        # 1326 terms in fp32 and a product: 2^-24 each
        assert ((got[row] - want).abs() <= want * 1400 * 2.0 ** -24).all()
    assert policy_loss.hand_weights(beliefs[:0], to_act[:0], board[:0]).shape == (0, 1326)


@pytest.fixture(scope="module")
def handle():
    from poker2_b200 import build

    build.build()
    return _lib.lib()


def test_addresses_between_elements_are_refused(handle):
    """An odd address would be a misaligned access of the kernel."""
    import ctypes

    area = (ctypes.c_char * 8192)()
    p = (ctypes.addressof(area) + 63) // 64 * 64
    for rows in (2, 16):
        good = dict(x=p, xs=64, wg=p, gs=64, wu=p, us=64, bg=p, bu=p, rows=rows, width=64, hidden=8, dtype=0, act=0, h=p, hs=8, kept=None, scratch=p, size=1 << 20, stream=None)
        for name in ("x", "wg", "wu", "bg", "bu", "h"):
            assert handle.p2b_gated_forward(*{**good, name: p + 1}.values()) == -1 and b"2-byte" in handle.p2b_last_error(), name
        good = dict(dh=p, ds=8, x=p, xs=64, wg=p, gs=64, wu=p, us=64, bg=p, bu=p, rows=rows, width=64, hidden=8, dtype=0, act=0, dx=p, dxs=64, dwg=p, dwu=p, dbg=p,
                    dbu=p, kept=None, scratch=p, size=1 << 20, stream=None)
        for name in ("dh", "x", "wg", "wu", "bg", "bu", "dx", "dwg", "dwu", "dbg", "dbu"):
            assert handle.p2b_gated_backward(*{**good, name: p + 1}.values()) == -1 and b"2-byte" in handle.p2b_last_error(), name
    for args in ((p + 1, p, 4, 0, p), (p, p + 2, 4, 0, p), (p, p, 4, 1, p + 1), (p + 2, p, 4, 2, p), (p, p, 4, 2, p + 2)):
        assert handle.p2b_policy_loss_scale(*args, None) == -1 and b"boundaries" in handle.p2b_last_error()


def test_policy_loss_scales_that_are_refused(handle):
    import ctypes

    from poker2_b200 import policy_loss as pl

    area = (ctypes.c_char * 4096)()
    p = (ctypes.addressof(area) + 63) // 64 * 64
    good = dict(logits=p, old=p, adv=p, target=p, legal=p, weights=p, states=2, hands=3, actions=4, dtype=1, clip=0.2, kl=1.0, loss=p, grad=p, gdtype=1, factor=1.0, at=p,
                scratch=p, size=1 << 20, stream=None)
    for change in (dict(gdtype=0), dict(gdtype=3), dict(gdtype=-1), dict(factor=float("inf")), dict(factor=float("nan")), dict(at=p + 2), dict(gdtype=2, grad=p + 2),
                   dict(grad=p + 1), dict(dtype=2, gdtype=1), dict(logits=None), dict(states=-1), dict(scratch=None, states=3000)):
        assert handle.p2b_policy_loss_scaled(*{**good, **change}.values()) == -1 and b"p2b_policy_loss" in handle.p2b_last_error(), change
    for args in ((None, p, 4, p), (p, None, 4, p), (p, p, 4, None), (p, p, -1, p), (p + 2, p, 4, p), (p, p + 2, 4, p), (p, p, 4, p + 1)):
        assert handle.p2b_policy_loss_scale_fp32(*args, None) == -1
    assert handle.p2b_policy_loss_scale_fp32(None, None, 0, None, None) == 0
    there = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype).as_subclass(_Elsewhere)  # noqa: E731
    call = lambda scale: pl.clipped_policy_loss_and_grad(there(2, 3, 4), None, None, there(2, 3, 4), there(2, 4, dtype=torch.bool), scale=scale)  # noqa: E731
    for scale in (float("inf"), float("nan"), 1e300, there(2), there(1, dtype=torch.float64), torch.ones(1)):
        with pytest.raises(ValueError, match="scale"):
            call(scale)


def _quantise_here(x):
    """A stand-in for the kernel: different arrays for different weights."""
    rows, width = x.shape
    m = _quantised(rows, width)
    m.values.copy_(torch.arange(m.values.numel()).view_as(m.values).add_(int(1e6 * x.double().abs().sum())).remainder_(251))
    m.scales.fill_(int(1e6 * x.double().abs().sum()) % 250)
    return m


@pytest.fixture
def networks(monkeypatch):
    from poker2_b200 import leaf_eval

    monkeypatch.setattr(mx4, "quantise", _quantise_here)
    return lambda seed, width=64, dtype=torch.bfloat16: leaf_eval.Mx4ValueMLP(leaf_eval.ValueMLP(width, 2, seed=seed, dtype=dtype))


def _same_weights(a, b):
    return all(torch.equal(x.weight.values, y.weight.values) and torch.equal(x.weight.scales, y.weight.scales) and torch.equal(x.bias, y.bias)
               for x, y in zip(a.net, b.net))


def test_a_4_bit_network_is_saved_and_loaded_with_its_weights(networks, tmp_path):
    import copy

    one, two = networks(1), networks(2)
    assert not _same_weights(one, two)
    torch.save(one.state_dict(), tmp_path / "net.pt")
    state = torch.load(tmp_path / "net.pt", weights_only=True)
    assert {f"net.{i}.{k}" for i in range(3) for k in ("values", "scales", "bias")} <= set(state)
    for assign in (False, True):
        two = networks(2)
        two.load_state_dict(state, strict=True, assign=assign)
        assert _same_weights(one, two)
    assert _same_weights(copy.deepcopy(one), one)
    with pytest.raises(RuntimeError, match="Missing"):
        two.load_state_dict({k: v for k, v in state.items() if "bias" in k})
    with pytest.raises(RuntimeError, match="size mismatch|does not fit"):
        networks(3, 128).load_state_dict(state)
    # 60 and 64 columns have arrays of one size, and are not one matrix
    other = networks(3, 60)
    before = copy.deepcopy(other)
    with pytest.raises(RuntimeError, match="does not fit"):
        other.net[2].load_state_dict({k[6:]: v for k, v in state.items() if k.startswith("net.2.")})
    assert _same_weights(before, other)
    bias = one.net[0].bias
    one.net[0].bias = None
    assert "bias" not in one.net[0].state_dict() and bias is not None


def test_a_4_bit_network_keeps_its_type_and_moves_as_a_whole(networks):
    net = networks(1)
    same = networks(1)
    for change in (lambda: net.half(), lambda: net.float(), lambda: net.to(torch.float16), lambda: net.double(), lambda: net.type(torch.float32)):
        with pytest.raises(ValueError, match="type"):
            change()
        assert _same_weights(net, same) and net.net[0].bias.dtype == torch.bfloat16
    net.to(torch.bfloat16).to("cpu")
    assert _same_weights(net, same)
    away = net.to("meta")
    for layer in away.net:
        assert {layer.values.device.type, layer.scales.device.type, layer.bias.device.type} == {"meta"}
    assert networks(1, dtype=torch.float16).half().net[0].dtype == torch.float16


def test_a_4_bit_network_in_host_memory_refuses_its_calls(networks, launches):
    net = networks(1)
    for rows in (2, 40):
        with pytest.raises(ValueError, match="CUDA"):
            net.net(torch.zeros(rows, net.IN_PADDED, dtype=torch.bfloat16))
    assert not launches


def test_forward_mode_tangents_are_refused(launches):
    """A dual tensor requires no gradient, so it would pass for a constant and its tangent be lost."""
    from poker2_b200 import gated, policy_loss as pl

    bf16 = lambda *s: torch.zeros(*s, dtype=torch.bfloat16).as_subclass(_Elsewhere)  # noqa: E731
    f32 = lambda *s: torch.zeros(*s).as_subclass(_Elsewhere)  # noqa: E731
    legal, w = torch.ones(2, 4, dtype=torch.bool).as_subclass(_Elsewhere), _there(_quantised(4, 32))
    layer = [lambda: bf16(5, 32), lambda: bf16(8, 32), lambda: bf16(8, 32), lambda: bf16(8), lambda: bf16(8)]
    loss = [lambda: f32(2, 3, 4), lambda: f32(2, 3, 4), lambda: f32(2, 3, 4), lambda: f32(2, 3, 4), lambda: f32(2, 3)]
    calls = [
        (gated.gated_linear, layer), (gated.gated_linear_backward, [lambda: bf16(5, 8), *layer]), (mx4.quantise, [lambda: f32(3, 32)]),
        (lambda x, b: mx4.linear(x, w, b), [lambda: bf16(3, 32), lambda: bf16(4)]), (lambda b: mx4.linear(_there(_quantised(6, 32)), w, b), [lambda: bf16(4)]),
        (lambda x: mx4.linear(x, w, quantised=True), [lambda: bf16(3, 32)]),
        (lambda z, o, a, t, h: pl.clipped_policy_loss(z, o, a, t, legal, h), loss),
        (lambda z, o, a, t, h: pl.clipped_policy_loss_and_grad(z, o, a, t, legal, h), loss),
    ]
    for call, make in calls:
        with torch.autograd.forward_ad.dual_level():
            for i in range(len(make)):
                args = [m() for m in make]
                args[i] = torch.autograd.forward_ad.make_dual(args[i], torch.ones_like(args[i]))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call(*args)
                with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                    call(*args)
            assert not launches
            call(*(m() for m in make))  # (without a tangent it goes through there too)
            assert launches
            launches.clear()
        call(*(m() for m in make))
        launches.clear()


def test_hand_weights_have_no_gradient(monkeypatch):
    """One factor of the product comes from a kernel: a gradient through the other alone would be half of it."""
    from poker2_b200 import fused_cfr, policy_loss

    monkeypatch.setattr(_lib, "require_cuda", lambda t, what: None)
    monkeypatch.setattr(fused_cfr, "unblocked_mass_triton", lambda ranges: ranges.detach() * 0 + 1)
    beliefs, to_act, board = torch.rand(2, 2 * 1326), torch.tensor([0, 1]), torch.full((2, 5), -1)
    want = policy_loss.hand_weights(beliefs, to_act, board)
    leaf = beliefs.clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="detach"):
        policy_loss.hand_weights(leaf, to_act, board)
    with torch.no_grad():
        assert torch.equal(policy_loss.hand_weights(leaf, to_act, board), want)
    with torch.autograd.forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        policy_loss.hand_weights(torch.autograd.forward_ad.make_dual(beliefs, torch.ones_like(beliefs)), to_act, board)


def test_a_4_bit_network_whose_first_layer_stays(networks):
    from poker2_b200 import leaf_eval

    source = leaf_eval.ValueMLP(64, 2, seed=4)
    net = leaf_eval.Mx4ValueMLP(source, quantise_first=False)
    assert [type(m) for m in net.net] == [torch.nn.Linear, torch.nn.GELU, leaf_eval.Mx4Linear, leaf_eval.Mx4Linear]
    assert [m.hands_on for m in list(net.net)[2:]] == [True, False] and [m.activation for m in list(net.net)[2:]] == ["gelu", "none"]
    assert torch.equal(net.net[0].weight, source.net[0].weight) and net.net[0].weight is not source.net[0].weight and not net.net[0].weight.requires_grad
    other = leaf_eval.Mx4ValueMLP(leaf_eval.ValueMLP(64, 2, seed=5), quantise_first=False)
    other.load_state_dict(net.state_dict())
    assert all(torch.equal(a, b) for a, b in zip(net.buffers(), other.buffers())) and torch.equal(net.net[0].weight, other.net[0].weight)
    with pytest.raises(ValueError, match="type"):
        net.half()
    assert net.net[0].weight.dtype == torch.bfloat16
    with pytest.raises(ValueError, match="nothing"):
        leaf_eval.Mx4ValueMLP(leaf_eval.ValueMLP(64, 0), quantise_first=False)


def test_a_4_bit_network_has_the_type_of_its_layers(networks):
    """A source made in bf16 and turned into fp16 gives fp16 outputs, which the evaluators' short paths would read as bf16."""
    from poker2_b200 import leaf_eval

    source = leaf_eval.ValueMLP(64, 1)
    assert leaf_eval.Mx4ValueMLP(source).dtype == torch.bfloat16
    net = leaf_eval.Mx4ValueMLP(source.half())
    assert net.dtype == torch.float16 and all(layer.dtype == torch.float16 for layer in net.net)
    assert not leaf_eval.ChanceLeafEvaluator(net, torch.full((2, 5), -1), torch.zeros(2, 3), torch.device("cpu")).fused
    source.net[0].bfloat16()
    with pytest.raises(ValueError, match="one type"):
        leaf_eval.Mx4ValueMLP(source)
    with pytest.raises(ValueError, match="one type"):
        leaf_eval.Mx4ValueMLP(leaf_eval.ValueMLP(64, 1).float())
