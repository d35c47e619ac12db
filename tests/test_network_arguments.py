"""What the network operators refuse, before any launch: no GPU needed."""
import ctypes

import pytest
import torch

from poker2_b200 import _lib, build, gated


@pytest.fixture(scope="module")
def handle():
    build.build()
    return _lib.lib()


def _area():
    area = (ctypes.c_char * 4096)()
    return area, (ctypes.addressof(area) + 63) // 64 * 64


def _gated_forward(p, **change):
    a = dict(x=p, xs=64, wg=p, gs=64, wu=p, us=64, bg=None, bu=None, rows=16, width=64, hidden=8, dtype=0, act=0, h=p, hs=8, kept=None, scratch=None, size=0)
    a.update(change)
    return [*a.values(), None]


def _gated_backward(p, **change):
    a = dict(dh=p, ds=8, x=p, xs=64, wg=p, gs=64, wu=p, us=64, bg=None, bu=None, rows=16, width=64, hidden=8, dtype=0, act=0, dx=p, dxs=64,
             dwg=None, dwu=None, dbg=None, dbu=None, kept=None, scratch=p, size=None)
    a.update(change)
    if a["size"] is None:  # what the layer itself needs, nothing for copies
        a["size"] = max(0, _lib.lib().p2b_gated_backward_scratch_bytes(max(0, min(a["rows"], 1 << 29)), 64, 8))
    return [*a.values(), None]


LAYER = [dict(rows=-1), dict(rows=1 << 40), dict(width=0), dict(width=1 << 24), dict(hidden=0), dict(hidden=-3), dict(dtype=2), dict(dtype=-1),
         dict(act=2), dict(x=None), dict(wg=None), dict(wu=None), dict(xs=63), dict(gs=8), dict(us=0), dict(rows=1 << 29, hidden=1 << 19)]


@pytest.mark.parametrize("change", LAYER + [dict(h=None), dict(hs=7), dict(kept=64), dict(xs=65), dict(gs=68), dict(us=66)])
def test_gated_forward_refuses(handle, change):
    area, p = _area()
    assert handle.p2b_gated_forward(*_gated_forward(p, **change)) == -1 and b"p2b_gated_forward" in handle.p2b_last_error()


@pytest.mark.parametrize("change", LAYER + [dict(dh=None), dict(ds=7), dict(dxs=63), dict(scratch=None), dict(size=100), dict(kept=64), dict(xs=68), dict(us=65)])
def test_gated_backward_refuses(handle, change):
    area, p = _area()
    assert handle.p2b_gated_backward(*_gated_backward(p, **change)) == -1 and b"p2b_gated_backward" in handle.p2b_last_error()


def test_gated_addresses_off_their_boundaries_are_refused(handle):
    area, p = _area()
    for name in ("x", "wg", "wu"):
        assert handle.p2b_gated_forward(*_gated_forward(p, **{name: p + 2})) == -1 and b"16-byte" in handle.p2b_last_error()
        assert handle.p2b_gated_backward(*_gated_backward(p, **{name: p + 8})) == -1 and b"16-byte" in handle.p2b_last_error()
        assert handle.p2b_gated_forward(*_gated_forward(p, **{name: p + 2}, scratch=p, size=100)) == -1 and b"16-byte" in handle.p2b_last_error()
        assert handle.p2b_gated_forward(*_gated_forward(p, **{name: p + 2}, scratch=p + 8, size=1 << 20)) == -1 and b"16-byte" in handle.p2b_last_error()
    assert handle.p2b_gated_backward(*_gated_backward(p, scratch=p + 4)) == -1
    assert handle.p2b_gated_align_bytes(16, 65, 8) == 2 * 32 * 72 and handle.p2b_gated_align_bytes(-1, 65, 8) == -1
    assert handle.p2b_gated_forward(*_gated_forward(None, rows=0, wg=p, wu=p)) == 0  # no rows: nothing to do
    assert handle.p2b_gated_few_rows() == gated.FEW_ROWS
    for sizes in ((-1, 8, 8), (8, 0, 8), (8, 8, 0)):
        assert handle.p2b_gated_backward_scratch_bytes(*sizes) == -1 and handle.p2b_gated_kept_bytes(*sizes) == -1
    assert gated.KEPT_PRODUCTS == 8192 * 1024 * 1024 and handle.p2b_gated_kept_bytes(8192, 1024, 1024) == 8 * 8192 * 1024
    assert handle.p2b_gated_kept_bytes(8192, 1024, 1025) == 8 * 8192 * 1152
    for sizes in ((8191, 1024, 1024), (8192, 1024, 1023), (9000, 1016, 1024), (4, 1 << 19, 4800), (512, 1 << 16, 1024)):
        assert handle.p2b_gated_kept_bytes(*sizes) == 0


def test_gated_linear_wants_the_gpu():
    x, w = torch.zeros(2, 8, dtype=torch.bfloat16), torch.zeros(4, 8, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        gated.gated_linear(x, w, w)


class _Elsewhere(torch.Tensor):
    """A CPU tensor that says it lies on a GPU, for the checks that come before any launch."""

    @property
    def device(self):
        return torch.device("cuda:0")

    def get_device(self):
        return 0


def _there(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype).as_subclass(_Elsewhere)


def test_gated_linear_refuses():
    x, w, b = _there(2, 8), _there(4, 8), _there(4)
    bad = [
        dict(x=_there(2, 8, dtype=torch.float32)), dict(x=_there(2, 7)), dict(gate_weight=_there(5, 8)), dict(up_weight=_there(4)),
        dict(gate_weight=_there(0, 8), up_weight=_there(0, 8)), dict(gate_weight=_there(4, 8, dtype=torch.float16)),
        dict(gate_bias=_there(5)), dict(up_bias=_there(4, dtype=torch.float32)), dict(up_bias=torch.zeros(4, dtype=torch.bfloat16)),
        dict(activation="relu"),
    ]
    for change in bad:
        args = dict(x=x, gate_weight=w, up_weight=w, gate_bias=b, up_bias=b, activation="gelu")
        args.update(change)
        with pytest.raises(ValueError):
            gated._check(*args.values())


def _refused(handle, name, **change):
    area, p = _area()
    calls = {
        "p2b_mx4_quantise": dict(x=p, stride=64, rows=4, width=64, dtype=0, values=p, scales=p, stream=None),
        "p2b_mx4_dequantise": dict(values=p, scales=p, rows=4, width=64, dtype=0, out=p, stride=64, stream=None),
        "p2b_mx4_linear_mx4": dict(a=p, sa=p, rows=4, w=p, sw=p, columns=8, width=64, bias=p, dtype=0, act=0, values=p, scales=p, stream=None),
        "p2b_mx4_linear_rows": dict(x=p, xs=64, xdtype=0, rows=40, w=p, sw=p, columns=8, width=64, bias=p, dtype=0, act=0, out=p, stride=8, scratch=p, size=4096,
                                    stream=None),
        "p2b_mx4_linear_few": dict(x=p, xs=64, xdtype=0, rows=4, w=p, sw=p, columns=8, width=64, bias=p, dtype=0, act=0, out=p, stride=8, stream=None),
        "p2b_mx4_linear": dict(a=p, sa=p, rows=4, w=p, sw=p, columns=8, width=64, bias=p, dtype=0, act=0, out=p, stride=8, stream=None),
    }
    args = calls[name]
    args.update({k: p + v[0] if isinstance(v, tuple) else v for k, v in change.items()})
    return getattr(handle, name)(*args.values()) == -1 and name.encode() in handle.p2b_last_error()


MATRIX = [dict(rows=-1), dict(rows=1 << 40), dict(width=0), dict(width=-5), dict(width=1 << 24), dict(dtype=3), dict(dtype=-1)]


@pytest.mark.parametrize("change", MATRIX + [dict(x=None), dict(values=None), dict(scales=None), dict(stride=-1), dict(values=(8,)), dict(scales=(4,)), dict(x=(1,))])
def test_mx4_quantise_refuses(handle, change):
    assert _refused(handle, "p2b_mx4_quantise", **change)


@pytest.mark.parametrize("change", MATRIX + [dict(out=None), dict(values=None), dict(scales=None), dict(stride=63), dict(values=(8,)), dict(scales=(4,)), dict(out=(1,))])
def test_mx4_dequantise_refuses(handle, change):
    assert _refused(handle, "p2b_mx4_dequantise", **change)


@pytest.mark.parametrize("change", MATRIX + [dict(dtype=2), dict(act=3), dict(act=-1), dict(columns=0), dict(columns=1 << 30), dict(a=None), dict(sa=None), dict(w=None),
                                             dict(sw=None), dict(out=None), dict(stride=7), dict(a=(8,)), dict(sa=(1,)), dict(w=(4,)), dict(sw=(8,)), dict(out=(1,)),
                                             dict(bias=(1,)), dict(rows=1 << 30, columns=1 << 20)])
def test_mx4_linear_refuses(handle, change):
    assert _refused(handle, "p2b_mx4_linear", **change)


@pytest.mark.parametrize("change", [dict(rows=-1), dict(rows=5), dict(width=0), dict(columns=0), dict(columns=1 << 30), dict(dtype=2), dict(xdtype=3), dict(xdtype=-1), dict(act=3),
                                    dict(x=None), dict(w=None), dict(sw=None), dict(out=None), dict(xs=-1), dict(stride=7), dict(w=(8,)), dict(sw=(4,)), dict(x=(1,)),
                                    dict(xdtype=2, x=(2,)), dict(out=(1,)), dict(bias=(1,))])
def test_mx4_linear_few_refuses(handle, change):
    assert _refused(handle, "p2b_mx4_linear_few", **change)


@pytest.mark.parametrize("change", MATRIX + [dict(dtype=2), dict(act=3), dict(columns=0), dict(a=None), dict(sa=None), dict(w=None), dict(sw=None), dict(values=None),
                                             dict(scales=None), dict(values=(8,)), dict(scales=(4,)), dict(a=(8,)), dict(bias=(1,)), dict(rows=1 << 30, columns=1 << 20)])
def test_mx4_linear_mx4_refuses(handle, change):
    assert _refused(handle, "p2b_mx4_linear_mx4", **change)


@pytest.mark.parametrize("change", MATRIX[1:] + [dict(dtype=2), dict(act=3), dict(columns=0), dict(w=None), dict(sw=None), dict(out=None), dict(stride=7), dict(w=(8,)),
                                                 dict(sw=(4,)), dict(out=(1,)), dict(bias=(1,)), dict(scratch=None), dict(scratch=(8,)), dict(size=1663),
                                                 dict(x=None), dict(xs=-1), dict(xdtype=3), dict(x=(1,))])
def test_mx4_linear_rows_refuses(handle, change):
    assert _refused(handle, "p2b_mx4_linear_rows", **change)


def test_mx4_sizes(handle):
    from poker2_b200 import mx4

    assert handle.p2b_mx4_few_rows() == mx4.FEW_ROWS
    assert handle.p2b_mx4_linear_rows_scratch_bytes(4, 64) == 0 and handle.p2b_mx4_linear_rows_scratch_bytes(40, 65) == 1024 + 40 * 48
    assert handle.p2b_mx4_linear_rows_scratch_bytes(-1, 64) == -1
    assert handle.p2b_mx4_value_bytes(3, 33) == 96 and handle.p2b_mx4_scale_bytes(129, 257) == 2 * 4 * 512
    assert handle.p2b_mx4_value_bytes(-1, 33) == -1 and handle.p2b_mx4_scale_bytes(1, 0) == -1
    assert handle.p2b_mx4_quantise(None, 0, 0, 64, 0, None, None, None) == 0
    assert handle.p2b_mx4_linear(None, None, 0, None, None, 8, 64, None, 0, 0, None, 8, None) == 0


def test_mx4_python_refuses():
    from poker2_b200 import mx4

    with pytest.raises(ValueError, match="CUDA"):
        mx4.quantise(torch.zeros(2, 32))
    for bad in (_there(2, 0), _there(2, 32, dtype=torch.float64), torch.zeros((), dtype=torch.bfloat16).as_subclass(_Elsewhere)):
        with pytest.raises(ValueError):
            mx4.quantise(bad)
    w = mx4.Mx4(_there(4, 16, dtype=torch.uint8), _there(1024, dtype=torch.uint8), (4, 32))
    x = mx4.Mx4(_there(2, 16, dtype=torch.uint8), _there(1024, dtype=torch.uint8), (2, 32))
    with pytest.raises(ValueError):
        w.dequantise(torch.float64)
    for change in (dict(weight=_there(4, 32)), dict(activation="relu"), dict(dtype=torch.float32), dict(bias=_there(3)), dict(bias=_there(4, dtype=torch.float16)),
                   dict(x=mx4.Mx4(x.values, x.scales, (2, 31))), dict(weight=mx4.Mx4(w.values, w.scales, (2, 2, 32))), dict(weight=mx4.Mx4(w.values, w.scales, (0, 32)))):
        args = dict(x=x, weight=w, bias=None, activation="none", dtype=None)
        args.update(change)
        with pytest.raises(ValueError):
            mx4.linear(args["x"], args["weight"], args["bias"], activation=args["activation"], dtype=args["dtype"])
    with pytest.raises(ValueError):
        mx4.linear(_there(2, 32, dtype=torch.float64), w)
    with pytest.raises(RuntimeError, match="gradient"):
        mx4.linear(_there(2, 32).requires_grad_(True), w)


def _loss(p, **change):
    a = dict(logits=p, old=p, adv=p, target=p, legal=p, weights=p, states=2, hands=3, actions=4, dtype=0, clip=0.2, kl=1.0, loss=p, grad=p, scratch=p, size=1 << 20)
    a.update({k: p + v[0] if isinstance(v, tuple) else v for k, v in change.items()})
    return [*a.values(), None]


@pytest.mark.parametrize("change", [dict(states=-1), dict(states=1 << 40), dict(hands=0), dict(actions=0), dict(actions=17), dict(dtype=3), dict(clip=1.0), dict(clip=-0.1),
                                    dict(clip=float("nan")), dict(kl=-1.0), dict(kl=float("inf")), dict(kl=float("nan")), dict(loss=None), dict(states=3000, scratch=None),
                                    dict(states=3000, size=8), dict(states=3000, scratch=(4,)), dict(old=None), dict(adv=None), dict(logits=None), dict(target=None), dict(legal=None),
                                    dict(logits=(1,)), dict(old=(2,)), dict(target=(1,)), dict(weights=(2,)), dict(grad=(1,)), dict(loss=(2,)),
                                    dict(dtype=2, logits=(2,))])
def test_policy_loss_refuses(handle, change):
    area, p = _area()
    assert handle.p2b_policy_loss(*_loss(p, **change)) == -1 and b"p2b_policy_loss" in handle.p2b_last_error()


def test_policy_loss_scale_refuses(handle):
    area, p = _area()
    for args in ((None, p, 4, 0, p), (p, None, 4, 0, p), (p, p, 4, 0, None), (p, p, -1, 0, p), (p, p, 4, 3, p)):
        assert handle.p2b_policy_loss_scale(*args, None) == -1
    assert handle.p2b_policy_loss_scale(None, None, 0, 0, None, None) == 0
    assert handle.p2b_policy_loss_scratch_bytes(-1, 4) == -1 and handle.p2b_policy_loss_scratch_bytes(1, 0) == -1


def test_policy_loss_python_refuses():
    from poker2_b200 import policy_loss as pl

    with pytest.raises(ValueError, match="CUDA"):
        pl.clipped_policy_loss(torch.zeros(2, 3, 4), None, None, torch.zeros(2, 3, 4), torch.ones(2, 4, dtype=torch.bool))
    f32 = torch.float32
    good = dict(logits=_there(2, 3, 4), old_policy=_there(2, 3, 4, dtype=f32), advantages=_there(2, 3, 4, dtype=f32), target=_there(2, 3, 4, dtype=f32),
                legal=_there(2, 4, dtype=torch.bool), weights=_there(2, 3, dtype=f32), clip=0.2, kl=1.0)
    pl._check(*good.values())
    for change in (dict(logits=_there(2, 12)), dict(logits=_there(2, 3, 17)), dict(logits=_there(2, 3, 4, dtype=torch.float64)), dict(old_policy=None),
                   dict(advantages=None), dict(target=_there(2, 3, 4)), dict(target=_there(2, 3, 5, dtype=f32)), dict(target=torch.zeros(2, 3, 4)),
                   dict(legal=_there(2, 3, 4, dtype=torch.bool)), dict(legal=_there(2, 4, dtype=torch.uint8)), dict(weights=_there(2, 4, dtype=f32)),
                   dict(weights=_there(2, 3)), dict(clip=1.0), dict(clip=-0.5), dict(kl=-1.0), dict(kl=float("nan"))):
        with pytest.raises(ValueError):
            pl._check(*{**good, **change}.values())
    with pytest.raises(RuntimeError, match="detach"):
        pl._check(*{**good, "target": _there(2, 3, 4, dtype=f32).requires_grad_(True)}.values())
