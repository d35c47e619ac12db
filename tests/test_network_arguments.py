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
    a = dict(x=p, xs=64, wg=p, gs=64, wu=p, us=64, bg=None, bu=None, rows=16, width=64, hidden=8, dtype=0, act=0, h=p, hs=8)
    a.update(change)
    return [*a.values(), None]


def _gated_backward(p, **change):
    a = dict(dh=p, ds=8, x=p, xs=64, wg=p, gs=64, wu=p, us=64, bg=None, bu=None, rows=16, width=64, hidden=8, dtype=0, act=0, dx=p, dxs=64,
             dwg=None, dwu=None, dbg=None, dbu=None, scratch=p, size=1 << 30)
    a.update(change)
    return [*a.values(), None]


LAYER = [dict(rows=-1), dict(rows=1 << 40), dict(width=0), dict(width=1 << 24), dict(hidden=0), dict(hidden=-3), dict(dtype=2), dict(dtype=-1),
         dict(act=2), dict(x=None), dict(wg=None), dict(wu=None), dict(xs=63), dict(gs=8), dict(us=0), dict(rows=1 << 29, hidden=1 << 19)]


@pytest.mark.parametrize("change", LAYER + [dict(h=None), dict(hs=7), dict(xs=65), dict(gs=68), dict(us=66)])
def test_gated_forward_refuses(handle, change):
    area, p = _area()
    assert handle.p2b_gated_forward(*_gated_forward(p, **change)) == -1 and b"p2b_gated_forward" in handle.p2b_last_error()


@pytest.mark.parametrize("change", LAYER + [dict(dh=None), dict(ds=7), dict(dxs=63), dict(scratch=None), dict(size=100), dict(xs=68), dict(us=65)])
def test_gated_backward_refuses(handle, change):
    area, p = _area()
    assert handle.p2b_gated_backward(*_gated_backward(p, **change)) == -1 and b"p2b_gated_backward" in handle.p2b_last_error()


def test_gated_addresses_off_their_boundaries_are_refused(handle):
    area, p = _area()
    for name in ("x", "wg", "wu"):
        assert handle.p2b_gated_forward(*_gated_forward(p, **{name: p + 2})) == -1 and b"16-byte" in handle.p2b_last_error()
        assert handle.p2b_gated_backward(*_gated_backward(p, **{name: p + 8})) == -1 and b"16-byte" in handle.p2b_last_error()
    assert handle.p2b_gated_backward(*_gated_backward(p, scratch=p + 4)) == -1
    assert handle.p2b_gated_forward(*_gated_forward(None, rows=0, wg=p, wu=p)) == 0  # no rows: nothing to do
    assert handle.p2b_gated_backward_scratch_bytes(-1, 8) == -1 and handle.p2b_gated_backward_scratch_bytes(8, 0) == -1


def test_gated_linear_wants_the_gpu():
    x, w = torch.zeros(2, 8, dtype=torch.bfloat16), torch.zeros(4, 8, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        gated.gated_linear(x, w, w)


class _Elsewhere(torch.Tensor):
    """A CPU tensor that says it lies on a GPU, for the checks that come before any launch."""

    @property
    def device(self):
        return torch.device("cuda:0")


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
