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
