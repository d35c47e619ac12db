"""Edges of the network operators: values that are not finite, types at the end of their range, networks that are saved and moved."""
import pytest
import torch

from poker2_b200 import mx4

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
