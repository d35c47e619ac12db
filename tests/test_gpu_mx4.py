"""4-bit rows and their products against a search over all scales and levels in 64 bits."""
import pytest
import torch

import network_refs as refs
from poker2_b200 import mx4

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _same(got, want):
    want = want.to(got.dtype).double()  # (the largest finite magnitude rounds up to 4 * 2^126, which is an infinity in fp32)
    assert torch.equal(torch.isnan(got.double()), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got.double()), torch.nan_to_num(want))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width", [(1, 1), (1, 32), (3, 31), (2, 33), (129, 255), (128, 256), (5, 257), (40, 1300), (300, 2720), (17, 1536)])
def test_quantise_reads_back_as_its_definition(cuda_device, rows, width, dtype):
    g = torch.Generator(device=cuda_device).manual_seed(rows + width)
    x = torch.randn(rows, width, device=cuda_device, generator=g) * torch.exp2(torch.randint(-12, 6, (rows, 1), device=cuda_device, generator=g).float())
    x = x.to(dtype)
    q = mx4.quantise(x)
    assert q.values.shape == (rows, (width + 31) // 32 * 16) and q.shape == (rows, width)
    _same(q.dequantise(), refs.mx4_values(x))
    for to in TYPES[:2]:
        assert torch.equal(q.dequantise(to), refs.mx4_values(x).to(to))


@pytest.mark.parametrize("dtype", TYPES)
def test_borders_and_special_values(cuda_device, dtype):
    """Every border between two levels and its neighbours in the type, at several scales; largest magnitudes at and next to the
    borders between scales; zeros, the smallest and largest numbers, infinities and NaN."""
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0], dtype=torch.float64)
    info = torch.finfo(dtype)
    near = [borders, borders * (1 + info.eps), borders * (1 - info.eps / 2), -borders]
    row = torch.cat(near)  # 32 values, the largest above 6: their block's scale is one power higher
    rows = [row, row.clamp(-6, 6), torch.zeros(32, dtype=torch.float64)]
    for exponent in (-9, 0, 7):
        for top in (1.5, 1.5 * (1 + info.eps), 1.5 * (1 - info.eps), 1.0, 2.0 * (1 - info.eps)):
            block = torch.linspace(-1, 1, 32, dtype=torch.float64) * 2.0 ** exponent
            block[7] = -top * 2.0 ** exponent
            rows.append(block)
    for value in (info.max, info.min, info.tiny, info.smallest_normal / 4, float("inf"), float("-inf"), float("nan")):
        block = torch.ones(32, dtype=torch.float64) * 0.5
        block[31] = value
        rows.append(block)
        rows.append(torch.full((32,), value, dtype=torch.float64))
    x = torch.stack(rows).to(dtype).to(cuda_device)
    _same(mx4.quantise(x).dequantise(), refs.mx4_values(x))
    # the same blocks side by side: nothing of one reaches its neighbours
    wide = x.reshape(1, -1)
    _same(mx4.quantise(wide).dequantise().view(-1, 32), refs.mx4_values(x))


def test_strides_and_shapes(cuda_device):
    x = torch.randn(70, 96, device=cuda_device).bfloat16()
    want = mx4.quantise(x)
    area = torch.zeros(70 * 96 + 1, device=cuda_device, dtype=x.dtype)[1:].view(70, 96).copy_(x)
    wide = torch.randn(70, 200, device=cuda_device).bfloat16()
    wide[:, 3:99] = x
    for other in (area, wide[:, 3:99], x.t().contiguous().t(), x.view(7, 10, 96)):
        q = mx4.quantise(other)
        assert torch.equal(q.values, want.values) and torch.equal(q.scales, want.scales)
        assert q.dequantise(x.dtype).shape == other.shape
    row = mx4.quantise(x[:1].expand(70, 96))
    assert torch.equal(row.values, want.values[:1].expand(70, -1))
    assert mx4.quantise(x[:0]).dequantise().shape == (0, 96)
    assert mx4.quantise(x[0]).dequantise().shape == (96,)
    # a quantised row is left as it is when quantised again
    back = want.dequantise(torch.bfloat16)
    assert torch.equal(mx4.quantise(back).dequantise(torch.bfloat16), back)


@pytest.mark.parametrize("activation", ["none", "gelu", "silu"])
@pytest.mark.parametrize("dtype", TYPES[:2])
@pytest.mark.parametrize("rows,width,columns", [(1, 1536, 1536), (1, 32, 1), (2, 31, 7), (4, 1023, 9), (3, 2720, 130), (4, 1025, 16), (5, 1025, 16), (33, 256, 128), (128, 300, 129), (129, 64, 40),
                                                (200, 2720, 333), (385, 1000, 257), (600, 513, 2652), (3001, 128, 2652), (2800, 64, 1330),
                                                (1700, 300, 1500), (2500, 512, 1031), (5000, 64, 700)])
def test_linear(cuda_device, rows, width, columns, dtype, activation):
    g = torch.Generator(device=cuda_device).manual_seed(rows + width + columns)
    x = torch.randn(rows, width, device=cuda_device, generator=g).to(dtype)
    w = (torch.randn(columns, width, device=cuda_device, generator=g) / width ** 0.5).to(dtype)
    bias = torch.randn(columns, device=cuda_device, generator=g).to(dtype)
    q = mx4.quantise(w)
    want = refs.mx4_linear(refs.mx4_values(x), refs.mx4_values(w), bias, activation, dtype)
    y = mx4.linear(x, q, bias, activation=activation)
    assert y.dtype == dtype and y.shape == (rows, columns)
    refs.assert_within(y, *want)
    general = mx4.linear(mx4.quantise(x), q, bias, activation=activation, dtype=dtype)
    if rows > mx4.FEW_ROWS:
        assert torch.equal(general, y)
    else:  # another order of sums
        refs.assert_within(general, *want)
        fp32 = mx4.linear(x.float(), q, bias, activation=activation, dtype=dtype)
        assert torch.equal(fp32, y)
        assert torch.equal(mx4.linear(x.t().contiguous().t(), q, bias, activation=activation), y)
    if activation == "none":
        refs.assert_within(mx4.linear(x, q), *refs.mx4_linear(refs.mx4_values(x), refs.mx4_values(w), None, activation, dtype))


@pytest.mark.parametrize("activation", ["none", "gelu", "silu"])
@pytest.mark.parametrize("dtype", TYPES[:2])
@pytest.mark.parametrize("rows,width,columns", [(1, 64, 1), (5, 1536, 1536), (33, 256, 100), (128, 300, 129), (129, 64, 40), (300, 520, 256), (385, 1000, 257),
                                                (600, 513, 2652), (1700, 300, 1500), (2500, 512, 1031), (5000, 64, 700), (2400, 96, 1537)])
def test_linear_that_stays_quantised(cuda_device, rows, width, columns, dtype, activation):
    """To the bit what quantising the result gives, scales behind the last row and column included."""
    g = torch.Generator(device=cuda_device).manual_seed(rows + width + columns)
    x = mx4.quantise(torch.randn(rows, width, device=cuda_device, generator=g))
    w = mx4.quantise(torch.randn(columns, width, device=cuda_device, generator=g) / width ** 0.5)
    bias = torch.randn(columns, device=cuda_device, generator=g).to(dtype)
    for b in (bias, None):
        want = mx4.quantise(mx4.linear(x, w, b, activation=activation, dtype=dtype))
        # what was in memory before does not matter
        torch.full((rows * (columns + 300) * 2,), 255, dtype=torch.uint8, device=cuda_device)
        got = mx4.linear(x, w, b, activation=activation, dtype=dtype, quantised=True)
        assert got.shape == (rows, columns) and torch.equal(got.values, want.values) and torch.equal(got.scales, want.scales)
        refs.assert_within(mx4.linear(got, mx4.quantise(torch.ones(3, columns, device=cuda_device))),
                           *refs.mx4_linear(got.dequantise().double(), torch.ones(3, columns, device=cuda_device).double(), None, "none", torch.bfloat16))


def test_linear_that_stays_quantised_shapes_and_bad_rows(cuda_device):
    x, w = torch.randn(140, 96, device=cuda_device), mx4.quantise(torch.randn(50, 96, device=cuda_device))
    assert mx4.linear(x.view(14, 10, 96), w, quantised=True).shape == (14, 10, 50)
    assert mx4.linear(x[0], w, quantised=True).shape == (50,) and mx4.linear(x[:0], w, quantised=True).dequantise().shape == (0, 50)
    x[5, 40] = float("nan")
    bad = mx4.linear(x, w, quantised=True).dequantise()
    assert torch.isnan(bad[5]).all() and torch.isfinite(bad[:5]).all() and torch.isfinite(bad[6:]).all()


def test_linear_types_shapes_and_bad_rows(cuda_device):
    x = torch.randn(140, 96, device=cuda_device)
    q = mx4.quantise(torch.randn(50, 96, device=cuda_device))
    y = mx4.linear(x, q)
    assert y.dtype == torch.bfloat16
    assert mx4.linear(x, q, dtype=torch.float16).dtype == torch.float16
    assert torch.equal(mx4.linear(x.view(14, 10, 96), q), y.view(14, 10, 50))
    assert mx4.linear(x[:0], q).shape == (0, 50) and mx4.linear(x[:4].view(2, 2, 96), q).shape == (2, 2, 50)
    assert torch.equal(mx4.linear(x[0], q), mx4.linear(x[:1], q)[0])
    broken = x[:3].clone()
    broken[1, 3] = float("inf")
    few = mx4.linear(broken, q)
    assert torch.equal(few[[0, 2]], mx4.linear(x[:3], q)[[0, 2]]) and torch.isnan(few[1]).all()
    x[5, 40], x[139, 0] = float("nan"), float("inf")
    bad = mx4.linear(x, q)
    others = torch.ones(140, dtype=torch.bool, device=cuda_device)
    others[[5, 139]] = False
    assert torch.equal(bad[others], y[others]) and torch.isnan(bad[[5, 139]]).all()
    # wide ranges: scales from one end to the other, the sum stays exact where one term carries it
    a = torch.zeros(3, 64, device=cuda_device)
    w = torch.zeros(2, 64, device=cuda_device)
    a[0, 0], a[1, 33], a[2, 40], w[0, 0], w[1, 33], w[1, 40] = 2.0 ** 100, 3.0 * 2.0 ** -100, -1.5, 2.0 ** -90, 2.0 ** 110, 0.5 * 2.0 ** 110
    for rows in (a, a.repeat(3, 1)):
        got = mx4.linear(rows, mx4.quantise(w)).double()[:3]
        assert torch.equal(got, (refs.mx4_values(a) @ refs.mx4_values(w).T).bfloat16().double())


def test_streams_and_capture(cuda_device):
    x = torch.randn(300, 512, device=cuda_device).bfloat16()
    q = mx4.quantise(torch.randn(160, 512, device=cuda_device))
    y = mx4.linear(x, q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        aside = mx4.linear(x, q)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(aside, y)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append((mx4.linear(x, q, activation="silu"), mx4.quantise(x).dequantise(x.dtype)))
        graphs.append(graph)
    x.copy_(torch.randn(300, 512, device=cuda_device))
    graphs[0].replay()
    graphs[1].replay()
    for a, b in outs:
        assert torch.equal(a, mx4.linear(x, q, activation="silu")) and torch.equal(b, mx4.quantise(x).dequantise(x.dtype))


def test_offsets_beyond_32_bits_and_unaligned_biases(cuda_device):
    """1.6 million rows of 1400 values, and as many outputs; the first and last rows against their own call."""
    rows, width = 1_600_000, 1400
    x = torch.randn(rows, width, device=cuda_device, dtype=torch.bfloat16)
    q = mx4.quantise(x)
    back = q.dequantise(torch.bfloat16)
    ends = (slice(0, 200), slice(rows - 200, rows))
    for part in ends:
        assert torch.equal(back[part].double(), refs.mx4_values(x[part]))
    del back
    w = mx4.quantise(torch.randn(1400, width, device=cuda_device) / 37)
    bias = torch.randn(1401, device=cuda_device).bfloat16()[1:]
    y = mx4.linear(q, w, bias, activation="silu")
    for part in ends:
        refs.assert_within(y[part], *refs.mx4_linear(refs.mx4_values(x[part]), w.dequantise().double(), bias, "silu", torch.bfloat16))


def test_threads_and_another_current_device(cuda_device, monkeypatch):
    import threading

    from poker2_b200 import _lib

    x = torch.randn(2000, 512, device=cuda_device).bfloat16()
    q = mx4.quantise(torch.randn(1500, 512, device=cuda_device))
    want, got = mx4.linear(x, q), {}

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[i] = mx4.linear(x, q)
            torch.cuda.current_stream().synchronize()

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    monkeypatch.setattr(_lib, "_get_device", lambda: -1)
    got[2] = mx4.linear(x, q)
    assert all(torch.equal(y, want) for y in got.values()) and torch.equal(mx4.linear(x[:2], q), mx4.linear(x[:2].clone(), q))
