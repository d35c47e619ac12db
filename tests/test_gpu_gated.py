"""The gated hidden layer and its gradients against their formulas in 64 bits."""
import pytest
import torch

from poker2_b200 import _lib, gated
import network_refs as refs

pytestmark = pytest.mark.gpu

SIZES = [  # rows, width, hidden: single tokens, the step to the tensor cores, tiles and blocks just full, one over, odd numbers
    (1, 64, 32), (1, 1536, 1024), (1, 77, 5), (2, 2720, 40), (4, 65, 33), (5, 64, 1), (8, 65, 33), (9, 64, 1), (9, 1, 8), (13, 72, 64), (77, 100, 72),
    (128, 64, 128), (129, 63, 129), (257, 1536, 200), (300, 8, 1024), (700, 2720, 96), (1000, 333, 257),
    (40, 64, 2500), (600, 72, 2100),  # biases beyond what is staged
    (2000, 1536, 1024), (5200, 600, 300),  # several tiles a pair, both kinds of gradients' tiles
]


def _layer(rows, width, hidden, dtype, device, bias=True, seed=0):
    g = torch.Generator(device=device).manual_seed(seed + rows + 7 * width + 31 * hidden)
    new = lambda *s: torch.randn(*s, device=device, generator=g)  # noqa: E731
    x = new(rows, width).to(dtype)
    wg, wu = (new(hidden, width).div(width ** 0.5).to(dtype) for _ in range(2))
    bg, bu = ((new(hidden) * 0.2).to(dtype) for _ in range(2)) if bias else (None, None)
    return x, wg, wu, bg, bu, new(rows, hidden).to(dtype)


@pytest.mark.parametrize("activation", ["gelu", "silu"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", SIZES)
def test_forward(cuda_device, size, dtype, activation):
    x, wg, wu, bg, bu, _ = _layer(*size, dtype, cuda_device)
    h = gated.gated_linear(x, wg, wu, bg, bu, activation=activation)
    assert h.dtype == dtype and h.shape == (size[0], size[2])
    refs.assert_within(h, *refs.gated(x, wg, wu, bg, bu, activation, dtype))


@pytest.mark.parametrize("activation", ["gelu", "silu"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", SIZES)
def test_gradients(cuda_device, size, dtype, activation):
    x, wg, wu, bg, bu, dh = _layer(*size, dtype, cuda_device)
    leaves = [t.clone().requires_grad_(True) for t in (x, wg, wu, bg, bu)]
    h = gated.gated_linear(*leaves, activation=activation)
    got = torch.autograd.grad(h, leaves, dh)
    want = refs.gated_backward(dh, x, wg, wu, bg, bu, activation, dtype)
    for g, leaf, (name, (value, bound)) in zip(got, leaves, want.items()):
        assert g.dtype == dtype and g.shape == leaf.shape
        refs.assert_within(g, value, bound, name)
    again = gated.gated_linear_backward(dh, x, wg, wu, bg, bu, activation=activation)
    for a, b in zip(got, again):
        assert torch.equal(a, b)


def test_gradients_against_differences(cuda_device):
    """Along a random direction v, (L(p + e v) - L(p - e v)) / 2e of the formula in 64 bits; the gradient's own rounding, a half
    step of each value and the two intermediate ones, moves its product with v by no more than the bounds of its values do."""
    x, wg, wu, bg, bu, dh = _layer(40, 96, 50, torch.bfloat16, cuda_device)
    got = gated.gated_linear_backward(dh, x, wg, wu, bg, bu)
    want = refs.gated_backward(dh, x, wg, wu, bg, bu, "gelu", torch.bfloat16)
    params = [t.double() for t in (x, wg, wu, bg, bu)]
    loss = lambda p: (refs.gated(*p, "gelu", torch.bfloat16)[0] * dh.double()).sum()  # noqa: E731
    g = torch.Generator(device=cuda_device).manual_seed(5)
    for i, (name, (_, bound)) in enumerate(want.items()):
        v = torch.randn(params[i].shape, device=cuda_device, generator=g, dtype=torch.float64)
        e = 1e-5
        ahead, back = list(params), list(params)
        ahead[i], back[i] = params[i] + e * v, params[i] - e * v
        difference = ((loss(ahead) - loss(back)) / (2 * e)).item()
        allowed = (bound * v.abs()).sum().item() + 1e-6 * abs(difference) + 1e-6
        assert abs((got[i].double() * v).sum().item() - difference) <= allowed, name


@pytest.mark.parametrize("rows", [3, 200])
def test_strides_offsets_and_shapes(cuda_device, rows):
    """Views at odd offsets, transposed weights, rows of a wider matrix, a broadcast row, more dimensions: as their copies."""
    x, wg, wu, bg, bu, dh = _layer(rows, 80, 48, torch.bfloat16, cuda_device)
    plain = gated.gated_linear(x, wg, wu, bg, bu)
    grads = gated.gated_linear_backward(dh, x, wg, wu, bg, bu)

    def offset(t):
        area = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:]
        return area.view(t.shape).copy_(t)

    wide = torch.randn(rows, 200, device=cuda_device).to(x.dtype)
    wide[:, 16:96] = x
    odd = torch.randn(rows, 203, device=cuda_device).to(x.dtype)
    odd[:, 5:85] = x
    for other in (offset(x), wide[:, 16:96], odd[:, 5:85], x.t().contiguous().t()):
        assert torch.equal(gated.gated_linear(other, offset(wg), wu.t().contiguous().t(), offset(bg), bu), plain)
        for a, b in zip(gated.gated_linear_backward(offset(dh), other, offset(wg), wu, offset(bg), bu), grads):
            assert torch.equal(a, b)
        for a, b in zip(gated.gated_linear_backward(dh.t().contiguous().t(), other, wg, wu, bg, bu), grads):
            assert torch.equal(a, b)
    assert torch.equal(gated.gated_linear(x.view(rows, 1, 80), wg, wu, bg, bu), plain.view(rows, 1, 48))
    one = gated.gated_linear(x[:1].expand(rows, 80), wg, wu, bg, bu)
    assert torch.equal(one, gated.gated_linear(x[:1].repeat(rows, 1), wg, wu, bg, bu))
    nothing = gated.gated_linear(x[:0], wg, wu, bg, bu)
    assert nothing.shape == (0, 48)
    empty = gated.gated_linear_backward(dh[:0], x[:0], wg, wu, bg, bu)
    assert empty[0].shape == (0, 80) and all(not bool(t.any()) for t in empty[1:])
    # a gradient of one value for all (the sum of the outputs) is a broadcast tensor
    leaf = x.clone().requires_grad_(True)
    gated.gated_linear(leaf, wg, wu, bg, bu).sum().backward()
    assert torch.equal(leaf.grad, gated.gated_linear_backward(torch.ones_like(dh), x, wg, wu, bg, bu)[0])


def test_without_biases_and_with_some_gradients(cuda_device):
    x, wg, wu, _, bu, dh = _layer(150, 72, 40, torch.float16, cuda_device)
    refs.assert_within(gated.gated_linear(x, wg, wu), *refs.gated(x, wg, wu, None, None, "gelu", x.dtype))
    refs.assert_within(gated.gated_linear(x, wg, wu, None, bu), *refs.gated(x, wg, wu, None, bu, "gelu", x.dtype))
    want = refs.gated_backward(dh, x, wg, wu, None, bu, "gelu", x.dtype)
    got = gated.gated_linear_backward(dh, x, wg, wu, None, bu, needs=(False, True, False, True, True))
    assert got[0] is None and got[2] is None and got[3] is None
    refs.assert_within(got[1], *want["dwg"])
    refs.assert_within(got[4], *want["dbu"])
    frozen = x.clone().requires_grad_(True)
    dx, = torch.autograd.grad(gated.gated_linear(frozen, wg, wu, None, bu), frozen, dh)
    refs.assert_within(dx, *want["dx"])
    # gate and up weights may be one tensor
    shared = wg.clone().requires_grad_(True)
    both, = torch.autograd.grad(gated.gated_linear(x, shared, shared), shared, dh)
    apart = gated.gated_linear_backward(dh, x, wg, wg)
    assert torch.equal(both, apart[1] + apart[2])


def test_values_that_are_not_finite_stay_in_their_rows(cuda_device):
    x, wg, wu, bg, bu, dh = _layer(140, 72, 40, torch.bfloat16, cuda_device)
    h = gated.gated_linear(x, wg, wu, bg, bu)
    dx = gated.gated_linear_backward(dh, x, wg, wu, bg, bu)[0]
    x[3, 5], x[130, 0] = float("nan"), float("inf")
    bad = gated.gated_linear(x, wg, wu, bg, bu)
    dbad = gated.gated_linear_backward(dh, x, wg, wu, bg, bu)[0]
    others = torch.ones(140, dtype=torch.bool, device=cuda_device)
    others[[3, 130]] = False
    assert torch.equal(bad[others], h[others]) and torch.equal(dbad[others], dx[others])
    assert not torch.isfinite(bad[3]).any() and not torch.isfinite(bad[130]).all()


def test_streams_capture_and_repetition(cuda_device):
    x, wg, wu, bg, bu, dh = _layer(400, 256, 160, torch.bfloat16, cuda_device)
    h, grads = gated.gated_linear(x, wg, wu, bg, bu), gated.gated_linear_backward(dh, x, wg, wu, bg, bu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        aside = gated.gated_linear(x, wg, wu, bg, bu), gated.gated_linear_backward(dh, x, wg, wu, bg, bu)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(aside[0], h) and all(torch.equal(a, b) for a, b in zip(aside[1], grads))
    # two captured steps, replayed in turn on new inputs
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append((gated.gated_linear(x, wg, wu, bg, bu), gated.gated_linear_backward(dh, x, wg, wu, bg, bu)))
        graphs.append(graph)
    x.copy_(torch.randn(400, 256, device=cuda_device).to(x.dtype))
    graphs[1].replay()
    graphs[0].replay()
    want = gated.gated_linear(x, wg, wu, bg, bu), gated.gated_linear_backward(dh, x, wg, wu, bg, bu)
    for got in outs:
        assert torch.equal(got[0], want[0]) and all(torch.equal(a, b) for a, b in zip(got[1], want[1]))


def test_capture_through_autograd_is_refused(cuda_device):
    x, wg, wu, bg, bu, dh = _layer(32, 64, 32, torch.bfloat16, cuda_device)
    wg.requires_grad_(True)
    alive = gated.gated_linear(x, wg, wu, bg, bu)  # an eager graph of the same leaf
    graph = torch.cuda.CUDAGraph()
    refused = None
    with torch.cuda.graph(graph):
        try:
            gated.gated_linear(x, wg, wu, bg, bu)
        except RuntimeError as e:
            refused = str(e)
        with torch.no_grad():
            h = gated.gated_linear(x, wg, wu, bg, bu)
    assert refused and "gated_linear_backward" in refused
    graph.replay()
    assert torch.equal(h, alive.detach())
    assert torch.isfinite(torch.autograd.grad(alive, wg, dh)[0]).all()


def test_outputs_beyond_32_bits(cuda_device):
    """1.6 million rows of 1400 hidden units: 2.2e9 outputs; the first and last rows against their own call."""
    rows, width, hidden = 1_600_000, 64, 1400
    _, wg, wu, bg, bu, _ = _layer(1, width, hidden, torch.bfloat16, cuda_device)
    x = torch.randn(rows, width, device=cuda_device, dtype=torch.bfloat16)
    h = gated.gated_linear(x, wg, wu, bg, bu)
    for part in (slice(0, 300), slice(rows - 300, rows)):
        refs.assert_within(h[part], *refs.gated(x[part], wg, wu, bg, bu, "gelu", x.dtype))
    del h
    dh = torch.randn(rows, hidden, device=cuda_device, dtype=torch.bfloat16)
    dx = gated.gated_linear_backward(dh, x, wg, wu, bg, bu, needs=(True, False, False, False, False))[0]
    for part in (slice(0, 300), slice(rows - 300, rows)):
        refs.assert_within(dx[part], *refs.gated_backward(dh[part], x[part], wg, wu, bg, bu, "gelu", x.dtype)["dx"])


def test_another_current_device_and_two_threads(cuda_device, monkeypatch):
    """The way a call takes when its tensors' device is not the current one (the same device here), and calls from two threads."""
    import threading

    from poker2_b200 import _lib

    x, wg, wu, bg, bu, dh = _layer(300, 256, 160, torch.bfloat16, cuda_device)
    want = gated.gated_linear(x, wg, wu, bg, bu), gated.gated_linear_backward(dh, x, wg, wu, bg, bu)
    got = {}

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[i] = gated.gated_linear(x, wg, wu, bg, bu), gated.gated_linear_backward(dh, x, wg, wu, bg, bu)
            torch.cuda.current_stream().synchronize()

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    monkeypatch.setattr(_lib, "_get_device", lambda: -1)
    got[2] = gated.gated_linear(x, wg, wu, bg, bu), gated.gated_linear_backward(dh, x, wg, wu, bg, bu)
    for h, grads in got.values():
        assert torch.equal(h, want[0]) and all(torch.equal(a, b) for a, b in zip(grads, want[1]))


def test_second_derivatives_are_refused(cuda_device):
    x, wg, wu, bg, bu, dh = _layer(16, 64, 32, torch.bfloat16, cuda_device)
    x.requires_grad_(True)
    with pytest.raises(RuntimeError, match="second"):
        torch.autograd.grad(gated.gated_linear(x, wg, wu, bg, bu), x, dh, create_graph=True)


def test_the_leaf_of_a_broadcast_input_gets_its_sum(cuda_device):
    x, wg, wu, bg, bu, dh = _layer(200, 72, 40, torch.bfloat16, cuda_device)
    row = x[0].clone().requires_grad_(True)
    got, = torch.autograd.grad(gated.gated_linear(row.expand(200, 72), wg, wu, bg, bu), row, dh)
    each = gated.gated_linear_backward(dh, x[:1].expand(200, 72), wg, wu, bg, bu)[0]
    assert torch.equal(got, each.sum(0))


@pytest.mark.parametrize("dtype,activation", [(torch.bfloat16, "gelu"), (torch.float16, "silu")])
@pytest.mark.parametrize("size,keeps", [
    ((8192, 1024, 1024), True), ((8195, 1100, 1000), True), ((20001, 1027, 701), True), ((40, 65536, 4800), True),
    ((8191, 1024, 1024), False), ((9000, 1016, 1024), False), ((512, 16392, 1024), False),
])
def test_what_the_forward_pass_keeps(cuda_device, size, keeps, dtype, activation):
    """Gate and up as the forward pass left them give the bits that the projections taken again give."""
    x, wg, wu, bg, bu, dh = _layer(*size, dtype, cuda_device)
    assert (_lib.lib().p2b_gated_kept_bytes(*size) > 0) == keeps
    if size[0] == 8195:
        leaves = [t.clone().requires_grad_(True) for t in (x, wg, wu, bg, bu)]
        got = torch.autograd.grad(gated.gated_linear(*leaves, activation=activation), leaves, dh)
        for g, (name, (value, bound)) in zip(got, refs.gated_backward(dh, x, wg, wu, bg, bu, activation, dtype).items()):
            refs.assert_within(g, value, bound, name)
    x[2, 1], x[3, 0], dh[1, 0] = float("inf"), float("nan"), float("nan")
    for bias in (True, False):
        plain = (x, wg, wu, bg, bu) if bias else (x, wg, wu)
        leaves = [t.clone().requires_grad_(True) for t in plain]
        h = gated.gated_linear(*leaves, activation=activation)
        assert torch.equal(h.detach().view(torch.int16), gated.gated_linear(*plain, activation=activation).view(torch.int16))
        apart = gated.gated_linear_backward(dh, *plain, activation=activation)
        for _ in range(2):
            for a, b in zip(torch.autograd.grad(h, leaves, dh, retain_graph=True), apart):
                assert torch.equal(a.view(torch.int16), b.view(torch.int16))
        for i, leaf in enumerate(leaves):  # one gradient by itself
            (a,) = torch.autograd.grad(h, [leaf], dh, retain_graph=True)
            assert torch.equal(a.view(torch.int16), apart[i].view(torch.int16))


def test_kept_rows_beyond_one_launch(cuda_device):
    rows, width, hidden = 65535 * 32 + 45, 1024, 5
    x, wg, wu, bg, bu, dh = _layer(rows, width, hidden, torch.bfloat16, cuda_device)
    assert _lib.lib().p2b_gated_kept_bytes(rows, width, hidden) > 1 << 31
    leaves = [t.clone().requires_grad_(True) for t in (wg, wu, bg, bu)]
    got = torch.autograd.grad(gated.gated_linear(x, *leaves), leaves, dh)
    apart = gated.gated_linear_backward(dh, x, wg, wu, bg, bu, needs=(False, True, True, True, True))
    for a, b in zip(got, apart[1:]):
        assert torch.equal(a, b)
