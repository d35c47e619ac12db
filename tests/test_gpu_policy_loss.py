"""The clipped policy loss and its gradient against the definition in 64 bits."""
import pytest
import torch

import network_refs as refs
from poker2_b200 import policy_loss as pl

pytestmark = pytest.mark.gpu
SIZES = [(1, 1326, 5), (1, 1, 1), (3, 1326, 8), (7, 100, 2), (40, 7, 3), (2, 256, 4), (5, 1326, 7), (300, 1, 6), (17, 300, 16), (9, 511, 11),
         (6, 256, 4), (1537, 1, 3), (1201, 1326, 2), (700, 1326, 5)]  # one block's work just full, one over; blocks that take many tiles


def _batch(states, hands, actions, dtype, device, seed=0):
    g = torch.Generator(device=device).manual_seed(seed + states + 31 * hands + 7 * actions)
    new = lambda *s: torch.randn(*s, device=device, generator=g)  # noqa: E731
    logits = (2.0 * new(states, hands, actions)).to(dtype)
    legal = torch.rand(states, actions, device=device, generator=g) < 0.7
    legal[:, 0] = True
    if states > 4:
        legal[3] = False
    old = torch.softmax(logits.float() + 0.3 * new(states, hands, actions), -1)
    target = (new(states, hands, actions) + 0.3).clamp(min=0.0)
    target = target / target.sum(-1, keepdim=True).clamp(min=1e-6)
    adv = 0.2 * new(states, hands, actions)
    weights = torch.rand(states, hands, device=device, generator=g)
    if hands > 2:
        weights[:, ::3] = 0.0
    return logits, old, adv, target, legal, weights


def _check(batch, clip, kl, dtype, grad_only=False):
    loss, grad = pl.clipped_policy_loss_and_grad(*batch, clip=clip, kl=kl)
    want = refs.policy_loss(*batch, clip, kl, dtype)
    assert loss.dtype == torch.float32 and loss.shape == () and grad.dtype == dtype
    if not grad_only:
        refs.assert_within(loss, want[0], want[1], "loss")
    refs.assert_within(grad, want[2], want[3], "gradient")
    return loss, grad


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", SIZES)
def test_loss_and_gradient(cuda_device, size, dtype):
    batch = _batch(*size, dtype, cuda_device)
    loss, grad = _check(batch, 0.2, 0.5, dtype)
    again = pl.clipped_policy_loss_and_grad(*batch, clip=0.2, kl=0.5)
    assert torch.equal(again[0], loss) and torch.equal(again[1], grad)
    assert torch.equal(pl.clipped_policy_loss(*batch, clip=0.2, kl=0.5), loss)
    leaf = batch[0].clone().requires_grad_(True)
    value = pl.clipped_policy_loss(leaf, *batch[1:], clip=0.2, kl=0.5)
    assert torch.equal(value.detach(), loss)
    got, = torch.autograd.grad(value, leaf, retain_graph=True)
    assert torch.equal(got, grad)
    doubled, = torch.autograd.grad(2.0 * value, leaf)  # (exact: a power of two)
    assert torch.equal(doubled, grad * 2)


@pytest.mark.parametrize("clip,kl", [(0.0, 0.0), (0.0, 1.0), (0.3, 0.0), (0.99, 2.0)])
def test_settings(cuda_device, clip, kl):
    batch = _batch(6, 200, 5, torch.float32, cuda_device, seed=3)
    _check(batch, clip, kl, torch.float32)
    logits, old, adv, target, legal, weights = batch
    _check((logits, old, adv, target, legal, None), clip, kl, torch.float32)
    _check((logits, None, None, target, legal, weights), clip, kl, torch.float32)


def test_the_side_of_a_border_is_the_exact_one(cuda_device):
    """Probabilities exactly on, and a step or less than a step of fp32 beside, both ends of the clipped interval."""
    A, clip = 4, 0.2
    logits = torch.zeros(2, 600, A, device=cuda_device)
    logits[1] = torch.randn(600, A, device=cuda_device)
    p = torch.softmax(logits.double(), -1)
    steps = torch.arange(600, device=cuda_device)[None, :, None] % 9 - 4
    end = torch.where(torch.arange(600, device=cuda_device)[None, :, None] % 2 == 0, 1.0 - clip, 1.0 + clip)
    old = (p / end).float()
    old = old * (1.0 + steps * 2.0 ** -24)
    adv = torch.randn(2, 600, A, device=cuda_device).sign() * 0.5
    target = torch.full((2, 600, A), 0.25, device=cuda_device)
    legal = torch.ones(2, A, dtype=torch.bool, device=cuda_device)
    _check((logits, old, adv, target, legal, None), clip, 0.1, torch.float32)


def test_what_is_masked_adds_nothing(cuda_device):
    batch = _batch(6, 60, 5, torch.float32, cuda_device, seed=9)
    logits, old, adv, target, legal, weights = batch
    legal[:, 2] = False
    loss, grad = pl.clipped_policy_loss_and_grad(*batch)
    for bad in (float("nan"), float("inf"), float("-inf"), torch.finfo(torch.float32).min):
        dirty = [t.clone() for t in batch]
        for t in dirty[:4]:
            t[:, :, 2] = bad  # an illegal action
            t[:, ::3] = bad  # hands of weight 0
            t[3] = bad  # a state without a legal action
        got = pl.clipped_policy_loss_and_grad(*dirty)
        assert torch.equal(got[0], loss) and torch.equal(got[1], grad)
    assert not grad[:, :, 2].any() and not grad[:, ::3].any() and not grad[3].any()
    # hands whose legal logits are all -inf add no loss and count in the mean; one -inf is a probability of zero
    empty = logits.clone()
    empty[0, 1] = float("-inf")
    empty[1, 2, 0] = float("-inf")
    old[1, 2, 0] = target[1, 2, 0] = 0.0
    _check((empty, old, adv, target, legal, weights), 0.2, 1.0, torch.float32)
    # the type's lowest value at a legal action is a probability of zero too
    low = logits.clone()
    low[1, 2, 0] = torch.finfo(torch.float32).min
    target[1, 2, 0] = 0.0
    _check((low, old, adv, target, legal, weights), 0.2, 1.0, torch.float32)


def test_nothing_to_average(cuda_device):
    logits, old, adv, target, legal, weights = _batch(6, 60, 5, torch.float32, cuda_device)
    for other in ((logits, old, adv, target, torch.zeros_like(legal), weights), (logits, old, adv, target, legal, torch.zeros_like(weights))):
        loss, grad = pl.clipped_policy_loss_and_grad(*other)
        assert loss.item() == 0.0 and not grad.any()
    loss, grad = pl.clipped_policy_loss_and_grad(logits[:0], old[:0], adv[:0], target[:0], legal[:0], weights[:0])
    assert loss.item() == 0.0 and grad.shape == (0, 60, 5)


def test_extreme_logits(cuda_device):
    logits, old, adv, target, legal, weights = _batch(6, 60, 5, torch.float32, cuda_device)
    _check((logits * 40, old, adv, target, legal, weights), 0.2, 1.0, torch.float32)
    _check((logits + 1e4, old, adv, target, legal, weights), 0.2, 1.0, torch.float32)
    _check((logits * 1e-30, old * 0, adv, target, legal, weights * 1e-20), 0.2, 1.0, torch.float32)


def test_gradient_against_differences(cuda_device):
    """Along random directions, (L(z + e v) - L(z - e v)) / 2e of the definition in 64 bits.  The loss has kinks where p crosses an end of the
    interval; hands with one within reach of the step are given no weight."""
    logits, old, adv, target, legal, weights = _batch(5, 300, 6, torch.float32, cuda_device, seed=2)
    legal[3] = True
    e = 1e-6
    p = torch.softmax(torch.where(legal[:, None, :], logits.double(), -1e30), -1)
    near = ((p / old.double() - 0.8).abs() < 1e-4) | ((p / old.double() - 1.2).abs() < 1e-4)
    weights = torch.where(near.any(-1), 0.0, weights)
    _, grad = pl.clipped_policy_loss_and_grad(logits, old, adv, target, legal, weights)
    bound = refs.policy_loss(logits, old, adv, target, legal, weights, 0.2, 1.0, torch.float32)[3]
    loss = lambda z: refs.policy_loss(z, old, adv, target, legal, weights, 0.2, 1.0, torch.float32)[0].item()  # noqa: E731
    g = torch.Generator(device=cuda_device).manual_seed(4)
    for _ in range(4):
        v = torch.randn(logits.shape, device=cuda_device, dtype=torch.float64, generator=g)
        difference = (loss(logits.double() + e * v) - loss(logits.double() - e * v)) / (2 * e)
        # the difference itself: third derivatives (below 10 each way, |v|^3 e^2) and 64-bit cancellation (1e-16 / e)
        allowed = (bound * v.abs()).sum().item() + 1e-8
        assert abs((grad.double() * v).sum().item() - difference) <= allowed


def test_strides_offsets_streams_and_capture(cuda_device):
    batch = _batch(20, 300, 5, torch.bfloat16, cuda_device)
    want = pl.clipped_policy_loss_and_grad(*batch)
    same = lambda got, to=want: torch.equal(got[0], to[0]) and torch.equal(got[1], to[1])  # noqa: E731
    swapped = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in batch[:4]]
    assert same(pl.clipped_policy_loss_and_grad(*swapped, *batch[4:]))
    shifted = [torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape).copy_(t) for t in batch]
    assert same(pl.clipped_policy_loss_and_grad(*shifted))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        aside = pl.clipped_policy_loss_and_grad(*batch)
    torch.cuda.current_stream().wait_stream(side)
    assert same(aside)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(pl.clipped_policy_loss_and_grad(*batch))
        graphs.append(graph)
    batch[0].mul_(0.5)
    graphs[0].replay()
    graphs[1].replay()
    graphs[0].replay()
    now = pl.clipped_policy_loss_and_grad(*batch)
    assert same(outs[0], now) and same(outs[1], now) and not same(now)
    leaf = batch[0].clone().requires_grad_(True)
    alive = pl.clipped_policy_loss(leaf, *batch[1:])
    refused = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        try:
            pl.clipped_policy_loss(leaf, *batch[1:])
        except RuntimeError as e:
            refused = str(e)
        inside = pl.clipped_policy_loss(leaf.detach(), *batch[1:])
    graph.replay()
    assert refused and "clipped_policy_loss_and_grad" in refused and torch.equal(inside, alive.detach())


def test_hand_weights(cuda_device):
    n = 9
    g = torch.Generator(device=cuda_device).manual_seed(1)
    board = torch.full((n, 5), -1, dtype=torch.int64, device=cuda_device)
    board[1:] = torch.rand(n - 1, 52, device=cuda_device, generator=g).argsort(1)[:, :5]
    board[2, 4] = -1
    beliefs = torch.rand(n, 2 * 1326, device=cuda_device, generator=g)
    to_act = torch.arange(n, device=cuda_device) % 2
    got = pl.hand_weights(beliefs, to_act, board)
    c1, c2 = torch.triu_indices(52, 52, 1, device=cuda_device)
    apart = ((c1[:, None] != c1) & (c1[:, None] != c2) & (c2[:, None] != c1) & (c2[:, None] != c2)).double()
    ranges = beliefs.double().view(n, 2, 1326)
    rows = torch.arange(n, device=cuda_device)
    want = ranges[rows, to_act] * (ranges[rows, 1 - to_act] @ apart)
    for i in range(n):
        for card in board[i].tolist():
            want[i, (c1 == card) | (c2 == card)] = 0.0
    # the mass is summed in 64 bits and rounded, and rounded again by the product
    refs.assert_within(got, want, want * 2.0 ** -22)


def test_arrays_beyond_32_bits(cuda_device):
    """105,000 states of 1326 hands and 16 actions, 2.2e9 entries: every state the same, so loss and gradients are those of one."""
    states, A = 105_000, 16
    g = torch.Generator(device=cuda_device).manual_seed(8)
    one = torch.randn(1, 1326, A, device=cuda_device, generator=g)
    policy = torch.softmax(torch.randn(1, 1326, A, device=cuda_device, generator=g), -1)
    legal = torch.ones(1, A, dtype=torch.bool, device=cuda_device)
    logits, many = one.bfloat16().repeat(states, 1, 1), policy.repeat(states, 1, 1)
    loss, grad = pl.clipped_policy_loss_and_grad(logits, many, many, many, legal.expand(states, A))
    want = refs.policy_loss(one.bfloat16(), policy, policy, policy, legal, None, 0.2, 1.0, torch.float32)
    refs.assert_within(loss, want[0], want[1])
    for part in (0, states // 2, states - 1):
        value = want[2] / states
        refs.assert_within(grad[part: part + 1], value, want[3] / states + refs.rounded(value.abs() * 1.001, torch.bfloat16))


@pytest.mark.parametrize("size", [(5, 100, 4), (3, 77, 5), (400, 1326, 3)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_second_derivatives_are_refused_and_factors_scale(cuda_device, size, dtype):
    logits, *rest = _batch(*size, dtype, cuda_device)
    logits.requires_grad_(True)
    with pytest.raises(RuntimeError, match="second"):
        torch.autograd.grad(pl.clipped_policy_loss(logits, *rest), logits, create_graph=True)
    plain, = torch.autograd.grad(pl.clipped_policy_loss(logits, *rest), logits)
    scaled, = torch.autograd.grad(0.3 * pl.clipped_policy_loss(logits, *rest), logits)
    assert torch.equal(scaled, (plain.float() * torch.tensor(0.3, device=cuda_device)).to(dtype))
