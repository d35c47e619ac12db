"""The network operators together, as a training and serving loop uses them: networks of them behind the leaf evaluators, and a round
of search, replay, policy training and 4-bit serving."""
from types import SimpleNamespace

import pytest
import torch

import network_refs as refs
from poker2_b200 import chance, evaluator, gated, leaf_eval, mx4, policy_loss, tree as ptree, upstream_adapter as ua
from poker2_b200.replay import ReplayRing

pytestmark = pytest.mark.gpu


def _leaves(device, leaves=11, cards=4, seed=1):
    g = torch.Generator(device=device).manual_seed(seed)
    boards = torch.rand(leaves, 52, device=device, generator=g).argsort(dim=1)[:, :5]
    boards[:, cards:] = -1
    beliefs = torch.zeros(leaves, 2, 1344, device=device)
    beliefs[..., :1326] = torch.rand(leaves, 2, 1326, device=device, generator=g)
    beliefs /= beliefs.sum(-1, keepdim=True)
    return boards, beliefs, torch.rand(leaves, 3, device=device, generator=g)


def _plain_block(block, x):
    """GatedBlock in 64 bits, rounded to bf16 where its layers round."""
    n = block.norm(x)
    h = refs.gated(n, block.gate_weight.detach(), block.up_weight.detach(), block.gate_bias.detach(), block.up_bias.detach(), block.activation, x.dtype)[0]
    return x + block.down(h.to(x.dtype))


def test_gated_network_is_its_layers(cuda_device):
    net = leaf_eval.GatedValueMLP(128, 3, hidden=80, seed=2).to(cuda_device)
    boards, beliefs, context = _leaves(cuda_device)
    with torch.no_grad():
        got = net(beliefs[..., :1326], boards, context)
        x = torch.zeros(11, net.IN_PADDED, device=cuda_device, dtype=torch.bfloat16)
        x[:, :2652] = beliefs[..., :1326].reshape(11, -1)
        x[:, 2652:2704] = (boards[:, :, None] == torch.arange(52, device=cuda_device)).any(1)
        x[:, 2704:2707] = context
        y = torch.nn.functional.gelu(net.net[0](x))
        for block in list(net.net)[2:-1]:
            y = _plain_block(block, y)
        want = net.net[-1](y)[:, :2652].float().view(11, 2, 1326)
    # two layers whose bf16 inputs may differ by a step (2^-7 of a value) in places
    assert (got - want).norm() <= 2.0 ** -7 * want.norm()


@pytest.mark.parametrize("make", [lambda: leaf_eval.GatedValueMLP(96, 3, seed=3), lambda: leaf_eval.Mx4ValueMLP(leaf_eval.ValueMLP(96, 2, seed=4).cuda())])
@pytest.mark.parametrize("averaged", [False, True])
def test_leaf_evaluators_take_the_networks_on_their_short_paths(cuda_device, make, averaged):
    """The evaluators' own input rows and output reading against the network called on beliefs, boards and context."""
    net = make().to(cuda_device)
    boards, beliefs, context = _leaves(cuda_device)
    calls = []
    other = lambda b, c, x: (calls.append(b.shape[0]), net(b, c, x))[1]  # noqa: E731
    kind = leaf_eval.ChanceLeafEvaluator if averaged else leaf_eval.DirectLeafEvaluator
    short, plain = kind(net, boards, context, cuda_device), kind(other, boards, context, cuda_device)
    assert short.fused if averaged else short._direct()
    got, want = torch.zeros_like(beliefs), torch.zeros_like(beliefs)
    short.evaluate_into(beliefs, got)
    plain.evaluate_into(beliefs, want)
    assert calls
    if averaged:
        assert (got - want).norm() <= 2.0 ** -7 * want.norm()
    else:
        assert torch.equal(got[..., :1326], want[..., :1326])
    graph = torch.cuda.CUDAGraph()
    again = torch.zeros_like(beliefs)
    with torch.cuda.graph(graph):
        short.evaluate_into(beliefs, again)
    graph.replay()
    assert torch.equal(again, got)


def test_quantised_network_is_its_layers(cuda_device):
    source = leaf_eval.ValueMLP(96, 2, seed=5).to(cuda_device)
    net = leaf_eval.Mx4ValueMLP(source)
    boards, beliefs, context = _leaves(cuda_device, leaves=40)
    x = torch.randn(40, net.IN_PADDED, device=cuda_device).bfloat16()
    got, y = net.net(x), x
    layers = [m for m in source.net if isinstance(m, torch.nn.Linear)]
    assert all(isinstance(net.net[0](x[:r]), torch.Tensor) == (r <= mx4.FEW_ROWS) for r in (1, 4, 5, 40))
    for i, m in enumerate(layers):
        last = i + 1 == len(layers)
        a = mx4.linear(y, net.net[i].weight, net.net[i].bias, activation="none" if last else "gelu")
        refs.assert_within(a, *refs.mx4_linear(refs.mx4_values(y), refs.mx4_values(m.weight.detach()), m.bias.detach(), "none" if last else "gelu", y.dtype))
        y = a
    assert torch.equal(got, y)
    assert torch.equal(net(beliefs[..., :1326], boards, context), net(beliefs[..., :1326], boards, context))
    # the copy stays what it was when the source trains on
    with torch.no_grad():
        source.net[0].weight.zero_()
    assert torch.equal(net.net(x), got)
    for bad in (leaf_eval.GatedValueMLP(96, 2).to(cuda_device), leaf_eval.ValueMLP(96, 1, dtype=torch.float32).to(cuda_device), source.net):
        with pytest.raises((ValueError, AttributeError)):
            leaf_eval.Mx4ValueMLP(bad)
    odd = leaf_eval.ValueMLP(96, 1).to(cuda_device)
    odd.net = torch.nn.Sequential(odd.net[0], torch.nn.SiLU(), odd.net[2])
    with pytest.raises(ValueError):
        leaf_eval.Mx4ValueMLP(odd)


def _head(x, params):
    """A policy head on bf16 rows: a gated layer and a linear one, [n, 1326, A] logits."""
    from poker2_b200 import gated

    h = gated.gated_linear(x, *params[:4], activation="silu")
    return torch.nn.functional.linear(h, params[4]).view(x.shape[0], 1326, -1)


def test_a_round_of_search_training_and_serving(cuda_device):
    """Turn subgames valued by a gated network -> the data generator's policy batch -> the replay ring -> a minibatch's loss through
    gated layers, its gradients against 64 bits -> a step -> the value network served in 4 bits in the next search."""
    g = torch.Generator().manual_seed(3)
    boards = torch.stack([torch.randperm(52, generator=g)[:5] for _ in range(3)])
    boards[:, 4] = -1
    ranges = torch.rand(3, 2, 1326, generator=g)
    c1, c2 = torch.triu_indices(52, 52, 1)
    dealt = torch.zeros(3, 53, dtype=torch.bool).scatter_(1, torch.where(boards >= 0, boards, 52), True)
    ranges *= ~(dealt[:, c1] | dealt[:, c2])[:, None, :]
    ranges /= ranges.sum(-1, keepdim=True)
    roots = ptree.root_states(torch.tensor([40, 90, 150]).numpy(), torch.tensor([300, 200, 500]).numpy(), min_raise=2, street=2)
    env = evaluator.env_view(roots, boards.numpy())

    def search(model):
        ev = evaluator.SubgameEvaluator(cuda_device, iterations=6, max_depth=5, max_raises=2, generator=torch.Generator().manual_seed(0), model=model,
                                        chance_average=False)
        ev.initialize_subgame(env, torch.arange(3), ranges)
        ev.evaluate_cfr()
        return ev.training_data()[2]

    batch = search(leaf_eval.GatedValueMLP(64, 2, seed=6).to(cuda_device))
    n, A = batch.policy_targets.shape[0], batch.policy_targets.shape[2]
    st = batch.statistics
    view = ua.FeatureView(torch.zeros(n, 4, device=cuda_device), torch.full((n,), 2, device=cuda_device), st["to_act"].to(cuda_device), st["board"].to(cuda_device), batch.beliefs)
    ring = ReplayRing(64, A, 2, 4, cuda_device, value_targets=False, generator=torch.Generator(device=cuda_device).manual_seed(1))
    ring.add_batch(ua.RebelBatchLike(view, batch.legal_masks, policy_targets=batch.policy_targets))
    sample = ring.sample(min(24, len(ring)))
    m = len(sample)

    x = (sample.features.beliefs * 100).bfloat16()
    new = torch.Generator(device=cuda_device).manual_seed(2)
    params = [torch.randn(*s, device=cuda_device, generator=new).mul_(k).bfloat16().requires_grad_(True)
              for s, k in (((48, 2652), 0.3), ((48, 2652), 0.3), ((48,), 0.1), ((48,), 0.1), ((1326 * A, 48), 0.1))]
    logits = _head(x, params)
    loss = sample.policy_loss(logits)
    grads = torch.autograd.grad(loss, params)

    weights = policy_loss.hand_weights(sample.features.beliefs, sample.features.to_act, sample.features.board)
    assert (weights > 0).any(1).all()
    want, bound, dlogits, dbound = refs.policy_loss(logits.detach(), None, None, sample.policy_targets, sample.legal_masks, weights, 0.2, 1.0, torch.bfloat16)
    refs.assert_within(loss.detach(), want, bound)
    # the gradients that the layers hand on: each rounds once, the gated layer's inner ones once more
    grad_h = (dlogits.bfloat16().view(m, -1).double() @ params[4].detach().double()).bfloat16()
    inner = refs.gated_backward(grad_h, x, *(p.detach() for p in params[:4]), "silu", torch.bfloat16)
    for got, name in zip(grads, ("dwg", "dwu", "dbg", "dbu")):
        assert (got.double() - inner[name][0]).norm() <= 4 * 2.0 ** -8 * inner[name][0].norm(), name
    # with an old policy and advantages the clipped term joins in: zero advantages leave the KL term alone
    old = torch.softmax(logits.detach().float(), -1)
    assert torch.equal(sample.policy_loss(logits.detach(), old, torch.zeros_like(old)), loss.detach())
    with torch.no_grad():
        for p, d in zip(params, grads):
            p.sub_(0.01 * d)
    assert torch.isfinite(sample.policy_loss(_head(x, params)))

    served = search(leaf_eval.Mx4ValueMLP(leaf_eval.ValueMLP(64, 2, seed=6).to(cuda_device)))
    assert served.policy_targets.shape == batch.policy_targets.shape and torch.isfinite(served.policy_targets).all()


def test_gated_network_trains_through_autograd(cuda_device):
    net = leaf_eval.GatedValueMLP(96, 3, hidden=64, seed=7).to(cuda_device)
    x = torch.randn(50, net.IN_PADDED, device=cuda_device).bfloat16()
    net.net(x).float().square().mean().backward()
    for name, p in net.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad.double()).all() and bool(p.grad.any()), name


def test_policy_loss_of_batches_without_rows_or_targets(cuda_device):
    none = torch.zeros(0, 1326, 5, device=cuda_device)
    view = ua.FeatureView(torch.zeros(0, 4, device=cuda_device), *(torch.zeros(0, dtype=torch.long, device=cuda_device) for _ in range(2)),
                          torch.zeros(0, 5, dtype=torch.long, device=cuda_device), torch.zeros(0, 2652, device=cuda_device))
    legal = torch.zeros(0, 5, dtype=torch.bool, device=cuda_device)
    assert ua.RebelBatchLike(view, legal, policy_targets=none).policy_loss(none.clone().requires_grad_(True)).item() == 0.0
    with pytest.raises(ValueError, match="targets"):
        ua.RebelBatchLike(view, legal).policy_loss(none)


def test_threads_that_have_made_no_call_yet(cuda_device):
    """A thread's first call finds memory in the allocator's cache, so that no call of the runtime has gone before the operator's."""
    import threading

    x, dh = (torch.randn(300, 256, device=cuda_device).bfloat16() for _ in range(2))
    wg, wu = (torch.randn(256, 256, device=cuda_device).div(16).bfloat16() for _ in range(2))
    rows, weight = mx4.quantise(x), mx4.quantise(wg)
    weights, state = torch.rand(3, 1326, device=cuda_device), [torch.randn(3, 1326, 4, device=cuda_device) for _ in range(4)]
    calls = {
        "gated_linear": lambda: gated.gated_linear(x, wg, wu), "few rows": lambda: gated.gated_linear(x[:2], wg, wu),
        "gated_linear_backward": lambda: torch.cat(gated.gated_linear_backward(dh, x, wg, wu)[:3]),
        "linear": lambda: mx4.linear(rows, weight), "linear of rows": lambda: mx4.linear(x, weight), "few": lambda: mx4.linear(x[:2], weight),
        "quantised": lambda: mx4.linear(rows, weight, quantised=True).values, "quantise": lambda: mx4.quantise(x).values,
        "dequantise": lambda: rows.dequantise(),
        "loss": lambda: policy_loss.clipped_policy_loss_and_grad(*[state[0], state[1].softmax(-1), state[2], state[3].softmax(-1)],
                                                                torch.ones(3, 4, dtype=torch.bool, device=cuda_device), weights)[1],
    }
    for name, call in calls.items():
        want, got = call().clone(), {}
        call()

        def work():
            try:
                got["value"] = call()
            except RuntimeError as error:
                got["value"] = str(error)

        torch.cuda.synchronize()
        thread = threading.Thread(target=work)
        thread.start()
        thread.join()
        torch.cuda.synchronize()
        assert not isinstance(got["value"], str), (name, got["value"])
        assert torch.equal(got["value"], want), name
