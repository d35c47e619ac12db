"""The network operators of poker2_b200, as cases that can be timed.

A case is a dict of plain values; `kind` says which operator it is:

  gated      the gated hidden layer of a value network, h = act(x Wg^T + bg) * (x Wu^T + bu): `gated.gated_linear`, and with
             `train` its gradients too, as a training step takes them
  quantise   4-bit values with a power-of-two scale for every 32 of a row, written and read back: `mx4.quantise`, `dequantise`
  product    a linear layer on such values, act(q(x) q(W)^T + b), the weights quantised once: `mx4.linear`
  loss       the clipped policy loss with a KL term over the hands of a batch of states, and its gradient:
             `policy_loss.clipped_policy_loss` (`autograd`) or `policy_loss.clipped_policy_loss_and_grad`

With `own` false, `run` computes the same in elementary torch operations, in 32 bits (64 where a value's side of a border decides).
Inputs are synthetic: hidden activations, weights as the framework's networks initialise them, ranges over the combos that a
board leaves, policies with the zeros that regret matching leaves in them.
"""
from __future__ import annotations

import math

import torch

own = False

HANDS = 1326
WIDTH = 1536  # hidden width of the framework's value networks
GATED = 1024  # gate and up projections of that width together hold as many weights as 4/3 of a plain layer
INPUT = 2720  # a network's input row: two ranges, board, pot and stacks, padded
ACTIONS = (5, 8)  # actions a node: the production bet sizes, and those of the configuration dataclasses


def listed():
    return [
        # One leaf asked while a hand is played: a single row through a hidden layer.
        _gated("gated_leaf_1", 1, WIDTH, GATED, "bf16", "gelu"),
        # The leaves of one flop tree, an odd number of them.
        _gated("gated_leaves_77", 77, WIDTH, GATED, "fp16", "silu"),
        # Turn leaves expanded over the 48 river cards: 512 leaves a chunk.
        _gated("gated_chance_24576", 24576, WIDTH, GATED, "bf16", "gelu"),
        # A training step on a minibatch of the replay ring, ragged.
        _gated("gated_train_1000", 1000, WIDTH, GATED, "bf16", "gelu", train=True),
        # The largest minibatch, fp16, the first hidden layer on the network's input rows.
        _gated("gated_train_8192", 8192, INPUT, GATED, "fp16", "silu", train=True),
        # Network input rows of a chunk of turn leaves, quantised as they are written.
        {"name": "mx4_rows_24576", "kind": "quantise", "rows": 24576, "width": INPUT, "dtype": "bf16"},
        # A hidden activation of few leaves, fp32, a width that ends inside a block of 32.
        {"name": "mx4_rows_301", "kind": "quantise", "rows": 301, "width": 1300, "dtype": "fp32"},
        # One leaf through a 4-bit hidden layer.
        _product("mx4_leaf_1", 1, WIDTH, WIDTH, "bf16", "gelu"),
        # A chunk of turn leaves through a 4-bit hidden layer.
        _product("mx4_chance_24576", 24576, WIDTH, WIDTH, "bf16", "gelu"),
        # The output layer on the leaves of the production batch: both players' hand values, no activation.
        _product("mx4_output_3001", 3001, WIDTH, 2 * HANDS, "fp16", "none"),
        # The policy of the root that is being played.
        {"name": "loss_state_1", "kind": "loss", "states": 1, "actions": ACTIONS[0], "dtype": "fp32", "autograd": True},
        # The largest minibatch of the default bet sizes, logits of a bf16 head.
        {"name": "loss_batch_4096", "kind": "loss", "states": 4096, "actions": ACTIONS[1], "dtype": "bf16", "autograd": False},
    ]


def _gated(name, rows, width, hidden, dtype, activation, train=False):
    return {"name": name, "kind": "gated", "rows": rows, "width": width, "hidden": hidden, "dtype": dtype, "activation": activation, "train": train}


def _product(name, rows, width, out, dtype, activation):
    return {"name": name, "kind": "product", "rows": rows, "width": width, "out": out, "dtype": dtype, "activation": activation}


def _log_uniform(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def _size(rng, low, high):
    """Mostly whole groups of 8, as networks have them, and any number one time in four."""
    n = _log_uniform(rng, low, high)
    return n if rng.random() < 0.25 else max(low, (n + 4) // 8 * 8)


def draw(rng):
    kind = rng.choice(["gated", "gated", "quantise", "product", "product", "loss"])
    if kind == "gated":
        train = rng.random() < 0.5
        width, hidden = _size(rng, 64, INPUT), _size(rng, 32, 2048)
        most = min(24576, 24576 * WIDTH * GATED // (width * hidden))
        most = min(8192, 8192 * INPUT * GATED // (width * hidden)) if train else most
        return {"kind": kind, "rows": _log_uniform(rng, 1, most), "width": width, "hidden": hidden, "dtype": rng.choice(["bf16", "fp16"]),
                "activation": rng.choice(["gelu", "silu"]), "train": train}
    if kind == "quantise":
        width = _size(rng, 32, INPUT)
        return {"kind": kind, "rows": _log_uniform(rng, 1, 24576), "width": width, "dtype": rng.choice(["bf16", "fp16", "fp32"] if width <= INPUT // 2 else ["bf16", "fp16"])}
    if kind == "product":
        width, out = _size(rng, 64, INPUT), _size(rng, 32, 2 * HANDS)
        return {"kind": kind, "rows": _log_uniform(rng, 1, min(24576, 24576 * WIDTH * WIDTH // (width * out))), "width": width, "out": out,
                "dtype": rng.choice(["bf16", "fp16"]), "activation": rng.choice(["none", "gelu", "silu"])}
    return {"kind": kind, "states": _log_uniform(rng, 1, 4096), "actions": rng.randint(2, 8), "dtype": rng.choice(["fp32", "bf16"]) if rng.random() < 0.5 else "bf16",
            "autograd": rng.random() < 0.5}


_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CLIP, KL = 0.2, 0.5


def prepare(case, seed):
    device, dtype = torch.device("cuda"), _TYPES[case["dtype"]]
    g = torch.Generator(device=device).manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, device=device, generator=g)  # noqa: E731
    s = {"case": case, "dtype": dtype}
    if case["kind"] == "gated":
        M, K, F = case["rows"], case["width"], case["hidden"]
        s["x"] = normal(M, K).to(dtype)
        s["wg"], s["wu"] = (normal(F, K).div_(K ** 0.5).to(dtype) for _ in range(2))
        s["bg"], s["bu"] = (normal(F).mul_(0.1).to(dtype) for _ in range(2))
        if case["train"]:
            s["dh"] = normal(M, F).mul_(0.5).to(dtype)
            for name in ("x", "wg", "wu", "bg", "bu"):
                s[name].requires_grad_(own)
    elif case["kind"] == "quantise":
        s["x"] = _network_rows(case["rows"], case["width"], g).to(dtype)
    elif case["kind"] == "product":
        M, K, N = case["rows"], case["width"], case["out"]
        s["x"] = normal(M, K).mul_(0.7).clamp_(min=-0.17).to(dtype)  # what an activation leaves: a short side and a long one
        weight = normal(N, K).div_(K ** 0.5).to(dtype)
        s["bias"] = normal(N).mul_(0.1).to(dtype)
        # the weights of a network that serves, laid out once: 4-bit values, or in the plain form what these stand for
        if own:
            from poker2_b200 import mx4

            s["weight"] = mx4.quantise(weight)
        else:
            s["weight"] = _round_to_mx4(weight.float())
    else:
        N, A = case["states"], case["actions"]
        s["logits"] = normal(N, HANDS, A).to(dtype)
        legal = torch.rand(N, A, device=device, generator=g) < 0.8
        legal[:, min(1, A - 1)] = True  # check or call
        if N > 8:
            legal[N // 2] = False  # a finished hand among the sampled states
        open_ = legal[:, None, :].float()
        old = torch.exp(s["logits"].float() + 0.3 * normal(N, HANDS, A)) * open_
        s["old"] = old / old.sum(-1, keepdim=True).clamp(min=1e-30)
        regrets = normal(N, HANDS, A).add_(0.3).clamp_(min=0.0).mul_(open_)
        s["target"] = regrets / regrets.sum(-1, keepdim=True).clamp(min=1e-30)
        s["advantage"] = normal(N, HANDS, A).mul_(0.1)
        board = torch.rand(N, 52, device=device, generator=g).argsort(dim=1)[:, :5]
        c1, c2 = torch.triu_indices(52, 52, 1, device=device)
        dealt = torch.zeros(N, 52, dtype=torch.bool, device=device).scatter_(1, board, True)
        s["hands"] = torch.rand(N, HANDS, device=device, generator=g) * (~(dealt[:, c1] | dealt[:, c2]))
        s["legal"] = legal
        if own and case["autograd"]:
            s["logits"].requires_grad_(True)
    return s


def _network_rows(rows, width, g):
    """Ranges over most of the row (a hand in five blocked), a one-hot board and three fractions at its end."""
    x = torch.empty(rows, width, device=g.device).exponential_(generator=g)
    x *= torch.rand(rows, width, device=g.device, generator=g) < 0.8
    ranges = max(1, width - 55)
    x[:, :ranges] /= x[:, :ranges].sum(dim=1, keepdim=True).clamp(min=1e-12) / 2
    x[:, ranges: ranges + 52] = (torch.rand(rows, x[:, ranges: ranges + 52].shape[1], device=g.device, generator=g) < 0.1).float()
    return x


# ------------------------------------------------------------------ the calls


def run(s):
    kind = s["case"]["kind"]
    if own:
        return _OWN[kind](s)
    return _PLAIN[kind](s)


def _own_gated(s):
    from poker2_b200 import gated

    h = gated.gated_linear(s["x"], s["wg"], s["wu"], s["bg"], s["bu"], activation=s["case"]["activation"])
    if not s["case"]["train"]:
        return {"h": h}
    dx, dwg, dwu, dbg, dbu = torch.autograd.grad(h, (s["x"], s["wg"], s["wu"], s["bg"], s["bu"]), s["dh"])
    return {"h": h, "dx": dx, "dwg": dwg, "dwu": dwu, "dbg": dbg, "dbu": dbu}


def _own_quantise(s):
    from poker2_b200 import mx4

    return mx4.quantise(s["x"]).dequantise(s["dtype"])


def _own_product(s):
    from poker2_b200 import mx4

    return mx4.linear(s["x"], s["weight"], s["bias"], activation=s["case"]["activation"])


def _own_loss(s):
    from poker2_b200 import policy_loss

    call = policy_loss.clipped_policy_loss if s["case"]["autograd"] else policy_loss.clipped_policy_loss_and_grad
    got = call(s["logits"], s["old"], s["advantage"], s["target"], s["legal"], s["hands"], clip=CLIP, kl=KL)
    if s["case"]["autograd"]:
        return {"loss": got, "dlogits": torch.autograd.grad(got, s["logits"])[0]}
    return {"loss": got[0], "dlogits": got[1]}


_OWN = {"gated": _own_gated, "quantise": _own_quantise, "product": _own_product, "loss": _own_loss}


# ------------------------------------------------------------------ the plain forms


def _activation(z, name):
    """act(z) and its derivative."""
    if name == "gelu":
        below = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        return z * below, below + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    s = 1.0 / (1.0 + torch.exp(-z))
    return z * s, s * (1.0 + z * (1.0 - s))


def _plain_gated(s):
    t = s["dtype"]
    x, wg, wu, bg, bu = (s[k].float() for k in ("x", "wg", "wu", "bg", "bu"))
    gate, up = x @ wg.t() + bg, x @ wu.t() + bu
    a, slope = _activation(gate, s["case"]["activation"])
    out = {"h": (a * up).to(t)}
    if s["case"]["train"]:
        dh = s["dh"].float()
        dgate, dup = dh * up * slope, dh * a
        out.update(dx=(dgate @ wg + dup @ wu).to(t), dwg=(dgate.t() @ x).to(t), dwu=(dup.t() @ x).to(t),
                   dbg=dgate.sum(dim=0).to(t), dbu=dup.sum(dim=0).to(t))
    return out


def _round_to_mx4(x):
    """The values that the rows of x (fp32) stand for in 4 bits: in each block of 32, the scale is the smallest power of two that
    brings the largest magnitude to 6 or below; magnitudes then go to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6, ties to
    the one with the even code."""
    rows, width = x.shape
    padded = torch.zeros(rows, (width + 31) // 32 * 32, device=x.device)
    padded[:, :width] = x
    blocks = padded.view(rows, -1, 32)
    mantissa, exponent = torch.frexp(blocks.abs().amax(dim=-1, keepdim=True))
    exponent = torch.where(mantissa <= 0.75, exponent - 3, exponent - 2).clamp(min=-127)
    v = torch.ldexp(blocks.abs(), -exponent)
    code = ((v > 0.25).int() + (v >= 0.75).int() + (v > 1.25).int() + (v >= 1.75).int() + (v > 2.5).int() + (v >= 3.5).int() + (v > 5.0).int())
    level = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=x.device)[code]
    return (torch.ldexp(level, exponent) * torch.sign(blocks)).reshape(rows, -1)[:, :width]


def _plain_quantise(s):
    return _round_to_mx4(s["x"].float()).to(s["dtype"])


def _plain_product(s):
    y = _round_to_mx4(s["x"].float()) @ s["weight"].t() + s["bias"].float()
    name = s["case"]["activation"]
    return (y if name == "none" else _activation(y, name)[0]).to(s["dtype"])


def _plain_loss(s):
    """Per state and hand, over the legal actions: -sum min(p A, clip(p, (1-e) q, (1+e) q) A) + k sum t (log t - log p), with
    p = softmax(logits), q the old policy, t the target; the mean over the hands by their weights."""
    legal = s["legal"][:, None, :]
    any_ = legal.any(dim=-1, keepdim=True)
    # in 64 bits: whether p lies inside the clipped interval decides a gradient
    z = s["logits"].double().masked_fill(~legal, -math.inf)
    z = torch.where(any_, z - z.amax(dim=-1, keepdim=True), 0.0)
    e = torch.exp(z) * legal
    total = e.sum(dim=-1, keepdim=True)
    p = torch.where(any_, e / torch.where(any_, total, 1.0), 0.0)
    old, adv = s["old"].double(), s["advantage"].double()
    free, held = p * adv, torch.minimum(torch.maximum(p, (1.0 - CLIP) * old), (1.0 + CLIP) * old) * adv
    slope = torch.where(free <= held, adv, 0.0).float()
    p, z = p.float(), torch.where(legal, z - torch.log(torch.where(any_, total, 1.0)), 0.0).float()
    target = torch.where(legal, s["target"], 0.0)
    surrogate = torch.where(legal, torch.minimum(free, held), 0.0).float().sum(dim=-1)
    divergence = torch.where(target > 0.0, target * (torch.log(target) - z), 0.0).sum(dim=-1)
    hands = s["hands"] * any_[:, :, 0]
    mass = hands.double().sum()
    loss = (hands * (KL * divergence - surrogate)).double().sum() / mass
    slope = torch.where(legal, slope, 0.0)
    dz = -p * (slope - (slope * p).sum(dim=-1, keepdim=True)) + KL * (p * target.sum(dim=-1, keepdim=True) - target)
    return {"loss": loss.float(), "dlogits": (dz * (hands / mass.float())[:, :, None]).to(s["dtype"])}


_PLAIN = {"gated": _plain_gated, "quantise": _plain_quantise, "product": _plain_product, "loss": _plain_loss}


# ------------------------------------------------------------------ the floor, and the definition in 64 bits


def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
    if case["kind"] == "gated":
        M, K, F = case["rows"], case["width"], case["hidden"]
        once = size * (M * K + 2 * F * K + 2 * F + M * F)  # x, both weights, both biases in, h out
        if not case["train"]:
            return {"bytes": once, "flops": 4 * M * F * K}
        return {"bytes": once + size * (M * F + M * K + 2 * F * K + 2 * F), "flops": 12 * M * F * K}  # dh in, five gradients out
    if case["kind"] == "quantise":
        packed = case["rows"] * ((case["width"] + 31) // 32) * 17  # 16 bytes of values and one of scale a block
        return {"bytes": 2 * size * case["rows"] * case["width"] + 2 * packed, "flops": 0}
    if case["kind"] == "product":
        M, K, N = case["rows"], case["width"], case["out"]
        return {"bytes": size * (M * K + N + M * N) + N * ((K + 31) // 32) * 17, "flops": 2 * M * N * K}
    per_hand = case["actions"] * (2 * size + 12) + 4  # logits in, gradient out, three policies in fp32, the hand's weight
    return {"bytes": case["states"] * (HANDS * per_hand + case["actions"]), "flops": 0}


def exact(case, seed):
    s = prepare(case, seed)
    return {"gated": _exact_gated, "quantise": _exact_quantise, "product": _exact_product, "loss": _exact_loss}[case["kind"]](s)


def _exact_act(z, name):
    if name == "none":
        return z
    return torch.nn.functional.gelu(z) if name == "gelu" else z * torch.sigmoid(z)


def _exact_gated(s):
    leaves = [s[k].detach().double().requires_grad_(s["case"]["train"]) for k in ("x", "wg", "wu", "bg", "bu")]
    x, wg, wu, bg, bu = leaves
    h = _exact_act(torch.nn.functional.linear(x, wg, bg), s["case"]["activation"]) * torch.nn.functional.linear(x, wu, bu)
    if not s["case"]["train"]:
        return {"h": h}
    dx, dwg, dwu, dbg, dbu = torch.autograd.grad(h, leaves, s["dh"].double())
    return {"h": h.detach(), "dx": dx, "dwg": dwg, "dwu": dwu, "dbg": dbg, "dbu": dbu}


def _exact_values(x):
    """Rounded in steps of the value's own binade: halves below 2, ones below 4, twos up to 6."""
    x = x.double()
    parts = []
    for block in x.split(32, dim=1):
        top = block.abs().amax(dim=1, keepdim=True)
        scale = torch.exp2(torch.ceil(torch.log2(torch.where(top > 0, top, 1.0) / 6.0)).clamp(min=-127.0))
        scale = torch.where(scale * 3.0 >= top, scale / 2.0, scale)  # (a logarithm that came out a hair too large)
        v = block / scale
        step = torch.where(v.abs() < 2.0, 0.5, torch.where(v.abs() < 4.0, 1.0, 2.0))
        parts.append(torch.where(top > 0, torch.round(v / step) * step * scale, 0.0))
    return torch.cat(parts, dim=1)


def _exact_quantise(s):
    return _exact_values(s["x"])


def _exact_product(s):
    return _exact_act(torch.nn.functional.linear(_exact_values(s["x"]), s["weight"].double(), s["bias"].double()), s["case"]["activation"])


def _exact_loss(s):
    logits = s["logits"].detach().double().requires_grad_(True)
    legal = s["legal"][:, None, :].expand_as(logits)
    states = s["legal"].any(dim=1)
    logp = torch.log_softmax(logits[states].masked_fill(~legal[states], -1e300), dim=-1)
    ratio_p, old, adv, target = logp.exp(), s["old"][states].double(), s["advantage"][states].double(), s["target"][states].double()
    surrogate = torch.minimum(ratio_p * adv, torch.clamp(ratio_p, min=old * (1 - CLIP), max=old * (1 + CLIP)) * adv)
    kl = torch.special.xlogy(target, target) - target * logp
    per_hand = ((KL * kl - surrogate) * legal[states]).sum(dim=-1)
    hands = s["hands"][states].double()
    loss = (per_hand * hands).sum() / hands.sum()
    return {"loss": loss.detach(), "dlogits": torch.autograd.grad(loss, logits)[0]}
