"""Plain 64-bit forms of the network operators, and bounds on how far a kernel may be from them."""
import math

import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}  # of the value
SMALLEST = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}  # half a step below the normal numbers


def activation(z, name):
    if name == "none":
        return z
    return z * 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) if name == "gelu" else z * torch.sigmoid(z)


def slope(z, name):
    if name == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    s = torch.sigmoid(z)
    return s * (1.0 + z * (1.0 - s))


def rounded(value, dtype):
    """How far a rounding to dtype may move each value."""
    return value.abs() * HALF_STEP[dtype] + SMALLEST[dtype]


def summed(magnitudes, terms):
    """Error of a sum of `terms` fp32 terms whose magnitudes add up to `magnitudes`: a step of 2^-23 an addition (the tensor cores
    need not round to nearest), two more for what is added to the sum."""
    return magnitudes * ((terms + 2) * 2.0 ** -23)


def gated(x, wg, wu, bg, bu, name, dtype):
    """(h, bound) in 64 bits; h before its rounding to dtype."""
    x, wg, wu = x.double(), wg.double(), wu.double()
    zero = torch.zeros(wg.shape[0], dtype=torch.float64, device=x.device)
    bg, bu = (zero if b is None else b.double() for b in (bg, bu))
    gate, up = x @ wg.T + bg, x @ wu.T + bu
    mag_g, mag_u = x.abs() @ wg.abs().T + bg.abs(), x.abs() @ wu.abs().T + bu.abs()
    K = x.shape[-1]
    a = activation(gate, name)
    # |act'| <= 1.13; the activation itself: 2^-20 of its argument's size (a handful of fp32 steps); the product's own step
    err_a = 1.13 * summed(mag_g, K) + gate.abs() * 2.0 ** -20
    err = err_a * (up.abs() + summed(mag_u, K)) + a.abs() * summed(mag_u, K) + (a * up).abs() * 2.0 ** -22
    h = a * up
    return h, err + rounded(h.abs() + err, dtype)


def gated_backward(dh, x, wg, wu, bg, bu, name, dtype):
    """{name: (gradient, bound)}: the rounding of dgate and dup, taken at its worst in every term, the fp32 sums, the last rounding."""
    dh, x, wg, wu = dh.double(), x.double(), wg.double(), wu.double()
    zero = torch.zeros(wg.shape[0], dtype=torch.float64, device=x.device)
    bg, bu = (zero if b is None else b.double() for b in (bg, bu))
    gate, up = x @ wg.T + bg, x @ wu.T + bu
    K, F, M = x.shape[-1], wg.shape[0], x.shape[0]
    err_g, err_u = summed(x.abs() @ wg.abs().T + bg.abs(), K), summed(x.abs() @ wu.abs().T + bu.abs(), K)
    a, s = activation(gate, name), slope(gate, name)
    dg, du = dh * up * s, dh * a
    # |act''| <= 0.8, |act'| <= 1.13, functions to 2^-20
    e_dg = dh.abs() * (err_u * s.abs() + (up.abs() + err_u) * (0.8 * err_g + 2.0 ** -20 * (1 + gate.abs())))
    e_du = dh.abs() * (1.13 * err_g + gate.abs() * 2.0 ** -20)
    e_dg, e_du = e_dg + rounded(dg.abs() + e_dg, dtype), e_du + rounded(du.abs() + e_du, dtype)

    def with_bound(value, err, mag, terms):
        err = err + summed(mag + err, terms)
        return value, err + rounded(value.abs() + err, dtype)

    return {
        "dx": with_bound(dg @ wg + du @ wu, e_dg @ wg.abs() + e_du @ wu.abs(), dg.abs() @ wg.abs() + du.abs() @ wu.abs(), 2 * F),
        "dwg": with_bound(dg.T @ x, e_dg.T @ x.abs(), dg.abs().T @ x.abs(), M),
        "dwu": with_bound(du.T @ x, e_du.T @ x.abs(), du.abs().T @ x.abs(), M),
        "dbg": with_bound(dg.sum(0), e_dg.sum(0), dg.abs().sum(0), M),
        "dbu": with_bound(du.sum(0), e_du.sum(0), du.abs().sum(0), M),
    }


def assert_within(got, value, bound, what=""):
    off = (got.double() - value).abs() - bound
    worst = off.max().item() if off.numel() else 0.0
    assert torch.isfinite(got.double()).all(), what
    assert worst <= 0.0, f"{what}: {int((off > 0).sum())} of {off.numel()} outside, worst by {worst:.3g} (bound {bound.flatten()[off.argmax()].item():.3g})"


LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def mx4_values(x):
    """What x [rows, width] reads back as, in 64 bits: every scale from 2^-127 up is tried against the block's largest magnitude,
    every level against the value."""
    x = x.double()
    rows, width = x.shape
    padded = torch.zeros(rows, (width + 31) // 32 * 32, dtype=torch.float64, device=x.device)
    padded[:, :width] = x
    blocks = padded.view(rows, -1, 32)
    top = blocks.abs().amax(dim=-1)
    scales = torch.exp2(torch.arange(-127, 127, dtype=torch.float64, device=x.device))
    scale = scales[torch.searchsorted(6.0 * scales, torch.nan_to_num(top, nan=0.0, posinf=0.0))][..., None]
    levels = torch.tensor(LEVELS, dtype=torch.float64, device=x.device)
    distance = ((blocks.abs() / scale)[..., None] - levels).abs()
    best = distance == distance.amin(dim=-1, keepdim=True)
    even = torch.arange(8, device=x.device) % 2 == 0
    best = torch.where((best.sum(dim=-1, keepdim=True) > 1), best & even, best)
    value = levels[best.int().argmax(dim=-1)] * scale * torch.sign(blocks)
    value = torch.where(torch.isfinite(top)[..., None], value, float("nan"))
    return value.reshape(rows, -1)[:, :width]


def mx4_linear(a, w, bias, name, dtype):
    """(y, bound) of act(a w^T + bias) for matrices of 4-bit values in 64 bits."""
    zero = torch.zeros(w.shape[0], dtype=torch.float64, device=w.device)
    bias = zero if bias is None else bias.double()
    z, mag = a @ w.T + bias, a.abs() @ w.abs().T + bias.abs()
    y = activation(z, name)
    err = 1.13 * summed(mag, a.shape[1]) + z.abs() * 2.0 ** -20
    return y, err + rounded(y.abs() + err, dtype)


def policy_loss(logits, old, adv, target, legal, weights, clip, kl, dtype):
    """(loss, its bound, gradient, its bound) in 64 bits, from the definition."""
    z = logits.double()
    N, H, A = z.shape
    legal = legal[:, None, :].expand(N, H, A)
    w = torch.ones(N, H, dtype=torch.float64, device=z.device) if weights is None else weights.double()
    w = torch.where(legal.any(-1), w, 0.0)
    mass = w.sum()
    z = torch.where(legal, z, -math.inf)
    top = z.amax(-1, keepdim=True)
    counts = (w != 0) & (top[..., 0] != -math.inf)
    legal = legal & counts[..., None]
    d = torch.where(legal, z - torch.where(counts[..., None], top, 0.0), 0.0)
    e = torch.where(legal, torch.exp(d), 0.0)
    total = torch.where(counts, e.sum(-1), 1.0)[..., None]
    p = e / total
    t = torch.where(legal, target.double(), 0.0)
    logp = d - torch.log(total)
    kl_terms = torch.where(t > 0, t * (torch.log(torch.where(t > 0, t, 1.0)) - torch.where(t > 0, logp, 0.0)), 0.0)
    if old is None:
        surr, g = torch.zeros_like(p), torch.zeros_like(p)
    else:
        q, a = torch.where(legal, old.double(), 0.0), torch.where(legal, adv.double(), 0.0)
        low, high = (1.0 - clip) * q, (1.0 + clip) * q
        free = torch.where(a > 0, p <= high, p >= low)
        surr = torch.minimum(p * a, torch.minimum(torch.maximum(p, low), high) * a)
        g = torch.where(free, a, 0.0)
    per_hand = torch.where(counts, kl * kl_terms.sum(-1) - surr.sum(-1), 0.0)
    some = mass > 0
    loss = (w * per_hand).sum() / mass if some else torch.zeros_like(mass)
    scale = (w / mass if some else torch.zeros_like(w))[..., None]
    pull, targets = (g * p).sum(-1, keepdim=True), t.sum(-1, keepdim=True)
    grad = torch.where(legal, scale * (kl * (p * targets - t) - p * (g - pull)), 0.0)
    # fp32 steps u: z - top is off by u |d|, the exponential by 4 u, the sum by A u and its terms' own |d|; log by 4 u of its
    # value and u of the total's error
    u = 2.0 ** -24
    finite = torch.where(torch.isfinite(d), d, 0.0).abs()
    reach = finite.clamp(max=104.0).amax(-1, keepdim=True)
    e_p = u * (finite + reach + A + 16)
    size = kl * (p * targets + t) + p * (g.abs() + (g.abs() * p).sum(-1, keepdim=True))
    err = scale * size * (3 * e_p + (A + 12) * u)
    hand_size = kl * torch.where(t > 0, t * (torch.log(torch.where(t > 0, t, 1.0)).abs() + finite + torch.log(total) + 1), 0.0).sum(-1) + surr.abs().sum(-1)
    hand_err = hand_size * (3 * e_p.amax(-1) + (A + 12) * u)
    loss_err = (w * hand_err).sum() / mass if some else torch.zeros_like(mass)
    return loss, loss_err + loss.abs() * 2 * u + 1e-300, grad, err + rounded(grad.abs() + err, dtype)
