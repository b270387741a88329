"""The attribute network's operators in 64 bits, with bounds on what float products and sums may be off.

A sum of k products formed in float in any order is off by at most (k + 1) 2^-24 of the sum of the terms' sizes; 16
more terms cover products of split operands. A stored element is rounded once: half a unit of its type's last place.
"""
import numpy as np
import torch

EPS24 = 2.0 ** -24
# half a unit in the last place, and the smallest step (subnormals), of each type
UNIT = {torch.float32: EPS24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
STEP = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}
ACTIVATIONS = ("none", "relu", "silu", "gelu")
C0 = float(np.sqrt(2.0 / np.pi))


def act(z, name):
    if name == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if name == "silu":
        return z / (1.0 + torch.exp(-z))
    if name == "gelu":
        return 0.5 * z * (1.0 + torch.tanh(C0 * (z + 0.044715 * z ** 3)))
    return z


def act_slope(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "silu":
        p = 1.0 / (1.0 + torch.exp(-z))
        return p * (1.0 + z * (1.0 - p))
    if name == "gelu":
        t = torch.tanh(C0 * (z + 0.044715 * z ** 3))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * C0 * (1.0 + 3 * 0.044715 * z ** 2)
    return torch.ones_like(z)


# An activation or slope formed in float is off by a few units of its own size and by the argument's rounding, whose
# effect is at most |z| p (1 - p) |argument| 2^-24 < 4 2^-24: 16 2^-24 (|value| + 1) covers both.
ACT_ERROR = 16 * EPS24


def product_bound(a, b, k):
    """What a float product a b of depth k may be off, elementwise (a, b in 64 bits)."""
    return (k + 17) * EPS24 * (a.abs() @ b.abs())


def stored(value, bound, dtype):
    """The bound of an element whose float value is off by `bound` and which is then rounded to dtype."""
    return bound + UNIT[dtype] * (value.abs() + bound) + STEP[dtype]


def check(got, want, bound, what):
    d = (got.double().cpu() - want).abs()
    bad = ~(d <= bound)
    assert not bad.any(), (what, int(bad.sum()), float((d / bound.clamp_min(1e-300)).max()))


def linear(x, w, b, name, residual, dtype):
    """y, z and their bounds."""
    x, w = x.double().cpu(), w.double().cpu()
    z = x @ w.t()
    bound = product_bound(x, w.t(), x.shape[1])
    if b is not None:
        z = z + b.double().cpu()
        bound = bound + 2 * EPS24 * b.double().cpu().abs() + EPS24 * z.abs()
    y = act(z, name)
    # the activations' slopes lie within 1.13
    ybound = 1.13 * bound + (ACT_ERROR * (y.abs() + 1.0) if name in ("silu", "gelu") else 0.0)
    if residual is not None:
        r = residual.double().cpu()
        y = y + r
        ybound = ybound + EPS24 * (y.abs() + ybound)
    return y, stored(y, ybound, dtype), z, stored(z, bound, dtype)


def linear_backward(gy, x, w, z, name, dtype):
    gy, x, w = gy.double().cpu(), x.double().cpu(), w.double().cpu()
    dz, off = gy, torch.zeros_like(gy)
    if name != "none":
        slope = act_slope(z.double().cpu(), name)
        dz = gy * slope
        off = gy.abs() * (ACT_ERROR * (slope.abs() + 1.0) if name != "relu" else 0.0) + EPS24 * dz.abs()
    rounded = off + (UNIT[dtype] * dz.abs() + STEP[dtype] if name != "none" and dtype != torch.float32 else 0.0)
    gx = dz @ w
    gxb = product_bound(dz, w, w.shape[0]) + 1.01 * (rounded @ w.abs())
    gw = dz.t() @ x
    gwb = product_bound(dz.t(), x, x.shape[0]) + 1.01 * (rounded.t() @ x.abs())
    gb = dz.sum(0)
    gbb = (x.shape[0] + 1) * EPS24 * dz.abs().sum(0) + 1.01 * off.sum(0) + STEP[torch.float32]
    return (gx, stored(gx, gxb, dtype)), (gw, stored(gw, gwb, dtype)), (gb, gbb)


def layer_norm(x, gamma, beta, eps, dtype):
    x = x.double().cpu()
    n = x.shape[1]
    one, zero = torch.ones(n, dtype=torch.float64), torch.zeros(n, dtype=torch.float64)
    g = one if gamma is None else gamma.double().cpu()
    b = zero if beta is None else beta.double().cpu()
    mean = x.mean(1)
    d = x - mean[:, None]
    var = (d * d).mean(1)
    rstd = 1.0 / torch.sqrt(var + eps)
    y = d * rstd[:, None] * g + b
    # the mean's sum; the variance's, from differences off by the mean's error m: var + m^2 + its rounding
    m = (n + 2) * EPS24 * x.abs().mean(1)
    v = (n + 8) * EPS24 * var + m * m + 2 * EPS24 * x.abs().amax(1) * torch.sqrt(var)
    rel = 0.5 * v / (var + eps) + 8 * EPS24
    rel = torch.where(rel < 0.25, 1.5 * rel, torch.full_like(rel, torch.inf))
    dy = (m[:, None] + EPS24 * (d.abs() + m[:, None])) * rstd[:, None] * (1.0 + rel[:, None])
    dy = (dy + d.abs() * rstd[:, None] * rel[:, None] + 2 * EPS24 * d.abs() * rstd[:, None]) * g.abs()
    dy = dy + 2 * EPS24 * (y.abs() + b.abs())
    return (y, stored(y, dy, dtype)), (mean, m + STEP[torch.float32]), (rstd, rel * rstd)


def layer_norm_backward(gy, x, gamma, mean, rstd, residual, dtype):
    """Of the given mean and rstd, which are inputs."""
    gy, x, mean, rstd = (t.double().cpu() for t in (gy, x, mean, rstd))
    n, rows = x.shape[1], x.shape[0]
    gm = torch.ones(n, dtype=torch.float64) if gamma is None else gamma.double().cpu()
    h = (x - mean[:, None]) * rstd[:, None]
    hb = 3 * EPS24 * h.abs()
    g = gy * gm
    c1, c2 = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    c1b = (n + 4) * EPS24 * g.abs().mean(1, keepdim=True)
    c2b = (n + 8) * EPS24 * (g * h).abs().mean(1, keepdim=True)
    inner = g - c1 - h * c2
    innerb = EPS24 * 4 * (g.abs() + c1.abs() + (h * c2).abs()) + c1b + h.abs() * c2b + hb * c2.abs()
    gx = inner * rstd[:, None]
    gxb = innerb * rstd[:, None] * (1 + EPS24) + EPS24 * gx.abs()
    if residual is not None:
        gx = gx + residual.double().cpu()
        gxb = gxb + EPS24 * (gx.abs() + gxb)
    gg, gb = (gy * h).sum(0), gy.sum(0)
    ggb = (rows + 5) * EPS24 * (gy * h).abs().sum(0) + STEP[torch.float32]
    gbb = (rows + 1) * EPS24 * gy.abs().sum(0) + STEP[torch.float32]
    return (gx, stored(gx, gxb, dtype)), (gg, ggb), (gb, gbb)


def muon(w, m, g, p, scale=1.0):
    """The updated weights and momentum, and the update's X, of one matrix."""
    w, m, g = w.double().cpu(), m.double().cpu(), g.double().cpu() * scale
    mu = p["momentum"]
    m = mu * m + (1 - mu) * g
    u = (1 - mu) * g + mu * m if p["nesterov"] else m
    x = u / max(float(u.norm()), p["epsilon"])
    tall = w.shape[0] > w.shape[1]
    x = x.t() if tall else x
    for _ in range(p["iterations"]):
        a = x @ x.t()
        x = 3.4445 * x + (-4.7750 * a + 2.0315 * (a @ a)) @ x
    x = x.t() if tall else x
    step = p["lr"] * np.sqrt(max(1.0, w.shape[0] / w.shape[1]))
    return (1 - p["lr"] * p["weight_decay"]) * w - step * x, m, x
