"""Attention, head norms and clipping in 64 bits, with bounds on what float products, sums and exponentials may be off.

A sum of k products in float is off by at most (k + 17) 2^-24 of the sum of the terms' sizes (network_reference). An
exponential of a float argument is off by the argument's error and 4 units; the argument s - top (or s - lse) by its
terms' roundings, 4 2^-24 of their sizes. A running maximum is replaced at most once a tile of states: the factors that
carry the sums over are off by 2 units each, their arguments by what the telescoping differences add to. Weights and
their gradients are rounded once to 16-bit types ahead of a product: half a unit, or half the smallest step.
"""
import math

import torch

from network_reference import EPS24, STEP, UNIT, check, product_bound, stored  # noqa: F401

F64 = torch.float64


def split(x, batch, heads):
    """[batch, heads, rows, d] in 64 bits."""
    x = x.double().cpu()
    return x.reshape(batch, x.shape[0] // batch, heads, -1).transpose(1, 2)


def join(x):
    return x.transpose(1, 2).reshape(x.shape[0] * x.shape[2], -1)


def shared(x, times):
    return x.repeat_interleave(times, dim=1)


def unite(x, times):
    b, h, n, d = x.shape
    return x.reshape(b, h // times, times, n, d).sum(2)


class Scores:
    """s, its error, and the weights that exist."""

    def __init__(self, q, k, v, heads, kv_heads, batch, mask, scale):
        self.t = heads // kv_heads
        self.q = split(q, batch, heads)
        self.d = self.q.shape[3]
        self.scale = 1.0 / math.sqrt(self.d) if scale is None else scale
        k, v = split(k, batch, kv_heads), split(v, batch, kv_heads)
        self.n = k.shape[2]
        self.exists = torch.ones(batch, 1, 1, self.n, dtype=torch.bool)
        if mask is not None:
            self.exists = (mask.cpu() != 0)[:, None, None, :]
            gone = ~self.exists.transpose(2, 3)
            k, v = k.masked_fill(gone, 0.0), v.masked_fill(gone, 0.0)
        self.k, self.v = shared(k, self.t), shared(v, self.t)
        self.s = (self.q @ self.k.transpose(2, 3)) * self.scale
        self.off = self.scale * (self.d + 17) * EPS24 * (self.q.abs() @ self.k.abs().transpose(2, 3)) + 4 * EPS24 * self.s.abs()
        self.s = self.s.masked_fill(~self.exists, -math.inf)


def attention(q, k, v, heads, kv_heads, batch=1, mask=None, scale=None):
    """(out, bound), (lse [rows, heads], bound)."""
    a = Scores(q, k, v, heads, kv_heads, batch, mask, scale)
    dtype = q.dtype
    if a.n == 0:
        zero = torch.zeros(join(a.q).shape, dtype=F64)
        lse = torch.full((q.shape[0], heads), -math.inf, dtype=F64)
        return (zero, zero), (lse, torch.zeros_like(lse))
    top = a.s.amax(3, keepdim=True)
    lse = torch.logsumexp(a.s, 3, keepdim=True)
    dead = top == -math.inf
    top, safe = top.masked_fill(dead, 0.0), lse.masked_fill(dead, 0.0)
    w = torch.exp(a.s - safe).masked_fill(a.s == -math.inf, 0.0)
    out = w @ a.v
    tiles = (a.n + 31) // 32
    size = a.s.masked_fill(~a.exists, 0.0).abs()
    reach = size.amax(3, keepdim=True)
    e = a.off + 4 * EPS24 * (size + 2 * reach + 1.0) + 2 * tiles * EPS24
    mean_e = (w * e).sum(3, keepdim=True)
    u = 0.0 if dtype == torch.float32 else UNIT[dtype]
    bound = (w * (e + u)) @ a.v.abs() * 1.01 + out.abs() * mean_e * 1.01
    bound = bound + (a.n + 20) * EPS24 * (w @ a.v.abs() + out.abs())
    if dtype == torch.float16:   # weights below the type's normal range, in units of the largest
        bound = bound + STEP[dtype] * a.v.abs().sum(2, keepdim=True)
    lse_bound = 1.01 * mean_e + (a.n + 20) * EPS24 + 4 * EPS24 * (safe.abs() + reach)
    out, bound = join(out), join(bound)
    return (out, stored(out, bound, dtype)), (join(lse), join(lse_bound))


def attention_backward(go, q, k, v, out, lse, heads, kv_heads, batch=1, mask=None, scale=None):
    """(grad_q, bound), (grad_k, bound), (grad_v, bound) of the given out and lse."""
    a = Scores(q, k, v, heads, kv_heads, batch, mask, scale)
    dtype = q.dtype
    go, o = split(go, batch, heads), split(out, batch, heads)
    lse = split(lse, batch, heads)
    dead = lse == -math.inf
    safe = lse.masked_fill(dead, 0.0)
    p = torch.exp(a.s - safe).masked_fill((a.s == -math.inf) | dead, 0.0)
    size = a.s.masked_fill(~a.exists, 0.0).abs()
    e = a.off + 4 * EPS24 * (size + safe.abs() + 1.0)
    delta = (go * o).sum(3, keepdim=True)
    dp = go @ a.v.transpose(2, 3)
    off = (a.d + 17) * EPS24 * (go.abs() @ a.v.abs().transpose(2, 3) + (go * o).abs().sum(3, keepdim=True))
    off = off + 2 * EPS24 * (dp.abs() + delta.abs())
    ds = p * (dp - delta)
    eds = 1.01 * p * (e * (dp - delta).abs() + off) + 2 * EPS24 * ds.abs()
    ep = 1.01 * p * e
    if dtype != torch.float32:
        eds = eds + UNIT[dtype] * (ds.abs() + eds) + STEP[dtype] * a.exists
        ep = ep + UNIT[dtype] * (p + ep) + STEP[dtype] * a.exists
    n, rows = a.n, a.q.shape[2] * a.t

    def product(x, ex, y, depth, times=1.0):
        value, bound = x @ y, ex @ y.abs() + (depth + 20) * EPS24 * (x.abs() @ y.abs())
        return value * times, bound * times * (1 + 4 * EPS24) + 2 * EPS24 * (value * times).abs()

    gq, gqb = product(ds, eds, a.k, n, a.scale)
    gk, gkb = product(ds.transpose(2, 3), eds.transpose(2, 3), a.q, rows, a.scale)
    gv, gvb = product(p.transpose(2, 3), ep.transpose(2, 3), go, rows)
    sums = [(gq, gqb)] + [(unite(x, a.t), unite(y, a.t)) for x, y in ((gk, gkb), (gv, gvb))]
    return [(join(x), stored(join(x), join(y), dtype)) for x, y in sums]


def turned(u, positions, frequencies, sign):
    """u [rows, heads, d], and what turning leaves it off by: a sine and cosine are off by 4 2^-24 (the angle in
    turns is rounded to half a unit of a half, their own two units), the products and the sum by 2."""
    if positions is None:
        return u, torch.zeros_like(u)
    n = 2 * frequencies.shape[0]
    angle = (positions.double().cpu() @ frequencies.double().cpu().t())[:, None, :]
    c, s = torch.cos(angle), sign * torch.sin(angle)
    x, y = u[..., 0:n:2], u[..., 1:n:2]
    out, off = u.clone(), torch.zeros_like(u)
    out[..., 0:n:2], out[..., 1:n:2] = x * c - y * s, x * s + y * c
    e = 6 * EPS24 * (x.abs() + y.abs())
    off[..., 0:n:2], off[..., 1:n:2] = e, e
    return out, off


def _pairs(u, frequencies):
    """The sizes that an element's error is relative to: its own, and its pair's where it is turned."""
    a = u.abs()
    if frequencies is None:
        return a
    n = 2 * frequencies.shape[0]
    a = a.clone()
    both = a[..., 0:n:2] + a[..., 1:n:2]
    a[..., 0:n:2], a[..., 1:n:2] = both, both
    return a


def head_norm(x, heads, gamma, positions, frequencies, eps):
    dtype = x.dtype
    x = x.double().cpu().reshape(x.shape[0], heads, -1)
    d = x.shape[2]
    g = torch.ones(d, dtype=F64) if gamma is None else gamma.double().cpu()
    r = 1.0 / torch.sqrt((x * x).mean(2, keepdim=True) + eps)
    u = x * r * g
    y, off = turned(u, positions, frequencies, 1.0)
    # the sum of squares is off by (d + 4) units, its root by half of that and the division's and products' own
    bound = 1.01 * off + (0.5 * d + 10) * EPS24 * _pairs(u, frequencies)
    y, bound = (t.reshape(t.shape[0], -1) for t in (y, bound))
    return y, stored(y, bound, dtype)


def head_norm_backward(gy, x, heads, gamma, positions, frequencies, eps):
    dtype = x.dtype
    x = x.double().cpu().reshape(x.shape[0], heads, -1)
    gy = gy.double().cpu().reshape(x.shape)
    d = x.shape[2]
    gm = torch.ones(d, dtype=F64) if gamma is None else gamma.double().cpu()
    r = 1.0 / torch.sqrt((x * x).mean(2, keepdim=True) + eps)
    er = (0.5 * d + 6) * EPS24
    h = x * r
    g, eg = turned(gy, positions, frequencies, -1.0)
    gg, egg = g * gm, (eg + EPS24 * g.abs()) * gm.abs()
    dot = (gg * h).mean(2, keepdim=True)
    edot = (egg * h.abs()).mean(2, keepdim=True) + ((d + 6) * EPS24 + er) * (gg * h).abs().mean(2, keepdim=True)
    dx = r * (gg - h * dot)
    bound = r * (egg + h.abs() * edot + (2 * er + 6 * EPS24) * ((h * dot).abs() + gg.abs())) * 1.01
    n = x.shape[0] * heads
    dg = (g * h).sum((0, 1))
    gbound = (eg * h.abs()).sum((0, 1)) * 1.01 + ((n + 8) * EPS24 + er) * (g * h).abs().sum((0, 1)) + STEP[torch.float32]
    dx, bound = (t.reshape(t.shape[0], -1) for t in (dx, bound))
    return (dx, stored(dx, bound, dtype)), (dg, gbound)
