"""Timed cases of the attribute network's operators: what a network that maps per-Gaussian features to Gaussian
attributes runs in each training iteration and in each query.

The operators (T is the type of the activations and matrices: float32, float16 or bfloat16; vectors are float32):

  linear               z = x w^T + b, y = act(z) + residual; z is kept for the backward where the case trains
  linear_backward      dz = dy act'(z); dx = dz w, dw = dz^T x, db = the column sums of dz
  layer_norm           y = (x - mean) rstd gamma + beta over each row, and the rows' mean and rstd
  layer_norm_backward  dx (plus the gradient that the residual path brings, where the case has one), dgamma, dbeta
  muon                 m <- mu m + (1 - mu) g, u = mu m + (1 - mu) g, five Newton-Schulz steps on u / |u|, and
                       W <- (1 - lr wd) W - lr sqrt(max(1, rows / cols)) X, with W's copies in T written as well

Fields of a case: kind (one of these), dtype, rows (Gaussians, or queries), features / in_features / out_features,
activation ("none", "relu", "silu", "gelu" with the tanh), residual, train, pad (further columns of the buffers whose
first columns the matrices are: their rows then lie further apart than they are long). muon: width, hidden, blocks
(each an out x in = hidden x width and a width x hidden matrix), inputs and outputs (the first and the last matrix).

`own` False: elementary torch operations in 32 bits, rounded once at the end. `own` True: the package's operators.
"""
import math

import torch

own = False

DEVICE = "cuda"
EPS = 1e-5
MUON = {"lr": 0.02, "momentum": 0.95, "weight_decay": 0.01, "epsilon": 1e-12, "iterations": 5}
# the quintic's coefficients: a x + b x^3 + c x^5 lifts small singular values fast and keeps all near one
NS_A, NS_B, NS_C = 3.4445, -4.7750, 2.0315
# a Gaussian's optimised numbers: mean 3, scale 3, rotation 4, opacity 1, spherical harmonics 48
ATTRIBUTES = 59
# a position with 10 octaves of sines and cosines (63) and a time with 10 (21)
ENCODED = 84
SQRT_2_PI = math.sqrt(2.0 / math.pi)


def _dtype(name):
    return {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}[name]


def _linear(name, dtype, rows, in_features, out_features, activation, residual=False, train=False, pad=0):
    return {"name": name, "kind": "linear", "dtype": dtype, "rows": rows, "in_features": in_features,
            "out_features": out_features, "activation": activation, "residual": residual, "train": train, "pad": pad}


def _linear_backward(name, dtype, rows, in_features, out_features, activation, pad=0):
    return {"name": name, "kind": "linear_backward", "dtype": dtype, "rows": rows, "in_features": in_features,
            "out_features": out_features, "activation": activation, "pad": pad}


def _norm(name, kind, dtype, rows, features, residual=False, pad=0):
    c = {"name": name, "kind": kind, "dtype": dtype, "rows": rows, "features": features, "pad": pad}
    if kind == "layer_norm_backward":
        c["residual"] = residual
    return c


def _muon(name, dtype, width, hidden, blocks, inputs, outputs):
    return {"name": name, "kind": "muon", "dtype": dtype, "width": width, "hidden": hidden, "blocks": blocks,
            "inputs": inputs, "outputs": outputs}


def listed():
    return [
        # one query through a trained network (a time code or a picked Gaussian): latency is all
        _linear("linear-query", "float16", 1, 256, 256, "silu", residual=True),
        # the head of a small full-precision network: encoded positions to a Gaussian's 59 numbers, ragged everywhere
        _linear("linear-head-100k", "float32", 100_003, ENCODED, ATTRIBUTES, "none"),
        # a block's second layer over the million Gaussians of the large scene, in training
        _linear("linear-1m", "bfloat16", 1_000_000, 256, 256, "gelu", residual=True, train=True),
        # the wide first layer of a large network's block, over a chunk of rows
        _linear("linear-wide", "bfloat16", 32_768, 1024, 4096, "gelu", train=True),
        # the gradients of a hidden layer over the million Gaussians
        _linear_backward("linear-backward-1m", "bfloat16", 1_000_000, 256, 256, "gelu"),
        # the gradients of a small full-precision network's first layer, ragged, rows further apart than long
        _linear_backward("linear-backward-50k", "float32", 50_021, ENCODED, 128, "relu", pad=4),
        # the gradients of a wide layer over a chunk of rows, in halves
        _linear_backward("linear-backward-wide", "float16", 16_384, 1024, 2048, "silu"),
        # the norm ahead of each block, over the million Gaussians
        _norm("norm-1m", "layer_norm", "float16", 1_000_000, 256),
        # its gradients, joined with the residual path's
        _norm("norm-backward-1m", "layer_norm_backward", "bfloat16", 1_000_000, 256, residual=True),
        # a small scene in full precision, an odd width
        _norm("norm-backward-6k", "layer_norm_backward", "float32", 6_007, 323),
        # one optimiser step on the matrices of a small half-precision network
        _muon("muon-network", "bfloat16", 256, 256, 4, ENCODED, ATTRIBUTES),
        # and on those of a large one in full precision
        _muon("muon-wide", "float32", 1024, 4096, 2, ENCODED, ATTRIBUTES),
    ]


def _size(rng, low, high):
    """A size between low and high, spread over its logarithm: often a multiple of 16, else as it comes."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if n > 32 and rng.random() < 0.5:
        n -= n % 16
    return max(low, min(high, n))


def draw(rng):
    kind = rng.choice(["linear", "linear_backward", "layer_norm", "layer_norm_backward", "muon"])
    dtype = rng.choice(["float32", "float16", "bfloat16"])
    pad = rng.choice([0, 0, 0, 8, 3])
    if kind == "muon":
        while True:
            c = _muon("", dtype, _size(rng, 16, 1024), _size(rng, 16, 4096), rng.randint(1, 4), _size(rng, 3, 256),
                      _size(rng, 1, 128))
            if work(c)["flops"] <= 6e11:
                break
    elif kind.startswith("layer_norm"):
        while True:
            c = _norm("", kind, dtype, _size(rng, 1, 1 << 20), _size(rng, 8, 8192), rng.random() < 0.5, pad)
            if work(c)["bytes"] <= 2.2e9:
                break
    else:
        while True:
            sizes = (_size(rng, 1, 1 << 20), _size(rng, 1, 4096), _size(rng, 1, 4096))
            activation = rng.choice(["none", "relu", "silu", "gelu"])
            if kind == "linear":
                c = _linear("", dtype, *sizes, activation, rng.random() < 0.5, rng.random() < 0.5, pad)
            else:
                c = _linear_backward("", dtype, *sizes, activation, pad)
            w = work(c)
            if w["bytes"] <= 2.2e9 and w["flops"] <= (7e10 if dtype == "float32" else 2.7e11):
                break
    del c["name"]
    return c


def _matrices(case):
    """The shapes (rows = outputs, columns = inputs) of the network's matrices."""
    block = [(case["hidden"], case["width"]), (case["width"], case["hidden"])]
    return [(case["width"], case["inputs"])] + block * case["blocks"] + [(case["outputs"], case["width"])]


def work(case):
    size = torch.empty(0, dtype=_dtype(case["dtype"])).element_size()
    if case["kind"] == "muon":
        elements = sum(r * c for r, c in _matrices(case))
        # a step: the symmetric x x^T and its square (half of each), the product with x
        flops = 0
        for r, c in _matrices(case):
            m, n = min(r, c), max(r, c)
            flops += MUON["iterations"] * (m * (m + 1) * n + m * (m + 1) * m + 2 * m * m * n)
        # weights and momenta read and written, gradients read, half copies written
        return {"bytes": elements * (16 + size + (size if size == 2 else 0)), "flops": flops}
    rows = case["rows"]
    if case["kind"].startswith("layer_norm"):
        n = case["features"]
        if case["kind"] == "layer_norm":
            return {"bytes": 2 * rows * n * size + 8 * n + 8 * rows, "flops": 8 * rows * n}
        moved = (4 if case["residual"] else 3) * rows * n * size
        return {"bytes": moved + 12 * n + 8 * rows, "flops": 12 * rows * n}
    i, o, z = case["in_features"], case["out_features"], case["activation"] != "none"
    if case["kind"] == "linear":
        moved = rows * i + o * i + rows * o * (1 + case["residual"] + case["train"])
        return {"bytes": moved * size + 4 * o, "flops": 2 * rows * i * o}
    moved = rows * o * (1 + z) + 2 * rows * i + 2 * o * i
    return {"bytes": moved * size + 4 * o, "flops": 4 * rows * i * o}


def _inputs(case, seed):
    """Everything but the derived inputs, from the seed alone."""
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))
    t = _dtype(case["dtype"])

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEVICE)

    def matrix(rows, cols, scale, shift=0.0):
        """The first columns of a buffer whose other columns nothing may touch."""
        pad = case.get("pad", 0)
        return normal(rows, cols + pad).mul_(scale).add_(shift).to(t)[:, :cols]

    s = {"case": case}
    if case["kind"] == "muon":
        shapes = _matrices(case)
        s["weights"] = [normal(r, c).mul_(1.0 / math.sqrt(c)) for r, c in shapes]
        # momenta and gradients of a network in training: a few directions carry most of them
        s["momenta"] = [normal(r, c).mul_(1e-3) + normal(r, 1) * normal(1, c) * 2e-3 for r, c in shapes]
        s["grads"] = [(normal(r, c).mul_(3e-3) + normal(r, 1) * normal(1, c) * 2e-3).to(t) for r, c in shapes]
        s["copies"] = [w.to(t) for w in s["weights"]] if t != torch.float32 else None
        return s
    if case["kind"].startswith("layer_norm"):
        rows, n = case["rows"], case["features"]
        s["x"] = matrix(rows, n, 1.5, 0.25)
        s["gamma"] = 1.0 + 0.2 * normal(n)
        if case["kind"] == "layer_norm":
            s["beta"] = 0.2 * normal(n)
        else:
            s["grad_y"] = matrix(rows, n, 1e-2)
            s["residual_grad"] = matrix(rows, n, 1e-2) if case["residual"] else None
        return s
    rows, i, o = case["rows"], case["in_features"], case["out_features"]
    s["x"] = matrix(rows, i, 1.0)
    s["weight"] = matrix(o, i, 1.0 / math.sqrt(i))
    s["bias"] = 0.3 * normal(o)
    if case["kind"] == "linear":
        s["residual"] = matrix(rows, o, 1.0) if case["residual"] else None
    else:
        s["grad_y"] = matrix(rows, o, 1e-2)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "layer_norm_backward":   # the statistics that the forward left
        x = s["x"].float()
        s["mean"] = x.mean(1)
        s["rstd"] = torch.rsqrt((x - s["mean"][:, None]).square().mean(1) + EPS)
    if case["kind"] == "linear_backward" and case["activation"] != "none":   # and its values before the activation
        z = s["x"].float() @ s["weight"].float().t() + s["bias"]
        s["preact"] = torch.empty(case["rows"], case["out_features"] + case["pad"], dtype=s["x"].dtype,
                                  device=DEVICE)[:, :case["out_features"]]
        s["preact"].copy_(z)
    return s


# ---------------------------------------------------------------- the plain forms

def _act(z, activation):
    if activation == "relu":
        return torch.clamp_min(z, 0.0)
    if activation == "silu":
        return z * torch.sigmoid(z)
    if activation == "gelu":
        return 0.5 * z * (1.0 + torch.tanh(SQRT_2_PI * (z + 0.044715 * z * z * z)))
    return z


def _act_slope(z, activation):
    if activation == "relu":
        return (z > 0.0).to(z.dtype)
    if activation == "silu":
        g = torch.sigmoid(z)
        return g * (1.0 + z * (1.0 - g))
    t = torch.tanh(SQRT_2_PI * (z + 0.044715 * z * z * z))
    return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * (SQRT_2_PI * (1.0 + 0.134145 * z * z))


def _plain_linear(s):
    case = s["case"]
    z = s["x"].float() @ s["weight"].float().t() + s["bias"]
    y = _act(z, case["activation"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    t = s["x"].dtype
    return (y.to(t), z.to(t)) if case["train"] else (y.to(t),)


def _plain_linear_backward(s):
    dz = s["grad_y"].float()
    if s["case"]["activation"] != "none":
        dz = dz * _act_slope(s["preact"].float(), s["case"]["activation"])
    t = s["x"].dtype
    return (dz @ s["weight"].float()).to(t), (dz.t() @ s["x"].float()).to(t), dz.sum(0)


def _plain_layer_norm(s):
    x = s["x"].float()
    mean = x.mean(1)
    d = x - mean[:, None]
    rstd = torch.rsqrt(d.square().mean(1) + EPS)
    return (d * rstd[:, None] * s["gamma"] + s["beta"]).to(s["x"].dtype), mean, rstd


def _plain_layer_norm_backward(s):
    dy = s["grad_y"].float()
    h = (s["x"].float() - s["mean"][:, None]) * s["rstd"][:, None]
    g = dy * s["gamma"]
    dx = s["rstd"][:, None] * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
    if s["residual_grad"] is not None:
        dx = dx + s["residual_grad"].float()
    return dx.to(s["x"].dtype), (dy * h).sum(0), dy.sum(0)


def _plain_muon(s):
    mu, lr = MUON["momentum"], MUON["lr"]
    for k, (w, m, g) in enumerate(zip(s["weights"], s["momenta"], s["grads"])):
        g = g.float() * (1.0 - mu)
        m.mul_(mu).add_(g)
        u = g + mu * m
        x = u / torch.clamp_min(u.square().sum().sqrt(), MUON["epsilon"])
        tall = w.shape[0] > w.shape[1]
        if tall:
            x = x.t()
        for _ in range(MUON["iterations"]):
            a = x @ x.t()
            b = NS_B * a + NS_C * (a @ a)
            x = NS_A * x + b @ x
        if tall:
            x = x.t()
        w.mul_(1.0 - lr * MUON["weight_decay"]).sub_(x, alpha=lr * math.sqrt(max(1.0, w.shape[0] / w.shape[1])))
        if s["copies"] is not None:
            s["copies"][k].copy_(w)
    return s["weights"], s["momenta"], s["copies"]


PLAIN = {"linear": _plain_linear, "linear_backward": _plain_linear_backward, "layer_norm": _plain_layer_norm,
         "layer_norm_backward": _plain_layer_norm_backward, "muon": _plain_muon}


# ---------------------------------------------------------------- the package's operators

_kept = {}


def _layer_ops():
    """The handle that a program makes once and keeps: it owns the operators' workspace."""
    if "ops" not in _kept:
        from tinygs_amd.network import LayerOps
        _kept["ops"] = LayerOps()
    return _kept["ops"]


def _run_own(s):
    case = s["case"]
    if case["kind"] == "muon":
        if "optimizer" not in s:   # made once by a program, as SimpleAdam is, and kept
            from tinygs_amd.optim import Muon
            s["optimizer"] = Muon(s["weights"], s["grads"], momenta=s["momenta"], copies=s["copies"])
            s["optimizer"].set_params(MUON)
        s["optimizer"].step(1.0)
        return s["weights"], s["momenta"], s["copies"]
    ops = _layer_ops()
    if case["kind"] == "linear":
        got = ops.linear(s["x"], s["weight"], s["bias"], activation=case["activation"], residual=s["residual"],
                         keep_preact=case["train"])
        return got if case["train"] else (got,)
    if case["kind"] == "linear_backward":
        return ops.linear_backward(s["grad_y"], s["x"], s["weight"], preact=s.get("preact"),
                                   activation=case["activation"])
    if case["kind"] == "layer_norm":
        return ops.layer_norm(s["x"], s["gamma"], s["beta"], eps=EPS)
    return ops.layer_norm_backward(s["grad_y"], s["x"], s["gamma"], s["mean"], s["rstd"],
                                   residual_grad=s["residual_grad"])


def run(state):
    return _run_own(state) if own else PLAIN[state["case"]["kind"]](state)


# ---------------------------------------------------------------- the definitions in 64 bits

def _exact_activation(z, activation):
    """act(z) and act'(z), from the logistic function: the gelu's 1 + tanh(v) is 2 logistic(2 v)."""
    if activation == "none":
        return z, torch.ones_like(z)
    if activation == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z)), torch.where(z > 0, 1.0, 0.0).to(z.dtype)
    if activation == "silu":
        p = 1.0 / (1.0 + torch.exp(-z))
        return z * p, p + z * p * (1.0 - p)
    v = 2.0 * math.sqrt(2.0 / math.pi) * (z + 0.044715 * z ** 3)
    p = 1.0 / (1.0 + torch.exp(-v))
    return z * p, p + z * p * (1.0 - p) * 2.0 * math.sqrt(2.0 / math.pi) * (1.0 + 3.0 * 0.044715 * z ** 2)


def exact(case, seed):
    s = prepare(case, seed)
    d = torch.float64
    if case["kind"] == "muon":
        weights, momenta = [], []
        for w, m, g in zip(s["weights"], s["momenta"], s["grads"]):
            w, m, g = w.to(d), m.to(d), g.to(d)
            m = MUON["momentum"] * m + (1.0 - MUON["momentum"]) * g
            u = MUON["momentum"] * m + (1.0 - MUON["momentum"]) * g
            x = u / max(float(torch.linalg.norm(u)), MUON["epsilon"])
            for _ in range(MUON["iterations"]):   # a x + b (x x^T) x + c (x x^T)^2 x, by the shorter side's products
                if x.shape[0] <= x.shape[1]:
                    s2 = torch.mm(x, x.t())
                    cubed = torch.mm(s2, x)
                    fifth = torch.mm(s2, cubed)
                else:
                    s2 = torch.mm(x.t(), x)
                    cubed = torch.mm(x, s2)
                    fifth = torch.mm(cubed, s2)
                x = NS_A * x + NS_B * cubed + NS_C * fifth
            shape = math.sqrt(max(1.0, w.shape[0] / w.shape[1]))
            weights.append((1.0 - MUON["lr"] * MUON["weight_decay"]) * w - MUON["lr"] * shape * x)
            momenta.append(m)
        return weights, momenta, weights if s["copies"] is not None else None
    x = s["x"].to(d)
    if case["kind"].startswith("layer_norm"):
        n = case["features"]
        if case["kind"] == "layer_norm":
            mean = x.sum(1, keepdim=True) / n
            var = ((x - mean) ** 2).sum(1, keepdim=True) / n
            rstd = 1.0 / torch.sqrt(var + EPS)
            return (x - mean) * rstd * s["gamma"].to(d) + s["beta"].to(d), mean[:, 0], rstd[:, 0]
        rstd, dy = s["rstd"].to(d)[:, None], s["grad_y"].to(d)
        h = (x - s["mean"].to(d)[:, None]) * rstd
        g = dy * s["gamma"].to(d)
        dx = rstd * (g - g.sum(1, keepdim=True) / n - h * ((g * h).sum(1, keepdim=True) / n))
        if s["residual_grad"] is not None:
            dx = dx + s["residual_grad"].to(d)
        return dx, (dy * h).sum(0), dy.sum(0)
    w = s["weight"].to(d)
    if case["kind"] == "linear":
        z = torch.addmm(s["bias"].to(d), x, w.t())
        y = _exact_activation(z, case["activation"])[0]
        if s["residual"] is not None:
            y = y + s["residual"].to(d)
        return (y, z) if case["train"] else (y,)
    dz = s["grad_y"].to(d)
    if case["activation"] != "none":
        dz = dz * _exact_activation(s["preact"].to(d), case["activation"])[1]
    return torch.mm(dz, w), torch.mm(dz.t(), x), dz.sum(0)
