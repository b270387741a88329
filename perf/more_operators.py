"""Timed cases of the operators by which an attribute network attends to an encoder's states, and of its gradients' norm:
what such a network runs in each training iteration and in each query, next to its linear layers, norms and optimiser.

The operators (T is the type of the activations: float32, float16 or bfloat16; vectors are float32; d is the width of a
head; row r of a matrix holds its heads one after the other):

  attention            s = scale q k^T for each head over the states that the mask leaves, p = softmax(s), o = p v, and
                       lse = log sum exp s where the case trains. Heads may share keys and values in equal groups.
  attention_backward   delta = the sum of do o; dv = p^T do, ds = p (do v^T - delta), dq = scale ds k, dk = scale ds^T q
  head_norm            h = x / sqrt(mean x^2 + eps) over each head, u = h gamma; then the pairs (2i, 2i + 1) of u are
                       turned by the angle positions . frequencies[i]
  head_norm_backward   dx and dgamma of it
  clip                 norm = scale sqrt(sum of squares) over all tensors, g <- g scale min(1, bound / (norm + eps)),
                       in place or into tensors of another type

Fields of a case: kind (one of these), dtype; queries and states (of each element of the batch), batch, heads, kv_heads,
head (d), masked (the least number of states that an element of the batch keeps; all where it equals states), train,
pad (further columns of the buffers whose first columns the matrices are). head_norm: rows, heads, head, axes (0: no
turning), pairs, extent (of the positions), gamma, pad. clip: what the gradients belong to ("network" with width, hidden,
blocks, inputs, outputs; "gaussians" with their number), ratio (the bound over the norm), scale, apart (clipped float32
gradients next to the given ones, instead of in their place).

`own` False: elementary torch operations in 32 bits (angles and the norm in 64), rounded once at the end. `own` True: the
package's operators.
"""
import math

import torch

own = False

DEVICE = "cuda"
EPS = 1e-6
# a Gaussian's optimised numbers: mean 3, scale 3, rotation 4, opacity 1, spherical harmonics 3 + 45
GAUSSIAN = (3, 3, 4, 1, 3, 45)
ATTRIBUTES = 59
# a position with 10 octaves of sines and cosines (63) and a time with 10 (21)
ENCODED = 84


def _dtype(name):
    return {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}[name]


def _attention(name, kind, dtype, batch, queries, states, heads, kv_heads, head, masked=None, train=False, pad=0):
    c = {"name": name, "kind": kind, "dtype": dtype, "batch": batch, "queries": queries, "states": states,
         "heads": heads, "kv_heads": kv_heads, "head": head, "masked": states if masked is None else masked, "pad": pad}
    if kind == "attention":
        c["train"] = train
    return c


def _norm(name, kind, dtype, rows, heads, head, axes, pairs=None, extent=8.0, gamma=True, pad=0):
    return {"name": name, "kind": kind, "dtype": dtype, "rows": rows, "heads": heads, "head": head, "axes": axes,
            "pairs": (head // 2 if pairs is None else pairs) if axes else 0, "extent": extent, "gamma": gamma, "pad": pad}


def _clip_network(name, dtype, width, hidden, blocks, ratio, scale=1.0, apart=False):
    return {"name": name, "kind": "clip", "of": "network", "dtype": dtype, "width": width, "hidden": hidden,
            "blocks": blocks, "inputs": ENCODED, "outputs": ATTRIBUTES, "ratio": ratio, "scale": scale, "apart": apart}


def _clip_gaussians(name, number, ratio, scale=1.0):
    return {"name": name, "kind": "clip", "of": "gaussians", "dtype": "float32", "number": number, "ratio": ratio,
            "scale": scale, "apart": False}


def listed():
    return [
        # one query through a trained network (a picked Gaussian, a time code) at 256 states: latency is all
        _attention("attention-query", "attention", "float16", 1, 1, 256, 4, 4, 64),
        # the million Gaussians of the large scene at the 256 states of an image's encoder, in training
        _attention("attention-1m", "attention", "bfloat16", 1, 1_000_000, 256, 4, 4, 64, train=True),
        # chunks of rows for two views with many states each, the second's padded; heads in fours share theirs
        _attention("attention-long", "attention", "float16", 2, 8192, 4096, 8, 2, 128, masked=2500, train=True),
        # a small full-precision network: ragged everywhere, rows further apart than they are long
        _attention("attention-50k", "attention", "float32", 1, 50_021, 197, 4, 4, 21, masked=181, pad=4),
        # the gradients over the million Gaussians
        _attention("attention-backward-1m", "attention_backward", "bfloat16", 1, 1_000_000, 256, 4, 4, 64),
        # the gradients of the many states, in halves, with shared heads
        _attention("attention-backward-long", "attention_backward", "float16", 2, 8192, 4096, 8, 2, 128, masked=2500),
        # the queries of the million Gaussians, turned by their positions
        _norm("head-norm-1m", "head_norm", "bfloat16", 1_000_000, 4, 64, 3),
        # a small scene in full precision: odd sizes, some of a head turned
        _norm("head-norm-6k", "head_norm", "float32", 6_007, 3, 38, 3, pairs=15),
        # the gradients of the million Gaussians' queries
        _norm("head-norm-backward-1m", "head_norm_backward", "float16", 1_000_000, 4, 64, 3),
        # and of a sequence of states, by their places in it
        _norm("head-norm-backward-states", "head_norm_backward", "bfloat16", 8_192, 8, 128, 1, extent=4096.0),
        # the gradients of a half-precision network's tensors, scaled losses undone, into float32: latency
        _clip_network("clip-network", "float16", 256, 256, 4, ratio=0.3, scale=1.0 / 4096.0, apart=True),
        # the gradients of a million Gaussians, within the bound as in most steps: nothing to write
        _clip_gaussians("clip-gaussians", 1_000_000, ratio=2.0),
    ]


def _size(rng, low, high):
    """A size between low and high, spread over its logarithm: often a multiple of 16, else as it comes."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if n > 32 and rng.random() < 0.5:
        n -= n % 16
    return max(low, min(high, n))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention_backward", "attention_backward", "head_norm",
                       "head_norm_backward", "clip"])
    dtype = rng.choice(["float32", "float16", "bfloat16"])
    pad = rng.choice([0, 0, 0, 8, 3])
    if kind == "clip":
        ratio = math.exp(rng.uniform(math.log(0.05), math.log(4.0)))
        if rng.random() < 0.4:
            c = _clip_gaussians("", _size(rng, 1, 1_000_000), ratio)
        else:
            c = _clip_network("", dtype, _size(rng, 16, 1024), _size(rng, 16, 4096), rng.randint(1, 6), ratio,
                              rng.choice([1.0, 0.25, 1.0 / 1024.0]), rng.random() < 0.5)
    elif kind.startswith("head_norm"):
        while True:
            head = rng.choice([16, 32, 64, 64, 128, 128, 256, 2 * rng.randint(1, 128)])
            axes = rng.choice([0, 1, 2, 3, 3])
            c = _norm("", kind, dtype, _size(rng, 1, 1 << 20), rng.randint(1, 16), head, axes,
                      head // 2 if rng.random() < 0.7 else rng.randint(1, head // 2),
                      math.exp(rng.uniform(0.0, math.log(1e4))), rng.random() < 0.8, pad)
            if work(c)["bytes"] <= 1.6e9:
                break
    else:
        while True:
            kv_heads = rng.choice([1, 1, 2, 4])
            head = rng.choice([16, 32, 64, 64, 128, 128, rng.randint(1, 128)])
            states = _size(rng, 1, 8192)
            masked = states if rng.random() < 0.5 else rng.randint(1, states)
            c = _attention("", kind, dtype, rng.choice([1, 1, 2, 5]), _size(rng, 1, 1 << 20), states,
                           kv_heads * rng.choice([1, 1, 2, 4]), kv_heads, head, masked, rng.random() < 0.5, pad)
            w = work(c)
            scores = c["batch"] * c["heads"] * c["queries"] * c["states"]
            if scores <= 1.0e9 and w["flops"] <= (2e11 if dtype == "float32" else 6e11) and w["bytes"] <= 2e9:
                break
    del c["name"]
    return c


def _kept(case):
    """How many states, the first ones, each element of the batch keeps: from all of them down to `masked`."""
    n, b = case["states"], case["batch"]
    lost = n - case["masked"]
    return [n - (lost * (k + 1) // b if b > 1 else lost) for k in range(b)]


def _shapes(case):
    """Of the gradients: matrices (rows, columns), and vectors (length,)."""
    if case["of"] == "gaussians":
        return [(case["number"], k) for k in GAUSSIAN]
    block = [(case["hidden"], case["width"]), (case["width"], case["hidden"])]
    matrices = [(case["width"], case["inputs"])] + block * case["blocks"] + [(case["outputs"], case["width"])]
    return matrices + [(sum(r for r, _ in matrices),)]


def work(case):
    size = torch.empty(0, dtype=_dtype(case["dtype"])).element_size()
    if case["kind"] == "clip":
        shapes = _shapes(case)
        n = [math.prod(s) for s in shapes]
        # a network's vectors are float32 whatever its type
        read = sum(k * (4 if len(s) == 1 else size) for k, s in zip(n, shapes))
        factor = case["scale"] * min(1.0, case["ratio"])
        written = 0 if factor == 1.0 and not case["apart"] else sum(n) * 4 if case["apart"] else read
        return {"bytes": read + written + 4, "flops": 3 * sum(n)}
    if case["kind"].startswith("head_norm"):
        n = case["rows"] * case["heads"] * case["head"]
        moved = (2 if case["kind"] == "head_norm" else 3) * n * size
        vectors = 4 * case["head"] * case["gamma"] * (1 if case["kind"] == "head_norm" else 2)
        return {"bytes": moved + 4 * case["axes"] * (case["rows"] + case["pairs"]) + vectors, "flops": 12 * n}
    rows, d = case["batch"] * case["queries"], case["head"]
    states = sum(_kept(case))
    q, k = rows * case["heads"] * d * size, states * case["kv_heads"] * d * size
    flops = case["queries"] * states * case["heads"] * d
    mask = case["batch"] * case["states"] if case["masked"] < case["states"] else 0
    if case["kind"] == "attention":
        return {"bytes": 2 * q + 2 * k + mask + 4 * rows * case["heads"] * case["train"], "flops": 4 * flops}
    return {"bytes": 4 * q + 4 * k + mask + 4 * rows * case["heads"], "flops": 10 * flops}


def _inputs(case, seed):
    """Everything but the derived inputs, from the seed alone."""
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))
    t = _dtype(case["dtype"])

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEVICE)

    def matrix(rows, cols, scale):
        """The first columns of a buffer whose other columns nothing may touch."""
        return normal(rows, cols + case.get("pad", 0)).mul_(scale).to(t)[:, :cols]

    s = {"case": case}
    if case["kind"] == "clip":
        shapes = _shapes(case)
        # gradients of scaled losses; the tensors' sizes lie far apart, as those of a Gaussian's numbers do
        s["grads"] = [normal(*sh).mul_(10.0 ** (-(k % 4))).div_(case["scale"] * 1e3).to(torch.float32 if len(sh) == 1 else t)
                      for k, sh in enumerate(shapes)]
        total = math.sqrt(sum(math.prod(sh) * (1e-3 * 10.0 ** (-(k % 4))) ** 2 for k, sh in enumerate(shapes)))
        s["bound"] = case["ratio"] * total
        s["clipped"] = [torch.zeros(sh, device=DEVICE) for sh in shapes] if case["apart"] else None
        return s
    if case["kind"].startswith("head_norm"):
        rows, d = case["rows"], case["head"]
        s["x"] = matrix(rows, case["heads"] * d, 1.3)
        s["gamma"] = 1.0 + 0.2 * normal(d) if case["gamma"] else None
        s["positions"] = s["frequencies"] = None
        if case["axes"]:
            u = torch.rand(rows, case["axes"], generator=g, device=DEVICE)
            s["positions"] = u.mul_(2.0 * case["extent"]).sub_(case["extent"])
            # from one turn in a unit to one in the hundredfold, in directions all around
            size = torch.logspace(0.8, -1.2, case["pairs"], device=DEVICE)
            direction = normal(case["pairs"], case["axes"])
            s["frequencies"] = size[:, None] * direction / direction.norm(dim=1, keepdim=True).clamp_min(1e-3)
        if case["kind"] == "head_norm_backward":
            s["grad_y"] = matrix(rows, case["heads"] * d, 1e-2)
        return s
    b, d = case["batch"], case["head"]
    # queries and keys after their norms, whose learned factors make some states matter more than others
    s["q"] = matrix(b * case["queries"], case["heads"] * d, 1.5)
    s["k"] = matrix(b * case["states"], case["kv_heads"] * d, 1.5)
    s["v"] = matrix(b * case["states"], case["kv_heads"] * d, 1.0)
    s["mask"] = None
    if case["masked"] < case["states"]:
        kept = torch.tensor(_kept(case), device=DEVICE)
        s["mask"] = torch.arange(case["states"], device=DEVICE)[None, :] < kept[:, None]
    if case["kind"] == "attention_backward":
        s["grad_out"] = matrix(b * case["queries"], case["heads"] * d, 1e-2)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "attention_backward":   # what the forward left
        out, s["lse"] = _plain_attention(dict(s, case=dict(case, train=True)))
        s["out"] = torch.empty(out.shape[0], out.shape[1] + case["pad"], dtype=out.dtype, device=DEVICE)[:, :out.shape[1]]
        s["out"].copy_(out)
    return s


# ---------------------------------------------------------------- the plain forms

def _heads(x, batch, heads):
    """[batch, heads, rows, d] in 32 bits of a matrix of batch x rows."""
    return x.float().reshape(batch, x.shape[0] // batch, heads, -1).transpose(1, 2).contiguous()


def _rows(x, dtype):
    """The matrix of [batch, heads, rows, d], rounded."""
    return x.transpose(1, 2).reshape(x.shape[0] * x.shape[2], -1).to(dtype)


def _shared(x, times):
    return x if times == 1 else x.repeat_interleave(times, dim=1)


def _plain_scores(s):
    case = s["case"]
    b, h, g = case["batch"], case["heads"], case["kv_heads"]
    q = _heads(s["q"], b, h)
    k, v = (_shared(_heads(s[n], b, g), h // g) for n in ("k", "v"))
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(1.0 / math.sqrt(case["head"]))
    if s["mask"] is not None:
        scores.masked_fill_(~s["mask"][:, None, None, :], -math.inf)
    return q, k, v, scores


def _plain_attention(s):
    case = s["case"]
    _, _, v, scores = _plain_scores(s)
    top = scores.amax(3, keepdim=True)
    e = scores.sub_(top).exp_()
    total = e.sum(3, keepdim=True)
    out = _rows(torch.matmul(e, v).div_(total), s["q"].dtype)
    if not case["train"]:
        return (out,)
    lse = (top + total.log())[..., 0].transpose(1, 2).reshape(out.shape[0], case["heads"])
    return out, lse


def _plain_attention_backward(s):
    case, t = s["case"], s["q"].dtype
    b, h, g = case["batch"], case["heads"], case["kv_heads"]
    q, k, v, scores = _plain_scores(s)
    lse = s["lse"].reshape(b, case["queries"], h).transpose(1, 2)[..., None]
    p = scores.sub_(lse).exp_()
    do, o = _heads(s["grad_out"], b, h), _heads(s["out"], b, h)
    delta = (do * o).sum(3, keepdim=True)
    dv = torch.matmul(p.transpose(2, 3), do)
    ds = torch.matmul(do, v.transpose(2, 3).contiguous()).sub_(delta).mul_(p).mul_(1.0 / math.sqrt(case["head"]))
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(2, 3), q)
    if g < h:
        dk, dv = (x.reshape(b, g, h // g, case["states"], case["head"]).sum(2) for x in (dk, dv))
    return _rows(dq, t), _rows(dk, t), _rows(dv, t)


def _turns(s):
    """Cosines and sines [rows, 1, pairs] of the pairs' angles."""
    angle = (s["positions"].double()[:, None, :] * s["frequencies"].double()[None, :, :]).sum(2)
    return torch.cos(angle).float()[:, None, :], torch.sin(angle).float()[:, None, :]


def _plain_turn(u, s, sign):
    if s["positions"] is None:
        return u
    n = 2 * s["frequencies"].shape[0]
    c, sn = _turns(s)
    sn = sn * sign
    x, y = u[..., 0:n:2], u[..., 1:n:2]
    turned = torch.stack((x * c - y * sn, x * sn + y * c), dim=-1).flatten(2)
    return torch.cat((turned, u[..., n:]), dim=2)


def _plain_head_norm(s):
    case, x = s["case"], s["x"].float()
    x = x.reshape(case["rows"], case["heads"], case["head"])
    u = x * torch.rsqrt(x.square().mean(2, keepdim=True) + EPS)
    if s["gamma"] is not None:
        u = u * s["gamma"]
    return (_plain_turn(u, s, 1.0).reshape(s["x"].shape).to(s["x"].dtype),)


def _plain_head_norm_backward(s):
    case, x = s["case"], s["x"].float()
    shape = (case["rows"], case["heads"], case["head"])
    x = x.reshape(shape)
    r = torch.rsqrt(x.square().mean(2, keepdim=True) + EPS)
    h = x * r
    g = _plain_turn(s["grad_y"].float().reshape(shape), s, -1.0)
    grad_gamma = (g * h).sum((0, 1)) if s["gamma"] is not None else None
    if s["gamma"] is not None:
        g = g * s["gamma"]
    dx = r * (g - h * (g * h).mean(2, keepdim=True))
    return dx.reshape(s["x"].shape).to(s["x"].dtype), grad_gamma


def _plain_clip(s):
    case = s["case"]
    total = sum(g.double().square().sum() for g in s["grads"])
    norm = total.sqrt() * case["scale"]
    factor = torch.clamp_max(s["bound"] / (norm + EPS), 1.0) * case["scale"]
    into = s["grads"] if s["clipped"] is None else s["clipped"]
    for g, c in zip(s["grads"], into):
        c.copy_(g.float() * factor.float())
    return into, norm.float()


PLAIN = {"attention": _plain_attention, "attention_backward": _plain_attention_backward, "head_norm": _plain_head_norm,
         "head_norm_backward": _plain_head_norm_backward, "clip": _plain_clip}


# ---------------------------------------------------------------- the package's operators

_handles = {}


def _layer_ops():
    """The handle that a program makes once and keeps: it owns the operators' workspace."""
    if "ops" not in _handles:
        from tinygs_amd.network import LayerOps
        _handles["ops"] = LayerOps()
    return _handles["ops"]


def _run_own(s):
    case = s["case"]
    if case["kind"] == "clip":
        if "clip" not in s:   # made once by a program, as its optimiser is, and kept
            from tinygs_amd.optim import GradientClip
            s["clip"] = GradientClip(s["grads"], clipped=s["clipped"])
        norm = s["clip"].clip(s["bound"], scale=case["scale"], epsilon=EPS)
        return s["grads"] if s["clipped"] is None else s["clipped"], norm
    ops = _layer_ops()
    if case["kind"] == "attention":
        got = ops.attention(s["q"], s["k"], s["v"], case["heads"], kv_heads=case["kv_heads"], batch=case["batch"],
                            mask=s["mask"], keep_lse=case["train"])
        return got if case["train"] else (got,)
    if case["kind"] == "attention_backward":
        return ops.attention_backward(s["grad_out"], s["q"], s["k"], s["v"], s["out"], s["lse"], case["heads"],
                                      kv_heads=case["kv_heads"], batch=case["batch"], mask=s["mask"])
    if case["kind"] == "head_norm":
        return (ops.head_norm(s["x"], case["heads"], s["gamma"], positions=s["positions"],
                              frequencies=s["frequencies"], eps=EPS),)
    return ops.head_norm_backward(s["grad_y"], s["x"], case["heads"], s["gamma"], positions=s["positions"],
                                  frequencies=s["frequencies"], eps=EPS)


def run(state):
    return _run_own(state) if own else PLAIN[state["case"]["kind"]](state)


# ---------------------------------------------------------------- the definitions in 64 bits

def _exact_attention(case, s):
    """By element of the batch and head, over the states that exist alone."""
    d = torch.float64
    nq, nk, w, shared = case["queries"], case["states"], case["head"], case["heads"] // case["kv_heads"]
    backward = case["kind"] == "attention_backward"
    grads = [torch.zeros(s[n].shape, dtype=d, device=DEVICE) for n in ("q", "k", "v")]
    out = torch.zeros(s["q"].shape, dtype=d, device=DEVICE)
    lse = torch.zeros(s["q"].shape[0], case["heads"], dtype=d, device=DEVICE)
    for b, kept in enumerate(_kept(case)):
        rows, states = slice(b * nq, (b + 1) * nq), slice(b * nk, b * nk + kept)
        for h in range(case["heads"]):
            cols = slice(h * w, (h + 1) * w)
            kv_cols = slice(h // shared * w, (h // shared + 1) * w)
            q, k, v = s["q"][rows, cols].to(d), s["k"][states, kv_cols].to(d), s["v"][states, kv_cols].to(d)
            z = torch.mm(q, k.t()) / math.sqrt(w)
            if not backward:
                total = torch.logsumexp(z, dim=1)
                lse[rows, h] = total
                out[rows, cols] = torch.mm(torch.exp(z - total[:, None]), v)
                continue
            p = torch.exp(z.sub_(s["lse"][rows, h].to(d)[:, None]))
            g = s["grad_out"][rows, cols].to(d)
            grads[2][states, kv_cols] += torch.mm(p.t(), g)
            dot = torch.einsum("rc,rc->r", g, s["out"][rows, cols].to(d))
            dz = p * (torch.mm(g, v.t()) - dot[:, None]) / math.sqrt(w)
            grads[0][rows, cols] = torch.mm(dz, k)
            grads[1][states, kv_cols] += torch.mm(dz.t(), q)
    if backward:
        return tuple(grads)
    return (out, lse) if case["train"] else (out,)


def _exact_head_norm(case, s):
    """Pairs as complex numbers, multiplied by e^(i angle); columns beyond the pairs by one."""
    d, n = torch.float64, case["head"]
    shape = (case["rows"], case["heads"], n)
    x = s["x"].to(d).reshape(shape)
    gamma = torch.ones(n, dtype=d, device=DEVICE) if s["gamma"] is None else s["gamma"].to(d)
    pairs = case["pairs"]
    if pairs:
        angle = torch.mm(s["positions"].to(d), s["frequencies"].to(d).t())[:, None, :]
        turn = torch.complex(torch.cos(angle), torch.sin(angle))

    def turned(u, by):
        if not pairs:
            return u
        z = torch.view_as_complex(u[..., :2 * pairs].reshape(*shape[:2], pairs, 2).contiguous()) * by
        return torch.cat((torch.view_as_real(z).reshape(*shape[:2], 2 * pairs), u[..., 2 * pairs:]), dim=2)

    root = torch.sqrt((x ** 2).sum(2, keepdim=True) / n + EPS)
    if case["kind"] == "head_norm":
        return (turned(x / root * gamma, turn if pairs else None).reshape(s["x"].shape),)
    g = turned(s["grad_y"].to(d).reshape(shape), turn.conj() if pairs else None)
    grad_gamma = (g * x / root).sum((0, 1)) if s["gamma"] is not None else None
    g = g * gamma
    # d(x / root) = (dx - x (x . dx) / (n root^2)) / root
    dx = g / root - x * ((g * x).sum(2, keepdim=True) / (n * root ** 3))
    return dx.reshape(s["x"].shape), grad_gamma


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "clip":
        wide = [g.to(torch.float64) for g in s["grads"]]
        norm = case["scale"] * math.sqrt(sum(float((g * g).sum()) for g in wide))
        factor = case["scale"] * min(1.0, s["bound"] / (norm + EPS))
        return [g * factor for g in wide], torch.tensor(norm, dtype=torch.float64, device=DEVICE)
    if case["kind"].startswith("attention"):
        return _exact_attention(case, s)
    return _exact_head_norm(case, s)
