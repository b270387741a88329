"""Muon against its definition in 64 bits: several matrices a step, momenta, copies, odd shapes, extreme gradients."""
import numpy as np
import pytest
import torch

import network_reference as R

pytestmark = pytest.mark.gpu

SHAPES = [(1, 1), (1, 9), (7, 1), (3, 5), (16, 16), (17, 33), (59, 256), (64, 64), (65, 63), (128, 300), (200, 129),
          (256, 84), (256, 256), (257, 255), (40, 1030), (700, 130), (520, 520)]
# A step's X is off by what its products' operands lose (22 bits and float sums), which each iteration lifts by at
# most a = 3.4445 in the directions that it lifts: 5 iterations, 485 in all, on sums of entries of one sign at worst
# over the side; normwise 2^-22 485 sqrt(5) is 2.6e-4 of |X|.
X_BOUND = 2.6e-4


def tensors(shape, seed, grad_dtype, pad=0):
    g = torch.Generator().manual_seed(seed)
    r, c = shape

    def one(scale, dtype):
        full = torch.full((r, c + pad), float("nan"), dtype=dtype, device="cuda")
        full[:, :c] = (scale * torch.randn(r, c, generator=g)).to(dtype).cuda()
        return full[:, :c]

    return one(c ** -0.5, torch.float32), one(1e-3, torch.float32), one(1e-2, grad_dtype)


def agrees(before, got_w, got_m, p, scale=1.0, what=None):
    w, m, g = before
    want_w, want_m, x = R.muon(w, m, g, p, scale)
    assert bool(((got_m.double().cpu() - want_m).abs() <= 6 * R.EPS24 * (m.double().cpu().abs() + scale * g.double().cpu().abs())).all()), what
    step = p["lr"] * np.sqrt(max(1.0, w.shape[0] / w.shape[1]))
    d = (got_w.double().cpu() - want_w).norm()
    assert float(d) <= step * X_BOUND * float(x.norm()) + 4 * R.EPS24 * float(w.double().norm()), (what, float(d))


@pytest.mark.parametrize("grad_dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("pad", [0, 5])
def test_step(hip, grad_dtype, pad):
    from tinygs_amd.optim import Muon
    sets = [tensors(s, k, grad_dtype, pad) for k, s in enumerate(SHAPES)]
    copies = None if grad_dtype == torch.float32 else [torch.full_like(g, -7.0) for _, _, g in sets]
    opt = Muon([w for w, _, _ in sets], [g for _, _, g in sets], momenta=[m for _, m, _ in sets], copies=copies)
    assert opt.get_params()["iterations"] == 5
    for k, more in enumerate([{}, {"nesterov": 0, "weight_decay": 0.1}, {"momentum": 0.5, "lr": 0.1}]):
        opt.set_params(more)
        p = opt.get_params()
        before = [[t.clone() for t in s] for s in sets]
        print(f"[muon] step {k} {grad_dtype} pad {pad}", flush=True)
        opt.step(0.5)
        torch.cuda.synchronize()
        for i, ((w, m, g), b) in enumerate(zip(sets, before)):
            agrees(b, w, m, p, 0.5, (k, SHAPES[i]))
            assert torch.equal(g, b[2])
            if copies is not None:
                assert torch.equal(copies[i], w.to(grad_dtype))


@pytest.mark.parametrize("iterations", [0, 1, 2, 12])
def test_iterations(hip, iterations):
    from tinygs_amd.optim import create_optimizer
    sets = [tensors(s, 7 + k, torch.float32) for k, s in enumerate([(48, 80), (90, 31)])]
    opt = create_optimizer("muon", [s[0] for s in sets], [s[2] for s in sets])
    opt.set_params({"iterations": iterations})
    before = [(w.clone(), torch.zeros_like(w), g.clone()) for w, _, g in sets]
    opt.step(1.0)
    for (w, _, _), m, b in zip(sets, opt.momenta(), before):
        agrees(b, w, m, opt.get_params(), 1.0, iterations)


def test_update_does_not_depend_on_the_gradients_size(hip):
    """The update is normalised: gradients of 1e-28 and of 1e28 step as those of 1 do, and none leave W to its decay."""
    from tinygs_amd.optim import Muon
    w0, _, g = tensors((96, 40), 3, torch.float32)
    got = []
    for size in (2.0 ** -93, 1.0, 2.0 ** 93, 0.0):
        w = w0.clone()
        opt = Muon([w], [g * size])
        opt.set_params({"weight_decay": 0.5, "epsilon": 1e-37})
        opt.step(1.0)
        got.append(w)
    assert torch.equal(got[0], got[1]) and torch.equal(got[1], got[2])
    assert torch.equal(got[3], w0 * np.float32(1 - np.float32(0.02) * np.float32(0.5)))


def test_nan_stays_in_its_matrix(hip):
    from tinygs_amd.optim import Muon
    a, b = tensors((64, 96), 1, torch.float32), tensors((64, 96), 2, torch.float32)
    twin = [t.clone() for t in b]
    a[2][3, 4] = float("nan")
    Muon([a[0], b[0]], [a[2], b[2]], momenta=[a[1], b[1]]).step(1.0)
    Muon([twin[0]], [twin[2]], momenta=[twin[1]]).step(1.0)
    assert bool(torch.isnan(a[0]).all()) and torch.equal(b[0], twin[0])


def test_reset_lr_rebinding_and_replays(hip):
    from tinygs_amd.optim import Muon
    s = torch.cuda.Stream()
    sets = [tensors(sh, k, torch.bfloat16) for k, sh in enumerate([(64, 64), (130, 50), (256, 84)])]
    eager = [[t.clone() for t in x] for x in sets]
    torch.cuda.synchronize()

    def make(x):
        return Muon([t[0] for t in x], [t[2] for t in x], momenta=[t[1] for t in x])

    a, b = make(sets), make(eager)
    for o in (a, b):
        o.set_lr(0.5)
        assert o.get_lr() == 0.5
        o.step(1.0, stream=s)
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        a.step(1.0, stream=s)
    for k in range(3):
        g.replay()
        b.step(1.0, stream=s)
        torch.cuda.synchronize()
        for x, y in zip(sets, eager):
            assert torch.equal(x[0], y[0]) and torch.equal(x[1], y[1]), k
    other = [t[2].clone().mul_(-1) for t in eager]
    b.set_grads(other)
    before = [t[0].clone() for t in eager]
    b.reset(stream=s)
    b.step(1.0, stream=s)
    s.synchronize()
    p = dict(b.get_params(), lr=0.01)
    for x, w, gr in zip(eager, before, other):
        agrees((w, torch.zeros_like(w), gr), x[0], x[1], p, 1.0, "rebound")
