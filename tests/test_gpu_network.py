"""The attribute network's layer operators against their definitions in 64 bits, at the sizes, alignments and values
where they can go wrong, with bounds derived in network_reference."""
import pytest
import torch

import network_reference as R

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
IDS = ["f32", "f16", "bf16"]
# rows, in, out: single elements, single rows, odd and ragged edges, whole tiles and one past them, deep and wide
SHAPES = [(1, 1, 1), (1, 256, 256), (1, 1000, 3), (2, 7, 5), (5, 64, 1), (8, 512, 1030), (9, 40, 72), (17, 84, 59),
          (33, 256, 64), (64, 64, 64), (127, 128, 128), (129, 130, 257), (300, 1, 9), (1000, 323, 96),
          (1025, 256, 256), (640, 512, 384), (3, 1024, 2048), (4099, 84, 59), (70001, 72, 40), (20000, 256, 128),
          (33000, 72, 72), (33000, 520, 72), (70000, 264, 260), (4097, 256, 700), (66000, 24, 260), (70001, 260, 24), (150001, 130, 129),
          (33, 4096, 130), (200, 1300, 77), (70, 600, 2100),
          (39, 121, 59), (40, 1, 3), (41, 3, 1), (64, 5, 250), (72, 250, 7), (8193, 59, 123), (70001, 129, 250)]


@pytest.fixture(scope="module")
def ops(hip):
    from tinygs_amd.network import LayerOps
    return LayerOps()


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def matrix(seed, rows, cols, dtype, pad=0, lead=0, scale=1.0):
    """A matrix of normal values inside a buffer that holds NaN everywhere else."""
    full = torch.full((rows, lead + cols + pad), float("nan"), dtype=dtype, device="cuda")
    full[:, lead:lead + cols] = (scale * normal(seed, rows, cols)).to(dtype).cuda()
    return full[:, lead:lead + cols]


def output(rows, cols, dtype, pad=0, lead=0):
    full = torch.full((rows, lead + cols + pad), -7.0, dtype=dtype, device="cuda")
    return full[:, lead:lead + cols], full


def untouched(full, lead, cols):
    """The elements beside the output keep what they held."""
    assert bool((full[:, :lead] == -7.0).all()) and bool((full[:, lead + cols:] == -7.0).all())


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_linear(ops, shape, dtype):
    rows, i, o = shape
    for k, (name, pad, lead) in enumerate([("none", 0, 0), ("relu", 8, 0), ("silu", 3, 1), ("gelu", 0, 0)]):
        print(f"[linear] {shape} {dtype} {name} pad {pad} lead {lead}", flush=True)
        x = matrix(1 + k, rows, i, dtype, pad, lead)
        w = matrix(11 + k, o, i, dtype, pad, lead, i ** -0.5)
        b = normal(21 + k, o).cuda() if k != 0 else None
        r = matrix(31 + k, rows, o, dtype, pad, lead) if k % 2 else None
        y, yfull = output(rows, o, dtype, pad, lead)
        z, zfull = output(rows, o, dtype, pad, lead)
        got = ops.linear(x, w, b, activation=name, residual=r, out=y, preact=z)
        assert got[0] is y and got[1] is z
        wy, by, wz, bz = R.linear(x, w, b, name, r, dtype)
        R.check(y, wy, by, "y")
        R.check(z, wz, bz, "z")
        untouched(yfull, lead, o)
        untouched(zfull, lead, o)
        # without the values before the activation: the same y, bit for bit
        assert torch.equal(ops.linear(x, w, b, activation=name, residual=r), y)
        if r is not None:   # in the residual's place
            buf = r.contiguous().clone()
            assert torch.equal(ops.linear(x, w, b, activation=name, residual=buf, out=buf), y)


# enough rows that a call moves more than the caches hold; the first, the last and some of the others are compared
MANY = [(300001, 130, 200), (260001, 84, 520), (1200001, 59, 61), (700003, 256, 64), (400000, 24, 256), (140000, 128, 700)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", MANY, ids=str)
def test_linear_many_rows(ops, shape, dtype):
    rows, i, o = shape
    g = torch.Generator("cuda").manual_seed(5)
    at = torch.cat([torch.arange(200), torch.randint(rows, (2000,), generator=torch.Generator().manual_seed(6)),
                    torch.arange(rows - 200, rows)]).cuda()
    for k, (name, pad) in enumerate([("none", 0), ("silu", 3), ("gelu", 0)]):
        print(f"[linear] {shape} {dtype} {name} pad {pad}", flush=True)
        x = torch.full((rows, i + pad), float("nan"), dtype=dtype, device="cuda")[:, :i]
        x.copy_(torch.randn(rows, i, generator=g, device="cuda"))
        w = matrix(11 + k, o, i, dtype, pad, 0, i ** -0.5)
        b = normal(21 + k, o).cuda()
        r = torch.randn(rows, o, generator=g, device="cuda").to(dtype) if k else None
        y, yfull = output(rows, o, dtype, pad)
        z, zfull = output(rows, o, dtype, pad)
        ops.linear(x, w, b, activation=name, residual=r, out=y, preact=z)
        wy, by, wz, bz = R.linear(x[at], w, b, name, None if r is None else r[at], dtype)
        R.check(y[at], wy, by, "y")
        R.check(z[at], wz, bz, "z")
        assert bool(torch.isfinite(y).all()) and bool(torch.isfinite(z).all())
        untouched(yfull, 0, o)
        untouched(zfull, 0, o)
        again = ops.linear(x, w, b, activation=name, residual=r)
        R.check(again[at], wy, by, "y without the values before the activation")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_linear_backward(ops, shape, dtype):
    rows, i, o = shape
    for k, (name, pad, lead) in enumerate([("none", 0, 0), ("relu", 8, 0), ("silu", 3, 1), ("gelu", 0, 0)]):
        print(f"[linear_backward] {shape} {dtype} {name} pad {pad} lead {lead}", flush=True)
        x = matrix(1 + k, rows, i, dtype, pad, lead)
        w = matrix(11 + k, o, i, dtype, pad, lead, i ** -0.5)
        gy = matrix(41 + k, rows, o, dtype, pad, lead, 0.1)
        z = matrix(51 + k, rows, o, dtype, pad, lead, 2.0) if name != "none" else None
        gx, xfull = output(rows, i, dtype, pad, lead)
        gw, wfull = output(o, i, dtype, pad, lead)
        got = ops.linear_backward(gy, x, w, preact=z, activation=name, grad_x=gx, grad_weight=gw)
        assert got[0] is gx and got[1] is gw
        for t, (want, bound), what in zip(got, R.linear_backward(gy, x, w, z, name, dtype), ("gx", "gw", "gb")):
            R.check(t, want, bound, what)
        untouched(xfull, lead, i)
        untouched(wfull, lead, i)
        # again, and each gradient without the others: the same bits
        again = ops.linear_backward(gy, x, w, preact=z, activation=name)
        for a, b in zip(got, again):
            assert torch.equal(a, b)
        for n in range(3):
            part = ops.linear_backward(gy, x, w, preact=z, activation=name, need_x=n == 0, need_weight=n == 1,
                                       need_bias=n == 2)
            assert torch.equal(part[n], got[n]) and all(part[m] is None for m in range(3) if m != n)


def test_linear_gradients_are_the_slopes(ops):
    """The gradients against differences of the forward, in 32 bits with a step that leaves 1e-3."""
    rows, i, o = 5, 6, 7
    for name in R.ACTIVATIONS:
        x, w = matrix(1, rows, i, torch.float32), matrix(2, o, i, torch.float32)
        b, c = normal(3, o).cuda(), normal(4, rows, o).cuda()

        def loss():
            return float((ops.linear(x, w, b, activation=name).double() * c.double()).sum())

        _, z = ops.linear(x, w, b, activation=name, keep_preact=True)
        grads = ops.linear_backward(c, x, w, preact=z, activation=name)
        for t, g in zip((x, w, b), grads):
            for at in range(0, t.numel(), 3):
                flat = t.view(-1)
                keep, h = float(flat[at]), 2.0 ** -8
                flat[at] = keep + h
                up = loss()
                flat[at] = keep - h
                down = loss()
                flat[at] = keep
                # relu: a kink within the step moves the difference, so only points away from it
                if name == "relu" and bool((z.abs() < 0.1).any()) and abs((up - down) / (2 * h) - float(g.reshape(-1)[at])) > 1e-2:
                    continue
                assert abs((up - down) / (2 * h) - float(g.reshape(-1)[at])) <= 1e-3 * (1 + abs(float(g.reshape(-1)[at])))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_linear_infinities_stay_in_their_rows(ops, dtype):
    """A row with an infinity or a NaN leaves the others as they were; so does a column of w."""
    rows, i, o = 150, 96, 80
    x, w = matrix(1, rows, i, dtype), matrix(2, o, i, dtype, scale=i ** -0.5)
    b = normal(3, o).cuda()
    clean = ops.linear(x, w, b, activation="gelu")
    x2 = x.clone()
    x2[5, 7], x2[77, 0], x2[149, 95] = float("nan"), float("inf"), float("-inf")
    y = ops.linear(x2, w, b, activation="gelu")
    keep = [r for r in range(rows) if r not in (5, 77, 149)]
    assert torch.equal(y[keep], clean[keep])
    assert not bool(torch.isfinite(ops.linear(x2, w, b)[[5, 77, 149]]).any())


def test_linear_activations_at_the_ends(ops):
    """Values from -1e30 to 1e30 through each activation and its slope."""
    v = torch.tensor([-1e30, -1e4, -100.0, -30.5, -20.0, -9.0, -1.0, -1e-3, -1e-30, 0.0, 1e-30, 1e-3, 1.0, 9.0, 20.0,
                      30.5, 100.0, 1e4, 1e30])
    x, one = v[:, None].cuda(), torch.ones(1, 1, device="cuda")
    for name in R.ACTIVATIONS:
        z64 = v.double()
        y = ops.linear(x, one, None, activation=name)[:, 0].double().cpu()
        want = R.act(z64, name)
        want = torch.where(z64 < -1e3, torch.zeros_like(want) if name != "none" else want, want)
        assert bool(((y - want).abs() <= R.ACT_ERROR * (1 + want.abs())).all()), name
        if name == "none":
            continue
        gx = ops.linear_backward(torch.ones(len(v), 1, device="cuda"), x, one, preact=x, activation=name)[0]
        want = torch.where(z64.abs() > 1e3, (z64 > 0).double(), R.act_slope(z64.clamp(-1e3, 1e3), name))
        assert bool(((gx[:, 0].double().cpu() - want).abs() <= 2 * R.ACT_ERROR * (1 + want.abs())).all()), name


def test_linear_no_rows(ops):
    x, w = torch.empty(0, 8, device="cuda"), torch.ones(4, 8, device="cuda")
    assert ops.linear(x, w).shape == (0, 4)
    gx, gw, gb = ops.linear_backward(torch.empty(0, 4, device="cuda"), x, w)
    assert gx.shape == (0, 8) and bool((gw == 0).all()) and bool((gb == 0).all())


NORMS = [(1, 1), (1, 8), (3, 2), (5, 7), (64, 64), (33, 59), (1000, 84), (129, 256), (257, 257), (6007, 323),
         (40, 1024), (70, 1031), (9, 4096), (11, 8200), (20011, 128), (3, 20000)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", NORMS, ids=str)
def test_layer_norm(ops, shape, dtype):
    rows, n = shape
    for k, (pad, lead) in enumerate([(0, 0), (8, 0), (5, 3)]):
        print(f"[layer_norm] {shape} {dtype} pad {pad} lead {lead}", flush=True)
        x = matrix(1 + k, rows, n, dtype, pad, lead, 1.5)
        x += 0.25
        gamma, beta = (normal(5, n).cuda(), normal(6, n).cuda()) if k != 1 else (None, None)
        y, full = output(rows, n, dtype, pad, lead)
        got = ops.layer_norm(x, gamma, beta, eps=1e-5, out=y)
        for t, (want, bound), what in zip(got, R.layer_norm(x, gamma, beta, 1e-5, dtype), ("y", "mean", "rstd")):
            R.check(t, want, bound, what)
        untouched(full, lead, n)
        buf = x.contiguous().clone()
        assert torch.equal(ops.layer_norm(buf, gamma, beta, eps=1e-5, out=buf)[0], y)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", NORMS, ids=str)
def test_layer_norm_backward(ops, shape, dtype):
    rows, n = shape
    for k, (pad, lead) in enumerate([(0, 0), (8, 0), (5, 3)]):
        print(f"[layer_norm_backward] {shape} {dtype} pad {pad} lead {lead}", flush=True)
        x = matrix(1 + k, rows, n, dtype, pad, lead, 1.5)
        gy = matrix(11 + k, rows, n, dtype, pad, lead, 0.1)
        res = matrix(21 + k, rows, n, dtype, pad, lead, 0.1) if k else None
        gamma = normal(5, n).cuda() if k != 1 else None
        mean, rstd = ops.layer_norm(x, gamma, None, eps=1e-3)[1:]
        gx, full = output(rows, n, dtype, pad, lead)
        got = ops.layer_norm_backward(gy, x, gamma, mean, rstd, residual_grad=res, grad_x=gx)
        want = R.layer_norm_backward(gy, x, gamma, mean, rstd, res, dtype)
        for t, (v, bound), what in zip(got, want, ("gx", "ggamma", "gbeta")):
            R.check(t, v, bound, what)
        untouched(full, lead, n)
        again = ops.layer_norm_backward(gy, x, gamma, mean, rstd, residual_grad=res)
        for a, b in zip(got, again):
            assert torch.equal(a, b)
        buf = gy.contiguous().clone()
        assert torch.equal(ops.layer_norm_backward(buf, x, gamma, mean, rstd, residual_grad=res, grad_x=buf)[0], gx)


def test_layer_norm_constant_and_shifted_rows(ops):
    """Rows of one value have variance 0 and no NaN; a large common offset costs no more than its rounding."""
    for n in (8, 300, 2000):
        x = torch.full((4, n), 3.5, device="cuda")
        y, mean, rstd = ops.layer_norm(x, eps=1e-5)
        assert bool((y == 0).all()) and bool((mean == 3.5).all())
        assert bool(((rstd - 1e-5 ** -0.5).abs() <= 8 * R.EPS24 * 1e-5 ** -0.5).all())
        x = 4096.0 + normal(1, 6, n).cuda()
        for t, (want, bound) in zip(ops.layer_norm(x), R.layer_norm(x, None, None, 1e-5, torch.float32)):
            R.check(t, want, bound, n)
        x2 = x.clone()
        x2[3, 1] = float("nan")
        y, y2 = ops.layer_norm(x)[0], ops.layer_norm(x2)[0]
        assert torch.equal(y[[0, 1, 2, 4, 5]], y2[[0, 1, 2, 4, 5]]) and bool(torch.isnan(y2[3]).all())


def test_layer_norm_gradient_is_the_slope(ops):
    rows, n = 3, 9
    x, c = matrix(1, rows, n, torch.float32), normal(2, rows, n).cuda()
    gamma, beta = normal(3, n).cuda(), normal(4, n).cuda()

    def loss():
        return float((ops.layer_norm(x, gamma, beta)[0].double() * c.double()).sum())

    _, mean, rstd = ops.layer_norm(x, gamma, beta)
    for t, g in zip((x, gamma, beta), ops.layer_norm_backward(c, x, gamma, mean, rstd)):
        for at in range(t.numel()):
            flat = t.view(-1)
            keep, h = float(flat[at]), 2.0 ** -8
            flat[at] = keep + h
            up = loss()
            flat[at] = keep - h
            down = loss()
            flat[at] = keep
            assert abs((up - down) / (2 * h) - float(g.reshape(-1)[at])) <= 1e-3 * (1 + abs(float(g.reshape(-1)[at])))


def test_layer_norm_no_rows(ops):
    x = torch.empty(0, 8, device="cuda")
    y, mean, rstd = ops.layer_norm(x)
    assert y.shape == (0, 8)
    gx, gg, gb = ops.layer_norm_backward(x, x, None, mean, rstd)
    assert gx.shape == (0, 8) and bool((gg == 0).all()) and bool((gb == 0).all())


def test_other_stream_and_replays(hip):
    """The operators on a stream of their own, captured into a graph and replayed on new values."""
    from tinygs_amd.network import LayerOps
    ops, s = LayerOps(), torch.cuda.Stream()
    rows, i, o = 5000, 96, 64
    for dtype in DTYPES:
        x, w, b = matrix(1, rows, i, dtype), matrix(2, o, i, dtype, scale=0.1), normal(3, o).cuda()
        gamma = normal(4, i).cuda()
        gy = matrix(5, rows, o, dtype)
        torch.cuda.synchronize()

        def pass_():
            n, mean, rstd = ops.layer_norm(x, gamma, None, stream=s)
            y, z = ops.linear(n, w, b, activation="gelu", keep_preact=True, stream=s)
            gn, gw, gb = ops.linear_backward(gy, n, w, preact=z, activation="gelu", stream=s)
            return (y, gw, gb) + ops.layer_norm_backward(gn, x, gamma, mean, rstd, stream=s)

        with torch.cuda.stream(s):
            pass_()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                held = pass_()
        for k in range(3):
            x.copy_(normal(30 + k, rows, i).to(dtype).cuda())
            torch.cuda.synchronize()
            print(f"[replay] {dtype} {k}", flush=True)
            g.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in held]
            want = pass_()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))
