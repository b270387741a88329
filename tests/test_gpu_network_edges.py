"""The attribute network's operators where their definitions meet the types' ends and each other's places: outputs over
inputs, infinities, matrices of a few columns."""
import pytest
import torch

import network_reference as R

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
IDS = ["f32", "f16", "bf16"]


@pytest.fixture(scope="module")
def ops(hip):
    from tinygs_amd.network import LayerOps
    return LayerOps()


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


# rows in a group of lanes, in a wave, in a workgroup's registers, and read again from memory (above 32 KB)
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(5, 9), (1000, 84), (70, 1031), (9, 8192), (11, 8200), (300, 8200), (7, 16384), (3, 20000)],
                         ids=str)
def test_layer_norm_backward_in_its_inputs_place(ops, shape, dtype):
    """grad_x in grad_y's own matrix, or in residual_grad's: all three gradients as with a matrix of its own."""
    rows, n = shape
    x = (1.5 * normal(1, rows, n)).to(dtype).cuda()
    gy, res = (0.1 * normal(2, rows, n)).to(dtype).cuda(), (0.1 * normal(3, rows, n)).to(dtype).cuda()
    gamma = normal(4, n).cuda()
    mean, rstd = ops.layer_norm(x, gamma, None, eps=1e-3)[1:]
    for residual in (None, res):
        apart = ops.layer_norm_backward(gy, x, gamma, mean, rstd, residual_grad=residual)
        for t, (want, bound), what in zip(apart, R.layer_norm_backward(gy, x, gamma, mean, rstd, residual, dtype),
                                          ("gx", "ggamma", "gbeta")):
            R.check(t, want, bound, what)
        buf = gy.clone()
        got = ops.layer_norm_backward(buf, x, gamma, mean, rstd, residual_grad=residual, grad_x=buf)
        for t, want, what in zip(got, apart, ("gx", "ggamma", "gbeta")):
            assert torch.equal(t, want), f"{what} over grad_y"
    buf = res.clone()
    got = ops.layer_norm_backward(gy, x, gamma, mean, rstd, residual_grad=buf, grad_x=buf)
    for t, want, what in zip(got, apart, ("gx", "ggamma", "gbeta")):
        assert torch.equal(t, want), f"{what} over residual_grad"


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("out", [3, 64, 600])
@pytest.mark.parametrize("name", ["relu", "silu", "gelu"])
def test_slopes_at_infinity(ops, name, out, dtype):
    """Values before the activation that left the type's range, as float16's do at 65520: slope 1 above, 0 below."""
    rows, i = 70, 20
    z = (2.0 * normal(1, rows, out)).to(dtype)
    z[3, 0], z[4, 1], z[69, out - 1] = float("inf"), float("-inf"), float("inf")
    x, w, gy = normal(2, rows, i).to(dtype), normal(3, out, i).to(dtype), normal(4, rows, out).to(dtype)
    got = ops.linear_backward(gy.cuda(), x.cuda(), w.cuda(), preact=z.cuda(), activation=name)
    # at +-200 the slopes are 1 and 0 to every bit
    want = R.linear_backward(gy, x, w, z.double().clamp(-200.0, 200.0), name, dtype)
    for t, (v, bound), what in zip(got, want, ("gx", "gw", "gb")):
        R.check(t, v, bound, what)


INF, NAN = float("inf"), float("nan")
HUGE = 3.4e38   # above bfloat16's largest number, below float's


def alike(got, want, bound, what):
    """Equal infinities and NaN, and everything else within its bound. What exceeds float's range is infinite."""
    got = got.double().cpu()
    want = torch.where(want.abs() > 3.4028236e38, want.sign() * INF, want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), (what, "NaN")
    ends = torch.isinf(want)
    assert torch.equal(torch.isinf(got), ends) and torch.equal(got[ends], want[ends]), (what, "infinities")
    held = torch.isfinite(want)
    assert bool(((got - want).abs() <= bound)[held].all()), what


def ends(rows, i, o):
    """x and w whose products meet the ends of float, in some rows of each, the first and the last among them. What
    HUGE is multiplied with stays below one, so that float sums overflow where exact ones do."""
    x, w = normal(1, rows, i), 0.3 * i ** -0.5 * normal(2, o, i)
    k = i // 2
    x[rows - 1] *= 0.1
    x[:, k] *= 0.1
    x[0, k] = INF
    x[rows // 3, 0], x[rows // 2, i - 1], x[rows - 1, k + 1] = -INF, NAN, HUGE
    x[rows // 4, k], x[rows // 4, i - 1] = INF, -INF   # NaN where w's signs there agree
    if o > 4:
        w[1, k] = 0.0             # times infinity: NaN
        w[2, k] = 1e-30           # times infinity: infinity
        w[o - 2, 0] = INF
    return x, w


# few rows; one, several and ragged tiles; k split; many large, middle and narrow tiles; many rows of a narrow layer
@pytest.mark.parametrize("shape", [(3, 8, 16), (20, 999, 17), (4, 4096, 40), (150, 96, 80), (97, 33, 5), (130, 4096, 64),
                                   (16384, 130, 1024), (8192, 130, 512), (100000, 300, 40), (800001, 50, 130),
                                   (700001, 128, 128)], ids=str)
@pytest.mark.parametrize("name", ["none", "relu"])
def test_linear_infinities_in_floats(ops, shape, name):
    """Infinities, NaN and floats past bfloat16's range: what float products and sums give."""
    rows, i, o = shape
    x, w = ends(rows, i, o)
    w[o // 2, i // 2] = HUGE
    b = normal(3, o)
    print(f"[linear] {shape} {name}", flush=True)
    y, z = ops.linear(x.cuda(), w.cuda(), b.cuda(), activation=name, keep_preact=True)
    at = torch.arange(rows) if rows < 5000 else torch.cat([torch.arange(300), torch.arange(rows // 4 - 40, rows // 4 + 40),
                                                           torch.arange(rows // 3 - 40, rows // 3 + 40),
                                                           torch.arange(rows // 2 - 40, rows // 2 + 40),
                                                           torch.arange(rows - 300, rows)])
    wz = x[at].double() @ w.double().t() + b.double()
    bound = torch.nan_to_num(R.product_bound(x[at].double(), w.double().t(), i), nan=INF) + 3 * R.EPS24 * b.double().abs() \
        + R.EPS24 * torch.nan_to_num(wz.abs(), nan=INF) + R.STEP[torch.float32]
    alike(z[at], wz, bound, "z")
    alike(y[at], R.act(wz, name), bound, "y")


# narrow layers, whole and ragged chunks; tiles, with their sums over out and over the rows split or not
@pytest.mark.parametrize("shape", [(3, 8, 16), (70, 72, 40), (5000, 128, 128), (4100, 83, 59), (40, 300, 20),
                                   (130, 260, 4096), (5000, 260, 300), (20000, 513, 64)], ids=str)
@pytest.mark.parametrize("name", ["none", "silu"])
def test_linear_backward_infinities_in_floats(ops, shape, name):
    rows, i, o = shape
    x, w = ends(rows, i, o)
    gy = normal(4, rows, o)
    gy[rows - 1] *= 0.1
    gy[rows // 2, o - 1], gy[rows // 2 - 1, 0], gy[1, o // 2], gy[rows - 1, o // 3] = INF, -INF, NAN, HUGE
    z = normal(5, rows, o) if name != "none" else None
    if z is not None:
        z[rows - 1, o // 3] = 0.0   # slope 1/2
    print(f"[linear_backward] {shape} {name}", flush=True)
    got = ops.linear_backward(gy.cuda(), x.cuda(), w.cuda(), preact=None if z is None else z.cuda(), activation=name)
    for t, (v, bound), what in zip(got, R.linear_backward(gy, x, w, z, name, torch.float32), ("gx", "gw", "gb")):
        alike(t, v, torch.nan_to_num(bound, nan=INF), what)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_optimizer_by_name_trains_the_network(hip, dtype):
    """A network's optimiser made by its name, as the network's documentation has it, steps as net.optimizer() does,
    and forward reads what it wrote."""
    from tinygs_amd.network import AttributeNetwork
    from tinygs_amd.optim import create_optimizer
    features, grad = normal(1, 300, 20).to(dtype).cuda(), normal(2, 300, 7).to(dtype).cuda()
    after = []
    for by_name in (False, True):
        net = AttributeNetwork(20, 7, width=48, blocks=1, dtype=dtype, seed=3)
        opt = create_optimizer("muon", net.weights, net.grads, copies=net.copies) if by_name else net.optimizer()
        first = net.forward(features)
        net.backward(grad)
        opt.step(1.0)
        after.append(net.forward(features, keep=False))
        assert not torch.equal(after[-1], first)
        for w, m in zip(net.weights, net.matrices()):
            assert torch.equal(w.to(dtype), m)
    assert torch.equal(after[0], after[1])


# rows of fewer elements than 16 bytes hold, one to a few of them after the last whole block of 64; the second number
# of columns makes the call one of the many-row kernel, or its residual as narrow as x
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("more", [1, 2, 6])
@pytest.mark.parametrize("i,o", [(1, 128), (3, 129), (7, 260), (3, 3), (5, 1)])
def test_linear_many_short_rows(ops, i, o, more, dtype):
    size = 4 if dtype == torch.float32 else 2
    if size == 4 and o < 128:
        i, o = i, 128 + o   # floats of fewer columns take tiles
    rows = ((400 if size == 4 else 270) << 20) // ((i + 2 * o) * size) // 64 * 64 + more
    print(f"[linear] {rows} x {i} -> {o} {dtype}", flush=True)
    g = torch.Generator("cuda").manual_seed(5)
    x = torch.randn(rows, i, generator=g, device="cuda").to(dtype)
    r = torch.randn(rows, o, generator=g, device="cuda").to(dtype)
    w, b = normal(11, o, i).to(dtype).cuda(), normal(21, o).cuda()
    y = ops.linear(x, w, b, activation="silu", residual=r)
    at = torch.cat([torch.arange(200), torch.arange(rows // 2, rows // 2 + 200), torch.arange(rows - 200, rows)]).cuda()
    want, bound = R.linear(x[at], w, b, "silu", r[at], dtype)[:2]
    R.check(y[at], want, bound, "y")
    assert bool(torch.isfinite(y).all())


# a narrow layer with many more outputs than inputs: several workgroups share the rows
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(33001, 84, 2001), (20003, 128, 4096), (70003, 30, 1030)], ids=str)
def test_linear_many_rows_and_columns(ops, shape, dtype):
    rows, i, o = shape
    if dtype == torch.float32:
        o = o // 2
    print(f"[linear] {rows} x {i} -> {o} {dtype}", flush=True)
    g = torch.Generator("cuda").manual_seed(5)
    x = torch.randn(rows, i, generator=g, device="cuda").to(dtype)
    r = torch.randn(rows, o, generator=g, device="cuda").to(dtype)
    w, b = (normal(11, o, i) * i ** -0.5).to(dtype).cuda(), normal(21, o).cuda()
    y, z = ops.linear(x, w, b, activation="gelu", residual=r, keep_preact=True)
    at = torch.cat([torch.arange(100), torch.arange(rows // 2, rows // 2 + 100), torch.arange(rows - 100, rows)]).cuda()
    wy, by, wz, bz = R.linear(x[at], w, b, "gelu", r[at], dtype)
    R.check(y[at], wy, by, "y")
    R.check(z[at], wz, bz, "z")
    assert bool(torch.isfinite(y).all()) and bool(torch.isfinite(z).all())


# many rows of few columns, in and out together at most 256 bytes (floats: half the columns named here)
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(300007, 32, 32), (300001, 64, 64), (400000, 3, 64), (300003, 59, 3), (350001, 1, 1),
                                   (300008, 100, 27)], ids=str)
@pytest.mark.parametrize("name,pad", [("none", 0), ("gelu", 3)])
def test_linear_backward_many_rows_of_few_columns(ops, shape, name, pad, dtype):
    rows, i, o = shape
    if dtype == torch.float32:
        i, o = (i + 1) // 2, (o + 1) // 2
    print(f"[linear_backward] {rows} x {i} -> {o} {dtype} {name} pad {pad}", flush=True)

    def padded(seed, cols, scale):
        full = torch.full((rows, cols + pad), NAN, dtype=dtype, device="cuda")
        full[:, :cols] = (scale * torch.randn(rows, cols, generator=torch.Generator("cuda").manual_seed(seed), device="cuda"))
        return full[:, :cols]

    x, gy, z = padded(1, i, 1.0), padded(2, o, 0.1), padded(3, o, 2.0) if name != "none" else None
    w = (normal(4, o, i) * i ** -0.5).to(dtype).cuda()
    full = torch.full((rows, i + pad), -7.0, dtype=dtype, device="cuda")
    got = ops.linear_backward(gy, x, w, preact=z, activation=name, grad_x=full[:, :i])
    for t, (want, bound), what in zip(got, R.linear_backward(gy, x, w, z, name, dtype), ("gx", "gw", "gb")):
        R.check(t, want, bound, what)
    assert bool((full[:, i:] == -7.0).all())
    again = ops.linear_backward(gy, x, w, preact=z, activation=name)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    for n in range(3):
        part = ops.linear_backward(gy, x, w, preact=z, activation=name, need_x=n == 0, need_weight=n == 1, need_bias=n == 2)
        assert torch.equal(part[n], got[n])


def test_linear_more_rows_than_a_launch_of_tiles(ops):
    """2^30 rows and some, of one column: 256 threads for 64 rows would be 2^32 threads."""
    rows = (1 << 30) + 100
    x = torch.arange(rows, dtype=torch.int32, device="cuda").remainder_(1021).to(torch.float32)[:, None]
    y = torch.full((rows, 1), -7.0, device="cuda")
    print("[linear] 2^30 + 100 x 1 -> 1", flush=True)
    ops.linear(x, torch.full((1, 1), 2.0, device="cuda"), torch.ones(1, device="cuda"), out=y)
    assert torch.equal(y, x.mul_(2.0).add_(1.0))


@pytest.mark.parametrize("dtype,n", [(torch.float32, 8193), (torch.bfloat16, 16385)], ids=["f32", "bf16"])
def test_layer_norm_more_wide_rows_than_workgroups(ops, dtype, n):
    """Rows above 32 KB, more of them than a launch has workgroups for."""
    rows = 65536 + 77
    x = torch.randn(64, n, device="cuda", generator=torch.Generator("cuda").manual_seed(3)).to(dtype).repeat(rows // 64 + 1, 1)[:rows]
    print(f"[layer_norm] {rows} x {n} {dtype}", flush=True)
    y, mean, rstd = ops.layer_norm(x)
    for t, (v, bound), what in zip((y, mean, rstd), R.layer_norm(x[:64], None, None, 1e-5, dtype), ("y", "mean", "rstd")):
        R.check(t[:64], v, bound, what)
        assert all(torch.equal(t[at:at + 64], t[:64][:rows - at]) for at in range(64, rows, 64)), what
    gx, gg, gb = ops.layer_norm_backward(y, x, None, mean, rstd)
    want, bound = R.layer_norm_backward(y[:64], x[:64], None, mean[:64], rstd[:64], None, dtype)[0]
    R.check(gx[:64], want, bound, "gx")
    assert all(torch.equal(gx[at:at + 64], gx[:64][:rows - at]) for at in range(64, rows, 64))


def test_relu_gradients_are_the_slopes(ops):
    """The gradients against differences of the forward, every value far from the kink: the loss is a plane there, so
    the step may be as wide as 2^-4 and leaves the forward's rounding (35 sums of size 20, 2^-24 each, over 2^-3)."""
    rows, i, o = 5, 6, 7
    x, w, c = normal(1, rows, i).cuda(), normal(2, o, i).cuda(), normal(4, rows, o).cuda()
    b = (12.0 * (1 - 2 * (torch.arange(o) % 2)) + normal(3, o)).cuda()

    def loss():
        return float((ops.linear(x, w, b, activation="relu").double() * c.double()).sum())

    _, z = ops.linear(x, w, b, activation="relu", keep_preact=True)
    h = 2.0 ** -4
    assert float(z.abs().min()) > 2 * h * max(1.0, float(x.abs().max()), float(w.abs().max()))
    assert bool((z > 0).any()) and bool((z < 0).any())
    for t, g in zip((x, w, b), ops.linear_backward(c, x, w, preact=z, activation="relu")):
        for at in range(t.numel()):
            flat, want = t.view(-1), float(g.reshape(-1)[at])
            keep = float(flat[at])
            flat[at] = keep + h
            up = loss()
            flat[at] = keep - h
            down = loss()
            flat[at] = keep
            assert abs((up - down) / (2 * h) - want) <= 1e-3 * (1 + abs(want)), (tuple(t.shape), at)


@pytest.mark.parametrize("shape", [(64, 64), (128, 300), (200, 129), (257, 255), (520, 520), (40, 1030), (700, 130),
                                   (1024, 1024), (1100, 2100)], ids=str)
@pytest.mark.parametrize("low_rank", [False, True])
def test_muon_is_as_near_as_floats(hip, shape, low_rank):
    """The update alone (no weights, rate 1) against 64 bits, beside the same formula in float products: operands of 22
    bits are four times as coarse as those of 24, and sums in another order are allowed twice the float's error. A
    product without one of its low halves is off some hundred times as much."""
    from tinygs_amd.optim import Muon
    r, c = shape
    g = normal(1, r, c) * (3e-3 if low_rank else 1.0)
    if low_rank:
        g = g + 2e-3 * normal(2, r, 1) * normal(3, 1, c)
    w = torch.zeros(r, c, device="cuda")
    opt = Muon([w], [g.cuda()])
    opt.set_params({"lr": 1.0, "momentum": 0.0, "weight_decay": 0.0, "nesterov": 0})
    opt.step(1.0)
    got = -w.double().cpu() / max(1.0, r / c) ** 0.5

    def update(dtype):
        x = (g.double() / g.double().norm()).to(dtype)
        x = x.t() if r > c else x
        for _ in range(5):
            a = x @ x.t()
            x = 3.4445 * x + (-4.7750 * a + 2.0315 * (a @ a)) @ x
        return (x.t() if r > c else x).double()

    want = update(torch.float64)
    plain, off = float((update(torch.float32) - want).norm()), float((got - want).norm())
    assert off <= 8 * plain, (off / float(want.norm()), plain / float(want.norm()))


def test_a_failed_allocation_fails_its_own_call_only(ops):
    """Muon's workspace for matrices that no card holds (their addresses are never read): that step fails, and the next
    call of another operator does not."""
    import ctypes as C
    from tinygs_amd import _lib
    lib, n, count = _lib.load(), 1 << 14, 200

    def array(slot):
        return (_lib.tgs_matrix * count)(*[_lib.tgs_matrix((1 << 44) * (slot + 1) + (4 * n * n) * k, n, n, n,
                                                           _lib.TGS_DTYPE_FLOAT32) for k in range(count)])
    h = C.c_void_p()
    assert lib.tgs_muon_create(array(0), array(1), array(2), None, count, C.byref(h)) == 0
    print("[muon] a workspace of a terabyte", flush=True)
    assert lib.tgs_muon_step(h, 1.0, None) == _lib.TGS_ERR_HIP
    x, w = normal(1, 40, 30), normal(2, 20, 30)
    y = ops.linear(x.cuda(), w.cuda())
    R.check(y, *R.linear(x, w, None, "none", None, torch.float32)[:2], "y")
    assert lib.tgs_muon_destroy(h) == 0


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_linear_to_a_single_row_between_columns(ops, dtype):
    """One row of a buffer's right half from the matrix in its left half: they share no element."""
    buf = normal(1, 12, 48).to(dtype).cuda()
    w, x = buf[:, :24], normal(2, 1, 24).to(dtype).cuda()
    y = buf[5:6, 30:42]
    keep = buf.clone()
    ops.linear(x, w, out=y)
    R.check(y, *R.linear(x, keep[:, :24], None, "none", None, dtype)[:2], "y")
    buf[5:6, 30:42] = keep[5:6, 30:42]
    assert torch.equal(buf, keep)
