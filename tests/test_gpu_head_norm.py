"""Head norms with their turning, and gradients, against 64 bits: types, widths, partial turns, far positions, strides,
outputs in the inputs' place, streams and replays."""
import pytest
import torch

import attention_reference as A

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
IDS = ["f32", "f16", "bf16"]
SENTINEL = 3.0e4


@pytest.fixture(scope="module")
def ops(hip):
    from tinygs_amd.network import LayerOps
    return LayerOps()


def buffer(rows, cols, pad, dtype, values=None):
    full = torch.full((rows, cols + pad), SENTINEL, dtype=dtype, device="cuda")
    if values is not None:
        full[:, :cols] = values.to(dtype).cuda()
    return full, full[:, :cols]


def turn_of(g, rows, axes, pairs, extent):
    if not axes:
        return None, None
    return (((torch.rand(rows, axes, generator=g) * 2 - 1) * extent).cuda(),
            (torch.randn(pairs, axes, generator=g) * torch.logspace(0.8, -1.2, pairs)[:, None]).cuda())


# rows, heads, d, axes, pairs, gamma, pad
SHAPES = [(1, 1, 1, 0, 0, True, 0), (1, 1, 2, 1, 1, False, 0), (3, 2, 7, 2, 3, True, 1), (5, 3, 8, 3, 4, True, 0),
          (33, 3, 38, 3, 15, False, 3), (64, 4, 64, 3, 32, True, 0), (100, 5, 64, 4, 32, True, 8), (31, 1, 128, 1, 64, True, 0),
          (17, 8, 128, 3, 20, True, 5), (9, 2, 256, 2, 128, True, 0), (12, 3, 255, 3, 127, True, 7), (7, 17, 16, 1, 8, True, 0),
          (2500, 2, 32, 3, 16, True, 0), (40, 4, 100, 0, 0, True, 4), (65, 6, 33, 1, 16, True, 0)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("extent", [2.0, 1e4])
def test_head_norm(ops, dtype, shape, extent):
    rows, heads, d, axes, pairs, has_gamma, pad = shape
    g = torch.Generator().manual_seed(sum(shape[:5]))
    x = buffer(rows, heads * d, pad, dtype, torch.randn(rows, heads * d, generator=g))[1]
    gy = buffer(rows, heads * d, pad, dtype, torch.randn(rows, heads * d, generator=g))[1]
    gamma = (1 + 0.3 * torch.randn(d, generator=g)).cuda() if has_gamma else None
    pos, freq = turn_of(g, rows, axes, pairs, extent)
    args = dict(gamma=gamma, positions=pos, frequencies=freq, eps=1e-6)
    print(f"[head norm] {shape} {dtype} {extent}", flush=True)
    full, out = buffer(rows, heads * d, pad, dtype)
    assert ops.head_norm(x, heads, out=out, **args) is out
    y, b = A.head_norm(x, heads, gamma, pos, freq, 1e-6)
    A.check(out, y, b, (shape, "out"))
    assert bool((full[:, heads * d:] == SENTINEL).all())
    full, gx = buffer(rows, heads * d, pad, dtype)
    _, gg = ops.head_norm_backward(gy, x, heads, grad_x=gx, **args)
    (wx, bx), (wg, bg) = A.head_norm_backward(gy, x, heads, gamma, pos, freq, 1e-6)
    A.check(gx, wx, bx, (shape, "grad_x"))
    assert bool((full[:, heads * d:] == SENTINEL).all())
    assert (gg is None) == (gamma is None)
    if gamma is not None:
        A.check(gg, wg, bg, (shape, "grad_gamma"))
        only = ops.head_norm_backward(gy, x, heads, need_x=False, **args)
        assert only[0] is None and torch.equal(only[1], gg)
    # in place: y over x, grad_x over grad_y
    again = x.clone()
    ops.head_norm(again, heads, out=again, **args)
    assert torch.equal(again, out)
    again = gy.clone()
    ops.head_norm_backward(again, x, heads, grad_x=again, **args)
    assert torch.equal(again, gx)


def test_sizes_past_the_range(ops):
    """Heads of zeros are zeros; infinite and NaN elements stay in their row and head."""
    x = torch.randn(20, 3 * 32, generator=torch.Generator().manual_seed(1)).cuda()
    x[4] = 0.0
    want = ops.head_norm(x, 3)
    assert not want[4].any()
    x[7, 40] = float("inf")
    x[9, 70] = float("nan")
    got = ops.head_norm(x, 3)
    assert bool(torch.isnan(got[7, 40])) and not got[7, 32:40].any() and bool(torch.isnan(got[9, 64:]).all())
    got[7, 32:64], got[9, 64:] = want[7, 32:64], want[9, 64:]
    assert torch.equal(got, want)


def test_turning_keeps_lengths_and_differences(ops):
    """Scores of turned queries and keys depend on the difference of their positions alone."""
    g = torch.Generator().manual_seed(2)
    d, n = 64, 50
    q, k = (torch.randn(n, d, generator=g).cuda() for _ in range(2))
    freq = torch.randn(d // 2, 3, generator=g).cuda()
    a, b = (torch.randint(-4, 5, (n, 3), generator=g).float().cuda() for _ in range(2))
    shift = torch.tensor([2.0, -8.0, 16.0], device="cuda")

    def scores(x, y):
        return (ops.head_norm(q, 1, positions=x, frequencies=freq).double() *
                ops.head_norm(k, 1, positions=y, frequencies=freq).double()).sum(1)

    # of unit-mean-square heads: 64 products, each off by a few units of at most its pair's sizes
    assert float((scores(a, b) - scores(a + shift, b + shift)).abs().max()) <= 64 * 64 * A.EPS24
    plain = ops.head_norm(q, 1).double().norm(dim=1)
    assert float((ops.head_norm(q, 1, positions=a, frequencies=freq).double().norm(dim=1) / plain - 1).abs().max()) <= 64 * A.EPS24


def test_gradients_against_differences(ops):
    """As for attention: e = 2^-6, off by less than 1 in 300 of the largest."""
    g = torch.Generator().manual_seed(5)
    x = torch.randn(4, 2 * 12, generator=g).cuda()
    gy = torch.randn(4, 2 * 12, generator=g).cuda()
    gamma = (1 + 0.3 * torch.randn(12, generator=g)).cuda()
    pos, freq = turn_of(g, 4, 3, 5, 3.0)
    args = dict(positions=pos, frequencies=freq)
    gx, gg = ops.head_norm_backward(gy, x, 2, gamma, **args)
    e = 2.0 ** -6
    for t, grad, places in ((x, gx, [(0, 0), (3, 23), (1, 11)]), (gamma, gg, [(0,), (11,), (4,)])):
        for at in places:
            kept = float(t[at])
            f = []
            for step in (e, -e):
                t[at] = kept + step
                f.append(float((ops.head_norm(x, 2, gamma, **args).double() * gy.double()).sum()))
            t[at] = kept
            d = (f[0] - f[1]) / (2 * e)
            assert abs(d - float(grad[at])) <= float(grad.abs().max()) / 300, (at, d, float(grad[at]))


def test_streams_replays_and_many_rows(ops):
    g = torch.Generator().manual_seed(6)
    rows, heads, d = 70_003, 2, 16
    x, gy = (torch.randn(rows, heads * d, generator=g).half().cuda() for _ in range(2))
    gamma = (1 + 0.3 * torch.randn(d, generator=g)).cuda()
    pos, freq = turn_of(g, rows, 2, 8, 30.0)

    def run(**kw):
        y = ops.head_norm(x, heads, gamma, pos, freq, **kw)
        return (y,) + ops.head_norm_backward(gy, x, heads, gamma, pos, freq, **kw)

    want = run()
    A.check(want[0], *A.head_norm(x, heads, gamma, pos, freq, 1e-6), "out")
    (wx, bx), (wg, bg) = A.head_norm_backward(gy, x, heads, gamma, pos, freq, 1e-6)
    A.check(want[1], wx, bx, "grad_x")
    A.check(want[2], wg, bg, "grad_gamma")
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    got = run(stream=s)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        held = run(stream=s)
    for _ in range(3):
        for t in held:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))
        assert all(torch.equal(a, b) for a, b in zip(run(), want))


def test_no_rows(ops):
    x = torch.empty(0, 64, device="cuda")
    gamma = torch.ones(32, device="cuda")
    assert ops.head_norm(x, 2, gamma).shape == (0, 64)
    gx, gg = ops.head_norm_backward(x, x, 2, gamma, grad_x=torch.empty(0, 64, device="cuda"))
    assert gx.shape == (0, 64) and not gg.any()
