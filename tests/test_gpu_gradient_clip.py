"""The norm of many gradients and clipping against 64 bits: mixed types, empty and strided tensors, bounds reached and
not, ranges, outputs apart, rebinding, replays."""
import math

import pytest
import torch

from network_reference import EPS24, STEP, UNIT, check

pytestmark = pytest.mark.gpu

SHAPES = [(1,), (0,), (7,), (3, 5), (64, 64), (8191,), (8192,), (8193,), (300, 45), (2, 3, 4, 5), (1, 20000), (50_001, 3), ()]


def tensors(seed, dtypes=(torch.float32, torch.float16, torch.bfloat16), scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(scale * torch.randn(s, generator=g)).to(dtypes[i % len(dtypes)]).cuda() for i, s in enumerate(SHAPES)]


def norm_of(grads, scale=1.0):
    return scale * math.sqrt(sum(float((t.double() ** 2).sum()) for t in grads))


def agrees(got, before, factor, what):
    """A factor in 32 bits (its double is off by far less), one product, one rounding."""
    for i, (t, b) in enumerate(zip(got, before)):
        want = b.double().cpu() * factor
        check(t, want, 2 * EPS24 * want.abs() + UNIT[t.dtype] * want.abs() * (1 + 4 * EPS24) + STEP[t.dtype], (what, i))


@pytest.mark.parametrize("scale", [1.0, 1.0 / 1024.0, 3.0])
@pytest.mark.parametrize("ratio", [0.1, 0.999, 1.5, math.inf])
@pytest.mark.parametrize("apart", [False, True])
def test_clip(hip, scale, ratio, apart):
    from tinygs_amd.optim import GradientClip
    grads = tensors(1)
    before = [t.clone() for t in grads]
    kinds = (torch.bfloat16, torch.float32, torch.float16)
    clipped = [torch.full_like(t, 7.0, dtype=kinds[i % 3]) for i, t in enumerate(grads)] if apart else None
    c = GradientClip(grads, clipped=clipped)
    n = norm_of(before, scale)
    bound = ratio * n
    print(f"[clip] scale {scale} ratio {ratio} apart {apart}", flush=True)
    got = c.clip(bound, scale=scale)
    assert got.shape == () and got.dtype == torch.float32 and abs(float(got) - n) <= 2 * EPS24 * n
    factor = scale * min(1.0, bound / (n + 1e-6) if math.isfinite(bound) else 1.0)
    agrees(clipped if apart else grads, before, factor, (scale, ratio))
    if apart:
        assert all(torch.equal(a, b) for a, b in zip(grads, before))
    elif factor == 1.0:
        assert all(torch.equal(a, b) for a, b in zip(grads, before))


def test_strided_and_padded(hip):
    from tinygs_amd.optim import GradientClip
    g = torch.Generator().manual_seed(3)
    wide = torch.randn(300, 96, generator=g).cuda()
    kept = wide.clone()
    cut, narrow = wide[:, 5:70], wide[:, 80:81]
    c = GradientClip([cut, narrow])
    n = norm_of([cut, narrow])
    assert abs(float(c.clip(0.5)) - n) <= 2 * EPS24 * n
    agrees([cut, narrow], [kept[:, 5:70], kept[:, 80:81]], 0.5 / (n + 1e-6), "strided")
    rest = torch.ones(96, dtype=torch.bool)
    rest[5:70] = rest[80] = False
    assert torch.equal(wide[:, rest.cuda()], kept[:, rest.cuda()])
    # out of strided tensors into packed ones and back
    packed = torch.zeros(300, 65, dtype=torch.float16, device="cuda")
    d = GradientClip([kept[:, 5:70]], clipped=[packed])
    d.clip(1.0)
    agrees([packed], [kept[:, 5:70]], 1.0 / (norm_of([kept[:, 5:70]]) + 1e-6), "packed")
    into = torch.full((300, 80), 9.0, device="cuda")
    d = GradientClip([packed], clipped=[into[:, 3:68]])
    d.clip(math.inf)
    assert torch.equal(into[:, 3:68], packed.float()) and bool((into[:, 68:] == 9.0).all() and (into[:, :3] == 9.0).all())


@pytest.mark.parametrize("size", [2.0 ** -140, 2.0 ** -90, 2.0 ** 90, 2.0 ** 120])
def test_ranges(hip, size):
    """Squares far past the range of floats."""
    from tinygs_amd.optim import GradientClip
    g = [torch.full((4097,), size, device="cuda"), torch.full((33, 3), -size, device="cuda")]
    n = norm_of(g)
    got = GradientClip(g).clip(math.inf)
    assert abs(float(got) - n) <= 2 * EPS24 * n + STEP[torch.float32]
    c = GradientClip(g)
    c.clip(n / 4 if n < 1e38 else 1e37, epsilon=0.0)
    factor = 0.25 if n < 1e38 else 1e37 / n
    assert abs(float(g[0][5]) / size - factor) <= 4 * EPS24 + 2.0 ** -9 * (size < 1e-40)


def test_not_finite(hip):
    from tinygs_amd.optim import GradientClip
    for value, rest in ((math.nan, math.nan), (math.inf, 0.0)):
        g = tensors(4)
        g[4][3, 3] = value
        got = float(GradientClip(g).clip(1.0))
        assert (math.isnan(got) if math.isnan(value) else got == math.inf)
        assert bool(torch.isnan(g[4][3, 3]))
        if math.isnan(rest):
            assert all(bool(torch.isnan(t).all()) for t in g)
        else:
            assert not g[8].any() and not g[0].any()
    g = tensors(4)
    g[4][3, 3] = math.nan
    kept = [t.clone() for t in g]
    assert math.isnan(float(GradientClip(g).clip(math.inf)))
    assert all(torch.equal(a.nan_to_num(1.0), b.nan_to_num(1.0)) for a, b in zip(g, kept))


def test_zero_gradients_and_bound(hip):
    from tinygs_amd.optim import GradientClip
    z = [torch.zeros(100, device="cuda"), torch.zeros(0, device="cuda")]
    c = GradientClip(z)
    assert float(c.clip(1.0)) == 0.0 and not z[0].any()
    g = [torch.ones(100, device="cuda")]
    assert float(GradientClip(g).clip(0.0)) == 10.0 and not g[0].any()
    assert float(GradientClip([torch.zeros(0, device="cuda")]).clip(1.0)) == 0.0


def test_many_tensors_and_rebinding(hip):
    from tinygs_amd.optim import GradientClip
    g = torch.Generator().manual_seed(9)
    many = [torch.randn(1 + i % 97, generator=g).cuda() for i in range(700)]
    before = [t.clone() for t in many]
    c = GradientClip(many)
    n = norm_of(many)
    assert abs(float(c.clip(1.0)) - n) <= 2 * EPS24 * n
    agrees(many, before, 1.0 / (n + 1e-6), "many")
    other = tensors(10)
    c.set_grads(other)
    n = norm_of(other)
    before = [t.clone() for t in other]
    assert abs(float(c.clip(0.3)) - n) <= 2 * EPS24 * n
    agrees(other, before, 0.3 / (n + 1e-6), "rebound")


def test_same_bits_streams_and_replays(hip):
    """Two handles captured into two graphs, replayed in turn between eager runs."""
    from tinygs_amd.optim import GradientClip
    s = torch.cuda.Stream()
    made = []
    for k in range(2):
        src = tensors(20 + k)
        g = [t.clone() for t in src]
        c = GradientClip(g)
        eager = [t.clone() for t in src]
        e = GradientClip(eager)
        torch.cuda.synchronize()
        c.clip(0.5, stream=s)
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            norm = c.clip(0.5, stream=s)
        made.append((src, g, c, graph, norm, eager, e))
    for turn in range(3):
        for src, g, _, graph, norm, eager, e in made:
            for a, b, x in zip(g, eager, src):
                a.copy_(x * (turn + 1))
                b.copy_(x * (turn + 1))
            torch.cuda.synchronize()
            graph.replay()
            want = e.clip(0.5)
            torch.cuda.synchronize()
            assert torch.equal(norm, want)
            assert all(torch.equal(a, b) for a, b in zip(g, eager)), turn


def test_large(hip):
    """More than 2^32 bytes in one tensor."""
    from tinygs_amd.optim import GradientClip
    big = torch.ones(1_200_000_000, dtype=torch.float32, device="cuda")
    assert abs(float(GradientClip([big]).clip(1.0, epsilon=0.0)) - math.sqrt(1.2e9)) <= 2 * EPS24 * math.sqrt(1.2e9)
    assert float(big[0]) == float(big[-1]) == float(torch.tensor(1.0 / math.sqrt(1.2e9)))
