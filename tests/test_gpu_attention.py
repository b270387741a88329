"""Attention to an encoder's states and its gradients against 64 bits: types, heads and shared heads, odd widths, lengths
of zero, one and many, masks that leave rows empty, NaN in states that do not exist, strides, streams, graphs."""
import itertools
import math

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


def buffer(rows, cols, pad, dtype, g=None, scale=1.0):
    """The first columns of a wider buffer of sentinels."""
    full = torch.full((rows, cols + pad), SENTINEL, dtype=dtype, device="cuda")
    if g is not None:
        full[:, :cols] = (scale * torch.randn(rows, cols, generator=g)).to(dtype).cuda()
    return full, full[:, :cols]


def untouched(full, cols):
    return bool((full[:, cols:] == SENTINEL).all())


def case(seed, dtype, batch, queries, states, heads, kv_heads, d, pad=0, q_scale=1.5):
    g = torch.Generator().manual_seed(seed)
    q = buffer(batch * queries, heads * d, pad, dtype, g, q_scale)[1]
    k = buffer(batch * states, kv_heads * d, pad, dtype, g, 1.5)[1]
    v = buffer(batch * states, kv_heads * d, pad, dtype, g)[1]
    go = buffer(batch * queries, heads * d, pad, dtype, g, 0.1)[1]
    return q, k, v, go


def mask_of(seed, batch, states, share, empty=()):
    g = torch.Generator().manual_seed(1000 + seed)
    m = torch.rand(batch, states, generator=g) < share
    for b in empty:
        m[b] = False
    return m.cuda()


def forget(t, mask, value):
    """What does not exist holds `value`."""
    rows = (~mask).reshape(-1)
    t[rows] = value


def run_both(ops, q, k, v, go, heads, kv_heads, batch=1, mask=None, scale=None, pad=0, what=None):
    """Forward and backward into sentinels, both checked; returns the results."""
    args = dict(kv_heads=kv_heads, batch=batch, mask=mask, scale=scale)
    out_full, out = buffer(*q.shape, pad, q.dtype)
    got, lse = ops.attention(q, k, v, heads, keep_lse=True, out=out, **args)
    assert got is out
    (o, ob), (l, lb) = A.attention(q, k, v, heads, kv_heads, batch, mask, scale)
    A.check(out, o, ob, (what, "out"))
    dead = l == -math.inf
    assert bool((lse.cpu().double()[dead] == -math.inf).all()), what
    A.check(torch.where(dead, torch.zeros_like(l), lse.cpu().double()), l.masked_fill(dead, 0.0),
            lb.masked_fill(dead, 0.0), (what, "lse"))
    assert untouched(out_full, q.shape[1]), what
    fulls = [buffer(*t.shape, pad, t.dtype) for t in (q, k, v)]
    grads = ops.attention_backward(go, q, k, v, out, lse, heads, grad_q=fulls[0][1], grad_k=fulls[1][1],
                                   grad_v=fulls[2][1], **args)
    want = A.attention_backward(go, q, k, v, out, lse, heads, kv_heads, batch, mask, scale)
    for name, g, (x, b), f in zip("qkv", grads, want, fulls):
        A.check(g, x, b, (what, "grad_" + name))
        assert untouched(f[0], g.shape[1]), (what, name)
    return out, lse, grads


# queries, states, heads, kv_heads, d
SHAPES = [(1, 1, 1, 1, 1), (1, 1, 2, 1, 8), (1, 7, 1, 1, 3), (3, 1, 2, 2, 16), (5, 33, 3, 1, 21), (16, 64, 2, 2, 32),
          (33, 65, 4, 4, 64), (64, 128, 4, 2, 64), (65, 31, 2, 1, 80), (70, 130, 2, 2, 96), (129, 257, 2, 1, 128),
          (31, 200, 8, 2, 40), (200, 17, 1, 1, 127), (257, 64, 6, 3, 33), (1, 1000, 4, 4, 64), (2, 777, 4, 1, 128),
          (700, 96, 1, 1, 64), (300, 300, 2, 2, 5), (40, 256, 16, 16, 16)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_shapes(ops, dtype, shape):
    queries, states, heads, kv_heads, d = shape
    for batch, pad in ((1, 0), (2, 3)):
        print(f"[attention] {shape} {dtype} batch {batch} pad {pad}", flush=True)
        t = case(sum(shape) + batch, dtype, batch, queries, states, heads, kv_heads, d, pad)
        run_both(ops, *t, heads, kv_heads, batch, pad=pad, what=(shape, batch))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(1, 40, 2, 1, 24), (37, 100, 2, 2, 64), (130, 300, 4, 2, 128), (3, 513, 1, 1, 32)],
                         ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("hidden", [float("nan"), float("inf"), "lowest"], ids=str)
def test_masks(ops, dtype, shape, hidden):
    """States that do not exist hold NaN, infinities or the type's lowest value; one element of the batch has none
    at all: its rows are 0 and so are its gradients."""
    queries, states, heads, kv_heads, d = shape
    batch = 4
    value = torch.finfo(dtype).min if hidden == "lowest" else hidden
    q, k, v, go = case(sum(shape), dtype, batch, queries, states, heads, kv_heads, d, 5)
    m = mask_of(states, batch, states, 0.6, empty=(2,))
    m[3, :] = False
    m[3, states - 1] = True
    forget(k, m, value)
    forget(v, m, value)
    print(f"[attention] masks {shape} {dtype} {hidden}", flush=True)
    out, lse, (gq, gk, gv) = run_both(ops, q, k, v, go, heads, kv_heads, batch, m, pad=5, what=(shape, hidden))
    rows = slice(2 * queries, 3 * queries)
    assert not out[rows].any() and not gq[rows].any() and bool((lse[rows] == -math.inf).all())
    gone = (~m).reshape(-1)
    assert not gk[gone].any() and not gv[gone].any()
    # uint8 masks, other nonzero values, one row for all elements
    again = ops.attention(q, k, v, heads, kv_heads=kv_heads, batch=batch, mask=m.to(torch.uint8) * 7)
    assert torch.equal(again, out)
    one = m[:1].expand(batch, states)
    k.nan_to_num_(0.5, 0.5, 0.5)
    v.nan_to_num_(0.5, 0.5, 0.5)
    # (lowest values that exist now may overflow to NaN: the same ones in both)
    a, b = (ops.attention(q, k, v, heads, kv_heads=kv_heads, batch=batch, mask=x).nan_to_num(9.0)
            for x in (one, one.contiguous()))
    assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_nothing(ops, dtype):
    """No queries, and no states: rows without a state are 0."""
    q, k, v, go = case(1, dtype, 2, 5, 0, 2, 2, 16)
    out, lse = ops.attention(q, k, v, 2, batch=2, keep_lse=True)
    assert not out.any() and bool((lse == -math.inf).all())
    gq, gk, gv = ops.attention_backward(go, q, k, v, out, lse, 2, batch=2)
    assert not gq.any() and gk.shape == (0, 32) and gv.shape == (0, 32)
    q, k, v, go = case(2, dtype, 2, 0, 9, 4, 2, 16)
    out, lse = ops.attention(q, k, v, 4, kv_heads=2, batch=2, keep_lse=True)
    assert out.shape == (0, 64) and lse.shape == (0, 4)
    gq, gk, gv = ops.attention_backward(go, q, k, v, out, lse, 4, kv_heads=2, batch=2)
    assert not gk.any() and not gv.any()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_large_and_small_scores(ops, dtype):
    """Scores far from zero, where the exponentials of all but a few states vanish, and a scale of zero, where all weigh
    the same; a scale of its own."""
    for q_scale, scale in ((40.0, None), (1.0, 0.0), (1.0, 3.0), (0.001, None)):
        t = case(5, dtype, 1, 50, 150, 2, 1, 48, q_scale=q_scale)
        run_both(ops, *t, 2, 1, scale=scale, what=(q_scale, scale))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_infinite_and_nan_values(ops, dtype):
    """What is not finite stays in the rows, heads and columns that it enters."""
    q, k, v, _ = case(9, dtype, 1, 70, 90, 2, 2, 32)
    want = ops.attention(q, k, v, 2)
    q[3, 5] = float("nan")             # row 3 of head 0
    got = ops.attention(q, k, v, 2)
    assert bool(torch.isnan(got[3, :32]).all())
    got[3, :32] = want[3, :32]
    assert torch.equal(got, want)
    q, k, v, _ = case(9, dtype, 1, 70, 90, 2, 2, 32)
    v[17, 40] = float("nan")           # column 8 of head 1
    got = ops.attention(q, k, v, 2)
    assert bool(torch.isnan(got[:, 40]).all())
    got[:, 40] = want[:, 40]
    assert torch.equal(got, want)
    q, k, v, _ = case(9, dtype, 1, 70, 90, 2, 2, 32)
    k[:, 0] = float("-inf")            # scores of +-infinity everywhere in head 0
    got, lse = ops.attention(q, k, v, 2, keep_lse=True)
    dead = q[:, 0] > 0
    assert bool(dead.any()) and not got[dead, :32].any() and bool((lse[dead, 0] == -math.inf).all())
    assert bool(torch.isnan(got[~dead, :32]).all()) and torch.equal(got[:, 32:], want[:, 32:])


def test_one_head_of_wider_tensors(ops):
    """q, k and v as column ranges of one buffer, as a joint projection leaves them; the gradients go back into one."""
    g = torch.Generator().manual_seed(4)
    d, rows = 64, 75
    both = torch.randn(rows, 6 * d, generator=g).to(torch.bfloat16).cuda()
    q, k, v = both[:, :2 * d], both[:, 2 * d:4 * d], both[:, 4 * d:]
    go = torch.randn(rows, 2 * d, generator=g).to(torch.bfloat16).cuda()
    out, lse = ops.attention(q, k, v, 2, keep_lse=True)
    assert torch.equal(out, ops.attention(q.contiguous(), k.contiguous(), v.contiguous(), 2))
    grads = torch.full_like(both, SENTINEL)
    ops.attention_backward(go, q, k, v, out, lse, 2, grad_q=grads[:, :2 * d], grad_k=grads[:, 2 * d:4 * d],
                           grad_v=grads[:, 4 * d:])
    apart = ops.attention_backward(go, q.contiguous(), k.contiguous(), v.contiguous(), out, lse, 2)
    assert torch.equal(grads, torch.cat(apart, 1))


def test_needed_gradients_alone(ops):
    t = case(6, torch.float16, 2, 60, 90, 4, 2, 32)
    q, k, v, go = t
    out, lse = ops.attention(q, k, v, 4, kv_heads=2, batch=2, keep_lse=True)
    every = ops.attention_backward(go, q, k, v, out, lse, 4, kv_heads=2, batch=2)
    for need in itertools.product((False, True), repeat=3):
        got = ops.attention_backward(go, q, k, v, out, lse, 4, kv_heads=2, batch=2, need_q=need[0], need_k=need[1],
                                     need_v=need[2])
        for x, y, n in zip(got, every, need):
            assert (x is None) if not n else torch.equal(x, y)


def test_tensors_elsewhere_are_refused(ops):
    """A tensor that is not on the current device, among those that are."""
    q, k, v, go = case(1, torch.float16, 1, 4, 6, 2, 2, 16)
    out, lse = ops.attention(q, k, v, 2, keep_lse=True)
    with pytest.raises(RuntimeError, match="mask: not on the current device"):
        ops.attention(q, k, v, 2, mask=torch.ones(1, 6, dtype=torch.bool))
    with pytest.raises(RuntimeError, match="lse"):
        ops.attention_backward(go, q, k, v, out, lse.cpu(), 2)
    with pytest.raises(RuntimeError, match="not on the device"):
        ops.attention(q, k.cpu(), v, 2)
    with pytest.raises(RuntimeError, match="lse"):
        ops.attention(q, k, v, 2, lse=torch.empty(4, 3, device="cuda"))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_many_small_elements(ops, dtype):
    """More elements of a batch than a card has room for at once, a row or two of each."""
    for queries, states, heads, kv_heads, d in ((1, 9, 2, 2, 16), (2, 40, 2, 1, 24), (40, 9, 1, 1, 64)):
        t = case(queries, dtype, 3000, queries, states, heads, kv_heads, d)
        m = mask_of(1, 3000, states, 0.6, empty=(5, 2999))
        run_both(ops, *t, heads, kv_heads, 3000, m, what=(queries, states))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_maxima_far_behind(ops, dtype):
    """Scores that rise with the states: the largest comes last, by more than a weight's range above the first ones, in
    some rows; the others' results do not change by a bit."""
    for rows, states, d in ((200, 300, 32), (40_003, 250, 64), (1, 400, 64), (30, 5000, 128)):
        heads = 4
        q, k, v, go = case(rows, dtype, 1, rows, states, heads, heads, d)
        want, wlse = ops.attention(q, k, v, heads, keep_lse=True)
        steep = q.clone()
        pick = torch.arange(0, rows, 7, device="cuda")
        steep[pick] = 0.0
        steep[pick, 0] = 24.0            # of head 0
        rising = k.clone()
        rising[:, 0] = torch.linspace(-6, 12, states).to(dtype).cuda()
        out, lse = ops.attention(steep, rising, v, heads, keep_lse=True)
        sample = torch.arange(0, rows, max(1, rows // 60), device="cuda")
        (o, ob), (l, lb) = A.attention(steep[sample].contiguous(), rising, v, heads, heads)
        A.check(out[sample], o, ob, (rows, "out"))
        A.check(lse[sample], l, lb, (rows, "lse"))
        # heads other than the first: the same inputs, but for the zeroed rows
        keep = torch.ones(rows, dtype=torch.bool, device="cuda")
        keep[pick] = False
        assert torch.equal(out[keep][:, d:], want[keep][:, d:]) and torch.equal(lse[keep][:, 1:], wlse[keep][:, 1:])


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("d", [5, 32, 64, 98, 128])
@pytest.mark.parametrize("masked", [False, True])
def test_one_state_has_no_gradient_of_scores(ops, dtype, d, masked):
    """Where a row has one state its weight is 1 whatever the score: grad_q and grad_k are 0, not the difference of two
    sums of the same terms."""
    states = 70 if masked else 1
    q, k, v, go = case(d, dtype, 2, 150, states, 4, 2, d)
    m = None
    if masked:
        m = torch.zeros(2, states, dtype=torch.bool, device="cuda")
        m[0, 40] = m[1, 69] = True
    out, lse = ops.attention(q, k, v, 4, kv_heads=2, batch=2, mask=m, keep_lse=True)
    for need_q in (True, False):
        gq, gk, gv = ops.attention_backward(go, q, k, v, out, lse, 4, kv_heads=2, batch=2, mask=m, need_q=need_q)
        assert (not need_q or not gq.any()) and not gk.any() and gv.any()


def test_gradients_against_differences(ops):
    """In 64 bits around float32 inputs: (f(x + e) - f(x - e)) / 2e of the sum of out with a direction is off by e^2 of
    the third derivative and 2^-24 / e of out; e = 2^-6 leaves less than 1 in 300 of the largest."""
    q, k, v, go = case(8, torch.float32, 1, 6, 9, 2, 1, 8)
    out, lse = ops.attention(q, k, v, 2, kv_heads=1, keep_lse=True)
    grads = ops.attention_backward(go, q, k, v, out, lse, 2, kv_heads=1)
    e = 2.0 ** -6
    for t, g in zip((q, k, v), grads):
        for r, c in ((0, 0), (t.shape[0] - 1, t.shape[1] - 1), (2, 3)):
            x = float(t[r, c])
            f = []
            for step in (e, -e):
                t[r, c] = x + step
                f.append(float((ops.attention(q, k, v, 2, kv_heads=1).double() * go.double()).sum()))
            t[r, c] = x
            d = (f[0] - f[1]) / (2 * e)
            assert abs(d - float(g[r, c])) <= float(g.abs().max()) / 300, (r, c, d, float(g[r, c]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_same_bits_streams_and_replays(ops, dtype):
    """The same inputs give the same bits: eagerly, on another stream, and in replays of two graphs that share the
    handle's workspace, with eager work between them."""
    sets = [case(s, dtype, 2, 300, 190, 4, 2, 32) for s in (1, 2)]
    m = mask_of(3, 2, 190, 0.7)

    def run(t, o=ops, **kw):
        q, k, v, go = t
        out, lse = o.attention(q, k, v, 4, kv_heads=2, batch=2, mask=m, keep_lse=True, **kw)
        return (out, lse) + o.attention_backward(go, q, k, v, out, lse, 4, kv_heads=2, batch=2, mask=m, **kw)

    want = [run(t) for t in sets]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for t, w in zip(sets, want):
        got = run(t, stream=s)
        s.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, w))
    graphs, outs = [], []
    for t in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(run(t, stream=s))
        graphs.append(g)
    for _ in range(3):
        for g, o, w, t in zip(graphs, outs, want, sets):
            for x in o:
                x.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(o, w))
            assert all(torch.equal(x, y) for x, y in zip(run(t), w))


def test_offsets_past_32_bits(ops):
    """Rows and states whose addresses lie more than 2^32 elements apart."""
    stride, d, states = (1 << 21) - 8, 32, 130
    big = torch.empty(2100 * stride, dtype=torch.float16, device="cuda")   # 8.8 GB
    rows = big.as_strided((2100, d), (stride, 1))
    g = torch.Generator().manual_seed(3)
    values = torch.randn(2100, d, generator=g).half().cuda()
    rows.copy_(values)
    k, v, go = (torch.randn(n, d, generator=g).half().cuda() for n in (states, states, 2100))
    out, lse = ops.attention(rows, k, v, 1, keep_lse=True)
    want, wlse = ops.attention(values, k, v, 1, keep_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, wlse)
    got = ops.attention_backward(go, rows, k, v, out, lse, 1)
    apart = ops.attention_backward(go, values, k, v, out, lse, 1)
    assert all(torch.equal(x, y) for x, y in zip(got, apart))
    # and as states
    out, lse = ops.attention(k, rows, values, 1, keep_lse=True)
    want, wlse = ops.attention(k, values, values, 1, keep_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, wlse)
    got = ops.attention_backward(go[:states], k, rows, values, out, lse, 1)
    apart = ops.attention_backward(go[:states], k, values, values, out, lse, 1)
    assert all(torch.equal(x, y) for x, y in zip(got, apart))


def test_many_rows(ops):
    """More rows than a launch has workgroups; a sample of them checked, and the states' gradients against float64 on
    the device."""
    rows, states, d = 300_001, 70, 16
    t = case(2, torch.bfloat16, 1, rows, states, 1, 1, d)
    q, k, v, go = t
    out, lse = ops.attention(q, k, v, 1, keep_lse=True)
    gq, gk, gv = ops.attention_backward(go, q, k, v, out, lse, 1)
    pick = torch.cat([torch.arange(0, rows, 4999), torch.tensor([rows - 1])])
    qs, gs, os, ls = (x[pick.cuda()].contiguous() for x in (q, go, out, lse))
    (o, ob), (l, lb) = A.attention(qs, k, v, 1, 1)
    A.check(os, o, ob, "out")
    A.check(ls, l, lb, "lse")
    x, b = A.attention_backward(gs, qs, k, v, os, ls, 1, 1)[0]
    A.check(gq[pick.cuda()], x, b, "grad_q")
    p = torch.exp(q.double() @ k.double().t() / 4.0 - lse.double())
    gvw = p.t() @ go.double()
    ds = p * (go.double() @ v.double().t() - (go.double() * out.double()).sum(1, keepdim=True))
    gkw = ds.t() @ q.double() / 4.0
    # rounded weights: independent errors of at most half a unit each, bounded by their sum
    for got, want, terms in ((gv, gvw, p.t() @ go.double().abs()), (gk, gkw, ds.abs().t() @ q.double().abs() / 4.0)):
        bound = (2 ** -8 + 2 ** -12) * terms + 2 ** -8 * want.abs()
        assert bool(((got.double() - want).abs() <= bound).all())


# batch, queries, states, heads, kv_heads, d, share of the states (None: no mask)
LARGE = [(1, 70_003, 256, 4, 4, 64, None), (1, 70_003, 197, 4, 1, 64, 0.7), (2, 70_001, 130, 2, 2, 32, 0.5),
         (3, 50_001, 65, 2, 1, 96, None), (1, 140_007, 256, 1, 1, 128, 0.9), (1, 60_001, 500, 3, 3, 24, None),
         (1, 140_001, 1, 1, 1, 64, None), (2, 33_333, 320, 4, 2, 80, 0.8), (1, 9_001, 90, 16, 16, 64, None)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", LARGE, ids=lambda s: "x".join(map(str, s)))
def test_many_rows_of_many_heads(ops, dtype, shape):
    """The card full of rows: a sample of them checked in each element of the batch, the states' gradients against
    float64 on the device. One element's states do not exist where there are several."""
    batch, rows, states, heads, kv_heads, d, share = shape
    q, k, v, go = case(rows + states, dtype, batch, rows, states, heads, kv_heads, d, 3)
    m = None
    if share is not None:
        m = mask_of(states, batch, states, share, empty=(1,) if batch > 1 else ())
        forget(k, m, float("nan"))
        forget(v, m, float("nan"))
    args = dict(kv_heads=kv_heads, batch=batch, mask=m)
    print(f"[attention] large {shape} {dtype}", flush=True)
    out, lse = ops.attention(q, k, v, heads, keep_lse=True, **args)
    gq, gk, gv = ops.attention_backward(go, q, k, v, out, lse, heads, **args)
    within = torch.cat([torch.arange(0, rows, 2777), torch.tensor([rows - 1])])
    pick = (within[None, :] + rows * torch.arange(batch)[:, None]).reshape(-1).cuda()
    qs, gs, os, ls = (x[pick].contiguous() for x in (q, go, out, lse))
    (o, ob), (l, lb) = A.attention(qs, k, v, heads, kv_heads, batch, m)
    A.check(os, o, ob, "out")
    dead = l == -math.inf
    assert torch.equal(ls.cpu() == -math.inf, dead)
    A.check(torch.where(dead, torch.zeros_like(l), ls.cpu().double()), l.masked_fill(dead, 0.0), lb.masked_fill(dead, 0.0),
            "lse")
    x, b = A.attention_backward(gs, qs, k, v, os, ls, heads, kv_heads, batch, m)[0]
    A.check(gq[pick], x, b, "grad_q")
    unit = A.UNIT[dtype]
    for e in range(batch):
        at, of = slice(e * rows, (e + 1) * rows), slice(e * states, (e + 1) * states)
        there = torch.ones(states, dtype=torch.bool, device="cuda") if m is None else m[e]
        for g in range(kv_heads):
            cols = slice(g * d, (g + 1) * d)
            ke, ve = (t[of, cols].double()[there] for t in (k, v))
            sums = [torch.zeros_like(ke) for _ in range(4)]
            own = torch.zeros_like(ke)
            for h in range(g * heads // kv_heads, (g + 1) * heads // kv_heads):
                hc = slice(h * d, (h + 1) * d)
                qe, oe, ye = (t[at, hc].double() for t in (q, go, out))
                p = torch.exp(qe @ ke.t() / math.sqrt(d) - lse[at, h].double()[:, None])
                ds = p * (oe @ ve.t() - (oe * ye).sum(1, keepdim=True))
                sums[0] += p.t() @ oe
                sums[1] += p.t() @ oe.abs()
                sums[2] += ds.t() @ qe / math.sqrt(d)
                sums[3] += ds.abs().t() @ qe.abs() / math.sqrt(d)
                # dp and delta are sums of d products each: off by (d + 17) 2^-24 of their terms' sizes, whatever
                # is left of them in the difference (nothing, for a single state)
                size = oe.abs() @ ve.abs().t() + (oe * ye).abs().sum(1, keepdim=True)
                own += (d + 20) * A.EPS24 * (p * size).t() @ qe.abs() / math.sqrt(d)
            # weights are rounded once: by a unit each at most, with the scores' error (d + 17 roundings of terms of
            # a few units' size, 2^-15 at the most here) and the sums' over as many rows, each far below a unit of
            # 16-bit types; floats: 2^-14 of the terms
            rel = max(unit + 2.0 ** -14, 2.0 ** -14)
            step = 2.0 ** -24 * 70 if dtype == torch.float16 else 0.0   # products' and results' smallest steps
            for got, want, terms, more in ((gv, sums[0], sums[1], 0.0), (gk, sums[2], sums[3], own)):
                y = got[of, cols].double()
                assert not y[~there].any()
                bound = rel * terms + 1.01 * more + unit * want.abs() + step
                assert bool(((y[there] - want).abs() <= bound).all()), (shape, e, g)
