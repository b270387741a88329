"""Gradients of 16-bit heads of up to 32 columns, however many rows there are: nothing is rounded to 16 bits but the
results. And the one-pass kernel's heads of partial tiles, and masks that leave one state."""
import math

import pytest
import torch

import attention_reference as A
from test_gpu_attention import case, forget, mask_of, ops  # noqa: F401

pytestmark = pytest.mark.gpu


def float64_gradients(q, k, v, go, out, lse, heads, kv_heads, d, mask=None):
    """Each (value, the sum of its terms' sizes, what dp and delta leave of their own roundings), in 64 bits on the
    device. dp and delta are sums of d products each: off by (d + 20) 2^-24 of their terms' sizes."""
    full = [torch.zeros(*t.shape, 3, dtype=torch.float64, device="cuda") for t in (q, k, v)]
    there = torch.ones(k.shape[0], dtype=torch.bool, device="cuda") if mask is None else mask
    for g in range(kv_heads):
        cols, group = slice(g * d, (g + 1) * d), range(g * heads // kv_heads, (g + 1) * heads // kv_heads)
        ke, ve = k[:, cols].double()[there], v[:, cols].double()[there]
        part = [torch.zeros(*ke.shape, 3, dtype=torch.float64, device="cuda") for _ in range(2)]
        for h in group:
            hc = slice(h * d, (h + 1) * d)
            qe, oe, ye = (t[:, hc].double() for t in (q, go, out))
            p = torch.exp(qe @ ke.t() / math.sqrt(d) - lse[:, h].double()[:, None])
            ds = p * (oe @ ve.t() - (oe * ye).sum(1, keepdim=True)) / math.sqrt(d)
            own = (d + 20) * A.EPS24 * p * (oe.abs() @ ve.abs().t() + (oe * ye).abs().sum(1, keepdim=True)) / math.sqrt(d)
            full[0][:, hc] = torch.stack([ds @ ke, ds.abs() @ ke.abs(), own @ ke.abs()], 2)
            part[0] += torch.stack([ds.t() @ qe, ds.abs().t() @ qe.abs(), own.t() @ qe.abs()], 2)
            part[1][..., :2] += torch.stack([p.t() @ oe, p.t() @ oe.abs()], 2)
        for to, x in zip(full[1:], part):
            at = torch.zeros(to.shape[0], *x.shape[1:], dtype=torch.float64, device="cuda")
            at[there] = x
            to[:, cols] = at
    return full


def check(got, want, dtype, rel, what):
    """rel: of the terms' sizes, for the weights; halves' smallest step, lifted by 2^10 or more, over 70000 rows of up to
    a half is below 2^-11 of a unit."""
    unit = A.UNIT[dtype]
    for name, g, x in zip("qkv", got, want):
        value, terms, own = x.unbind(2)
        step = A.STEP[dtype] + (2.0 ** -20 if dtype == torch.float16 else 0.0)
        bound = (1 + unit) * (rel * terms + 1.01 * own) + unit * value.abs() + step
        bad = ~((g.double() - value).abs() <= bound)
        assert not bad.any(), (what, name, int(bad.sum()), float(((g.double() - value).abs() / bound).max()))


def error(got, want):
    """The norm of the error, relative to that of what rounding the exact gradients leaves."""
    value = want[..., 0]
    return float((got.double() - value).norm() / (value.to(got.dtype).double() - value).norm())


# rows that take one pass over them (bfloat16, 1024 tiles and more) and rows that do not
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("rows", [900, 35_003, 70_003])
@pytest.mark.parametrize("d", [8, 16, 24, 32])
def test_no_rounding_but_the_results(ops, dtype, rows, d):
    """Weights in two parts hold 16 bits (bfloat16) or 22: off by 2^-17 of themselves at most. Scores, lse and their
    exponentials are off by less than 2^-17 at these sizes (terms of up to a hundred, 2^-24 each), sums over rows by
    far less in practice, by rows 2^-24 = 2^-8 of the terms at the worst; that is not allowed here, 2^-14 is."""
    q, k, v, go = case(rows + d, dtype, 1, rows, 200, 2, 1, d)
    m = mask_of(1, 1, 200, 0.8)
    forget(k, m, float("nan"))
    forget(v, m, float("nan"))
    out, lse = ops.attention(q, k, v, 2, kv_heads=1, mask=m, keep_lse=True)
    got = ops.attention_backward(go, q, k, v, out, lse, 2, kv_heads=1, mask=m)
    want = float64_gradients(q, k.nan_to_num(0.0), v.nan_to_num(0.0), go, out, lse, 2, 1, d, m[0])
    print(f"[attention] narrow {dtype} {rows} {d}", [round(error(g, x), 3) for g, x in zip(got, want)], flush=True)
    check(got, want, dtype, 2.0 ** -14, (rows, d))
    # one part would leave an error of 2^-10 (halves: 2^-13) of the terms in the mean, beside a result's of as much
    for g, x in zip(got, want):
        assert error(g, x) < 1.1


# batch, rows, states, heads, kv_heads, d, share of the states: one pass of bfloat16, and the same of the other types
ONCE = [(1, 70_003, 200, 2, 1, 24, 0.7), (2, 40_001, 33, 2, 2, 40, None), (1, 33_001, 256, 4, 2, 48, 0.5),
        (1, 70_003, 130, 1, 1, 56, 0.9), (3, 25_001, 64, 1, 1, 32, None)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", ONCE, ids=lambda s: "x".join(map(str, s)))
def test_one_pass_of_partial_tiles(ops, dtype, shape):
    batch, rows, states, heads, kv_heads, d, share = shape
    q, k, v, go = case(rows + states, dtype, batch, rows, states, heads, kv_heads, d, 3)
    m = None if share is None else mask_of(states, batch, states, share)
    args = dict(kv_heads=kv_heads, batch=batch, mask=m)
    print(f"[attention] one pass {shape} {dtype}", flush=True)
    out, lse = ops.attention(q, k, v, heads, keep_lse=True, **args)
    grads = ops.attention_backward(go, q, k, v, out, lse, heads, **args)
    rel = max(A.UNIT[dtype] + 2.0 ** -14, 2.0 ** -14)
    for e in range(batch):
        at, of = slice(e * rows, (e + 1) * rows), slice(e * states, (e + 1) * states)
        there = None if m is None else m[e]
        want = float64_gradients(q[at], k[of], v[of], go[at], out[at], lse[at], heads, kv_heads, d, there)
        check([grads[0][at], grads[1][of], grads[2][of]], want, dtype, rel, (shape, e))
        if there is not None:
            assert not grads[1][of][~there].any() and not grads[2][of][~there].any()


@pytest.mark.parametrize("d", [24, 32, 64])
def test_one_pass_over_a_single_state(ops, d):
    """A mask that leaves one of 90 states to 70003 rows: its weight is 1, grad_v is the sum of grad_out, and what is
    left of dp - delta in the other gradients is the rounding of two sums of d products."""
    rows, states = 70_003, 90
    q, k, v, go = case(d, torch.bfloat16, 1, rows, states, 2, 1, d)
    m = torch.zeros(1, states, dtype=torch.bool, device="cuda")
    m[0, 71] = True
    forget(k, m, float("nan"))
    forget(v, m, float("nan"))
    out, lse = ops.attention(q, k, v, 2, kv_heads=1, mask=m, keep_lse=True)
    got = ops.attention_backward(go, q, k, v, out, lse, 2, kv_heads=1, mask=m)
    want = float64_gradients(q, k.nan_to_num(0.0), v.nan_to_num(0.0), go, out, lse, 2, 1, d, m[0])
    check(got, want, torch.bfloat16, 2.0 ** -14, d)
    assert not got[1][~m[0]].any() and not got[2][~m[0]].any()


def test_some_gradients_of_one_pass(ops):
    """Which gradients are asked for chooses the kernels and so the order of the sums, not more: each set is right."""
    q, k, v, go = case(4, torch.bfloat16, 1, 70_003, 90, 1, 1, 64)
    out, lse = ops.attention(q, k, v, 1, keep_lse=True)
    want = float64_gradients(q, k, v, go, out, lse, 1, 1, 64)
    for need in ((True, True, True), (True, False, True), (True, True, False), (True, False, False), (False, True, True),
                 (False, False, True), (False, True, False)):
        got = ops.attention_backward(go, q, k, v, out, lse, 1, need_q=need[0], need_k=need[1], need_v=need[2])
        assert [x is not None for x in got] == list(need)
        some = [(x, w) for x, w in zip(got, want) if x is not None]
        check([x for x, _ in some], [w for _, w in some], torch.bfloat16, 2.0 ** -8 + 2.0 ** -14, need)
        again = ops.attention_backward(go, q, k, v, out, lse, 1, need_q=need[0], need_k=need[1], need_v=need[2])
        assert all(x is None or torch.equal(x, y) for x, y in zip(got, again))
