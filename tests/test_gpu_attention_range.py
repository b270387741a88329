"""Attention's range: values near the largest floats beside scores that rise with the states, infinite values of no weight,
and weights far below the first ones' in halves."""
import math

import pytest
import torch

import attention_reference as A
from test_gpu_attention import case, ops  # noqa: F401

pytestmark = pytest.mark.gpu


# states held in LDS, tiles of them, parts of them joined, one to four rows
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows, states, d", [(140_003, 200, 32), (70_000, 700, 64), (30, 5000, 128), (1, 400, 64)])
def test_large_values(ops, dtype, rows, states, d):
    """Values up to 2^95 with scores that rise by 30 from the first states on (weights of 2^43): averages of them are
    finite, and right."""
    q, k, v, _ = case(rows, dtype, 1, rows, states, 1, 1, d)
    q[::3] = 0.0
    q[::3, 0] = math.sqrt(d) * 2.0
    k[:, 0] = torch.linspace(-5, 10, states).to(dtype).cuda()
    v = (v / v.abs().max() * 2.0 ** 95).to(dtype)
    print(f"[attention] large values {rows} {states} {d} {dtype}", flush=True)
    out, lse = ops.attention(q, k, v, 1, keep_lse=True)
    pick = torch.cat([torch.arange(0, rows, max(1, rows // 50)), torch.tensor([rows - 1])]).cuda()
    (o, ob), (l, lb) = A.attention(q[pick].contiguous(), k, v, 1, 1)
    A.check(out[pick], o, ob, "out")
    A.check(lse[pick], l, lb, "lse")


@pytest.mark.parametrize("states", [20_000, 200_000])
def test_many_small_weights(ops, states):
    """Halves: one state of weight 1 and many of 1.4 2^-24, whose values are 1. Together they make 1.7% of the average of
    200000; rounded in steps of 2^-24 they would lose a third of it. The average is off by less than half a unit of the
    largest value, 2^-11 with the result's own rounding and 2^-12 for the weights. The sum of the weights, which lse is
    the logarithm of, is one of floats: a rounding of 2^-24 of it for sixteen weights of the half of the states that a
    lane adds, states / 32 in all, and 40 within the sixteen and around them; so is each value's sum, in steps of
    sixteen states."""
    rows, d = 20_000, 32
    q = torch.zeros(rows, d, dtype=torch.float16, device="cuda")
    q[:, 0] = 16.0
    k = torch.zeros(states, d, dtype=torch.float16, device="cuda")
    k[1:, 0] = -1.0185546875
    v = torch.ones(states, d, dtype=torch.float16, device="cuda")
    v[0] = 0.0
    out, lse = ops.attention(q, k, v, 1, scale=1.0, keep_lse=True)
    small = (states - 1) * math.exp(-16.0 * 1.0185546875)
    assert float((out.double() - small / (1.0 + small)).abs().max()) <= 2.0 ** -11 * small + 2.0 ** -12
    off = (states / 32 + 40) * A.EPS24
    assert float((lse.double() - math.log1p(small)).abs().max()) <= off
    v[0] = 1.0   # an average of ones
    out = ops.attention(q, k, v, 1, scale=1.0)
    assert float((out.double() - 1.0).abs().max()) <= 2.0 ** -11 + 2.0 ** -12 + off + (states / 16 + 40) * A.EPS24


def test_late_maxima_of_many_states(ops):
    """Halves at many states, the largest scores late: by a little, by more than a weight's range, and rows of each side
    by side; a row's bits do not depend on the others', nor a column's on another's NaN."""
    rows, states, d = 16_500, 30_000, 32
    q, k, v, _ = case(7, torch.float16, 1, rows, states, 1, 1, d, q_scale=0.3)
    k[:, 0] = torch.linspace(-1, 4, states).half().cuda()
    q[:, 0] = 0.0
    want = ops.attention(q, k, v, 1)
    steep = q.clone()
    steep[::5, 0] = 4.0 * math.sqrt(d) * torch.linspace(0.1, 1.0, 3300).half().cuda()
    out, lse = ops.attention(steep, k, v, 1, keep_lse=True)
    pick = torch.arange(0, rows, 331).cuda()
    (o, ob), (l, lb) = A.attention(steep[pick].contiguous(), k, v, 1, 1)
    A.check(out[pick], o, ob, "out")
    A.check(lse[pick], l, lb, "lse")
    keep = torch.ones(rows, dtype=torch.bool, device="cuda")
    keep[::5] = False
    assert torch.equal(out[keep], want[keep])
    v[17, 0] = float("nan")
    got = ops.attention(steep, k, v, 1)
    assert bool(torch.isnan(got[:, 0]).all()) and torch.equal(got[:, 1:], out[:, 1:])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_largest_values_of_a_single_row(ops, dtype):
    """One row, whose weights are at most 1: an average of the type's largest values is one of them."""
    q, k, v, _ = case(2, dtype, 1, 1, 300, 2, 2, 48)
    v = (v.abs() / v.abs().max() * 0.99 * torch.finfo(dtype).max).to(dtype)
    out, lse = ops.attention(q, k, v, 2, keep_lse=True)
    (o, ob), _ = A.attention(q, k, v, 2, 2)
    A.check(out, o, ob, "out")


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
def test_infinite_values_of_no_weight(ops, dtype):
    """A state with a score of minus infinity and infinite values: 0 times an infinity is NaN, for one row as for many."""
    for rows in (1, 3, 40):
        q, k, v, _ = case(rows, dtype, 1, rows, 70, 1, 1, 32)
        q[:, 0] = 1.0
        k[20, 0] = float("-inf")
        want = ops.attention(q, k, v, 1)
        assert bool(torch.isfinite(want).all())
        v[20, 7] = float("inf")
        got = ops.attention(q, k, v, 1)
        assert bool(torch.isnan(got[:, 7]).all()), rows
        got[:, 7] = want[:, 7]
        assert torch.equal(got, want)
