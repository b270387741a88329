"""Gradients of halves where a state's weight is small for every row."""
import pytest
import torch

from test_gpu_attention import ops  # noqa: F401

pytestmark = pytest.mark.gpu


def test_small_weights_of_every_row(ops):
    """Halves: a state whose weight is about 2^-27 for every row. Held times 2^13 it is off by half a step of 2^-24
    at 2^-14, 2^-11 of it, and the result by as much again; grad_v of that state is its share of the rows' gradients."""
    rows, states, d = 40_000, 50, 64
    g = torch.Generator().manual_seed(5)
    q = torch.zeros(rows, d, dtype=torch.float16, device="cuda")
    q[:, 0] = 16.0
    k = torch.zeros(states, d, dtype=torch.float16, device="cuda")
    k[9, 0] = -0.925
    v = torch.randn(states, d, generator=g).half().cuda()
    go = (8.0 + torch.randn(rows, d, generator=g)).half().cuda()
    out, lse = ops.attention(q, k, v, 1, scale=1.0, keep_lse=True)
    _, _, gv = ops.attention_backward(go, q, k, v, out, lse, 1, scale=1.0)
    p = torch.exp((q.double() @ k.double().t())[:1] - lse[:1].double())
    want = p[0, 9] * go.double().sum(0)
    assert float(p[0, 9]) < 2.0 ** -26
    assert bool(((gv[9].double() - want).abs() <= 2.0 ** -9 * want.abs()).all())
