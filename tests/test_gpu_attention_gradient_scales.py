"""Gradients of halves where one element of a batch, or the heads of one group, have gradients far larger than another's,
or infinite ones: each group's are what they would be beside any others."""
import pytest
import torch

import attention_reference as A
from test_gpu_attention import case, ops  # noqa: F401

pytestmark = pytest.mark.gpu

SMALL, LARGE = 2.0 ** -8, 2.0 ** 12


def gradients(ops, t, out, lse, batch, need_q=True):
    q, k, v, go = t
    return ops.attention_backward(go, q, k, v, out, lse, 4, kv_heads=2, batch=batch, need_q=need_q)


# two kernels with and without parts of the rows; wide heads, whose dk and dv are apart
@pytest.mark.parametrize("need_q", [True, False])
@pytest.mark.parametrize("queries, states, d", [(300, 150, 64), (2000, 700, 128), (37, 40, 32), (20_000, 300, 40)])
def test_elements(ops, queries, states, d, need_q):
    q, k, v, go = case(d, torch.float16, 2, queries, states, 4, 2, d)
    out, lse = ops.attention(q, k, v, 4, kv_heads=2, batch=2, keep_lse=True)
    go = (go / go.float().std() * SMALL).half()
    print(f"[attention] elements {queries} {states} {d} {need_q}", flush=True)
    want = gradients(ops, (q, k, v, go), out, lse, 2, need_q)
    for first in (LARGE / SMALL, float("inf")):
        other = go.clone()
        other[:queries] *= first
        got = gradients(ops, (q, k, v, other), out, lse, 2, need_q)
        for x, y in zip(got, want):
            half = 0 if x is None else x.shape[0] // 2
            assert x is None or torch.equal(x[half:], y[half:]), first
    if queries > 1000:
        return
    # and they are right: the second element's gradients against 64 bits
    one, of = slice(queries, None), slice(states, None)
    ref = A.attention_backward(go[one], q[one], k[of], v[of], out[one], lse[one], 4, 2)
    for name, g, (x, b) in zip("qkv", want, ref):
        if g is not None:
            A.check(g[one if name == "q" else of], x, b, "grad_" + name)


@pytest.mark.parametrize("need_q", [True, False])
def test_heads_that_share_no_states(ops, need_q):
    q, k, v, go = case(3, torch.float16, 1, 300, 150, 4, 2, 64)
    out, lse = ops.attention(q, k, v, 4, kv_heads=2, keep_lse=True)
    go = (go / go.float().std() * SMALL).half()
    want = gradients(ops, (q, k, v, go), out, lse, 1, need_q)
    for first in (LARGE / SMALL, float("inf")):
        other = go.clone()
        other[:, :128] *= first   # heads 0 and 1, which share the states' first head
        got = gradients(ops, (q, k, v, other), out, lse, 1, need_q)
        assert not need_q or torch.equal(got[0][:, 128:], want[0][:, 128:])
        assert torch.equal(got[1][:, 64:], want[1][:, 64:]) and torch.equal(got[2][:, 64:], want[2][:, 64:])
