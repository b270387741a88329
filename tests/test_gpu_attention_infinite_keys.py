"""A state whose key holds an infinity, with a score of minus infinity for every row: its weights are 0, and so are its
gradients, whether or not the rows fill the kernels' last tile; the others' are those beside a state that does not exist."""
import pytest
import torch

from test_gpu_attention import DTYPES, IDS, case, ops  # noqa: F401

pytestmark = pytest.mark.gpu


# rows that end inside a tile and rows that fill it, of both backward paths; 1094 tiles of bfloat16 take one pass
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows, states, d", [(70, 90, 32), (64, 90, 32), (1, 40, 64), (333, 500, 128), (70_003, 90, 64),
                                             (70_003, 40, 32), (70_016, 90, 64)])
def test_gradients(ops, dtype, rows, states, d):
    q, k, v, go = case(rows + d, dtype, 1, rows, states, 2, 1, d)
    for h in (0, d):
        q[:, h] = q[:, h].abs() + 0.5
    k[5, 0] = float("-inf")
    v[5] *= 0.125   # halves: not the value that the lift of grad_q's weights is taken from
    print(f"[attention] infinite key {rows} {states} {d} {dtype}", flush=True)
    out, lse = ops.attention(q, k, v, 2, kv_heads=1, keep_lse=True)
    gq, gk, gv = ops.attention_backward(go, q, k, v, out, lse, 2, kv_heads=1)
    assert not gk[5].any() and not gv[5].any()
    mask = torch.ones(1, states, dtype=torch.bool, device="cuda")
    mask[0, 5] = False
    want, wlse = ops.attention(q, k, v, 2, kv_heads=1, mask=mask, keep_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, wlse)
    wq, wk, wv = ops.attention_backward(go, q, k, v, out, lse, 2, kv_heads=1, mask=mask)
    assert torch.equal(gk, wk) and torch.equal(gv, wv)
    # column 0 of grad_q adds 0 times the infinity: NaN, as the formula says
    for h in (0, d):
        assert bool(torch.isnan(gq[:, h]).all()) and torch.equal(gq[:, h + 1:h + d], wq[:, h + 1:h + d])


# the infinite row is the last, beside rows that a tile lacks and beside none
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows, states, d", [(70, 90, 32), (128, 90, 32), (1, 40, 64), (333, 500, 128), (70_003, 90, 64),
                                             (70_003, 40, 32)])
def test_infinite_gradients(ops, dtype, rows, states, d):
    """An infinity in grad_out's last row: that column of grad_v is infinite for every state that has a weight, the others
    are as beside a finite one; grad_k of its head is what the formula leaves of infinities, no number. 16-bit heads up to
    32 columns hold a weight as w + r with r of either sign or 0, and an infinity times both is NaN as often."""
    q, k, v, go = case(rows + d, dtype, 1, rows, states, 2, 2, d, q_scale=0.3)
    print(f"[attention] infinite gradient {rows} {states} {d} {dtype}", flush=True)
    out, lse = ops.attention(q, k, v, 2, keep_lse=True)
    _, wk, wv = ops.attention_backward(go, q, k, v, out, lse, 2)
    go[rows - 1, 3] = float("-inf")
    _, gk, gv = ops.attention_backward(go, q, k, v, out, lse, 2)
    if d <= 32 and dtype != torch.float32:
        assert not bool(torch.isfinite(gv[:, 3]).any())
    else:
        assert bool((gv[:, 3] == float("-inf")).all())
    gv[:, 3] = wv[:, 3]
    assert torch.equal(gv, wv)
    assert torch.equal(gk[:, d:], wk[:, d:]) and not bool(torch.isfinite(gk[:, :d]).any())


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows, states, d", [(1, 70, 64), (70, 90, 32), (60_000, 200, 64), (20_000, 700, 128), (20, 5000, 96)])
def test_infinite_values(ops, dtype, rows, states, d):
    """An infinite value of a state that has a weight makes that column of every average infinite, and no other."""
    q, k, v, _ = case(rows, dtype, 1, rows, states, 2, 2, d, q_scale=0.3)
    print(f"[attention] infinite value {rows} {states} {d} {dtype}", flush=True)
    want = ops.attention(q, k, v, 2)
    v[states // 2, d + 3] = float("inf")
    v[3, 2] = float("-inf")
    got = ops.attention(q, k, v, 2)
    assert bool((got[:, d + 3] == float("inf")).all()) and bool((got[:, 2] == float("-inf")).all())
    got[:, d + 3], got[:, 2] = want[:, d + 3], want[:, 2]
    assert torch.equal(got, want)
