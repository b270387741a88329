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
