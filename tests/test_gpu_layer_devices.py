"""One handle on every device of the machine in turn: each has a workspace of its own, and the results are the same."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_one_handle_on_each_device(hip):
    from tinygs_amd.network import LayerOps
    ops = LayerOps()
    g = torch.Generator().manual_seed(1)
    cpu = [torch.randn(300, 64, generator=g) for _ in range(4)]
    w, gamma = torch.randn(64, 64, generator=g), torch.ones(64)
    want = None
    for device in list(range(torch.cuda.device_count())) * 2:
        with torch.cuda.device(device):
            q, k, v, go = (t.half().cuda() for t in cpu)
            out, lse = ops.attention(q, k, v, 4, keep_lse=True)
            got = [out, *ops.attention_backward(go, q, k, v, out, lse, 4)]
            got += ops.linear_backward(go, q, w.half().cuda())
            y, mean, rstd = ops.layer_norm(q, gamma.cuda(), gamma.cuda())
            got += ops.layer_norm_backward(go, q, gamma.cuda(), mean, rstd)
            got += ops.head_norm_backward(go, q, 1, gamma.cuda())
            got = [t.cpu() for t in got]
        want = want or got
        assert all(torch.equal(x, y) for x, y in zip(got, want)), device
