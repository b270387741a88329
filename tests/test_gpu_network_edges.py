"""The attribute network's operators where their definitions meet the types' ends and each other's places: outputs over
inputs, infinities, matrices of a few columns."""
import pytest
import torch

import network_reference as R

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
IDS = ["f32", "f16", "bf16"]


@pytest.fixture(scope="module")
def ops(hip):
    from tinygs_amd.network import LayerOps
    return LayerOps()


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


# rows in a group of lanes, in a wave, in a workgroup's registers, and read again from memory (above 32 KB)
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(5, 9), (1000, 84), (70, 1031), (9, 8192), (11, 8200), (300, 8200), (7, 16384), (3, 20000)],
                         ids=str)
def test_layer_norm_backward_in_its_inputs_place(ops, shape, dtype):
    """grad_x in grad_y's own matrix, or in residual_grad's: all three gradients as with a matrix of its own."""
    rows, n = shape
    x = (1.5 * normal(1, rows, n)).to(dtype).cuda()
    gy, res = (0.1 * normal(2, rows, n)).to(dtype).cuda(), (0.1 * normal(3, rows, n)).to(dtype).cuda()
    gamma = normal(4, n).cuda()
    mean, rstd = ops.layer_norm(x, gamma, None, eps=1e-3)[1:]
    for residual in (None, res):
        apart = ops.layer_norm_backward(gy, x, gamma, mean, rstd, residual_grad=residual)
        for t, (want, bound), what in zip(apart, R.layer_norm_backward(gy, x, gamma, mean, rstd, residual, dtype),
                                          ("gx", "ggamma", "gbeta")):
            R.check(t, want, bound, what)
        buf = gy.clone()
        got = ops.layer_norm_backward(buf, x, gamma, mean, rstd, residual_grad=residual, grad_x=buf)
        for t, want, what in zip(got, apart, ("gx", "ggamma", "gbeta")):
            assert torch.equal(t, want), f"{what} over grad_y"
    buf = res.clone()
    got = ops.layer_norm_backward(gy, x, gamma, mean, rstd, residual_grad=buf, grad_x=buf)
    for t, want, what in zip(got, apart, ("gx", "ggamma", "gbeta")):
        assert torch.equal(t, want), f"{what} over residual_grad"


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("out", [3, 64, 600])
@pytest.mark.parametrize("name", ["relu", "silu", "gelu"])
def test_slopes_at_infinity(ops, name, out, dtype):
    """Values before the activation that left the type's range, as float16's do at 65520: slope 1 above, 0 below."""
    rows, i = 70, 20
    z = (2.0 * normal(1, rows, out)).to(dtype)
    z[3, 0], z[4, 1], z[69, out - 1] = float("inf"), float("-inf"), float("inf")
    x, w, gy = normal(2, rows, i).to(dtype), normal(3, out, i).to(dtype), normal(4, rows, out).to(dtype)
    got = ops.linear_backward(gy.cuda(), x.cuda(), w.cuda(), preact=z.cuda(), activation=name)
    # at +-200 the slopes are 1 and 0 to every bit
    want = R.linear_backward(gy, x, w, z.double().clamp(-200.0, 200.0), name, dtype)
    for t, (v, bound), what in zip(got, want, ("gx", "gw", "gb")):
        R.check(t, v, bound, what)
