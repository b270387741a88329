"""Head norms of elements whose squares leave the range of floats: the formula's results are ordinary numbers."""
import pytest
import torch

import attention_reference as A
from test_gpu_attention import ops  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("d", [3, 16, 64, 200])
@pytest.mark.parametrize("scale, eps", [(2.0 ** 100, 1e-6), (2.0 ** 64, 0.0), (2.0 ** -80, 0.0), (2.0 ** -110, 0.0),
                                        (2.0 ** -80, 1e-38)])
def test_forward_and_backward(ops, dtype, d, scale, eps):
    g = torch.Generator().manual_seed(d)
    heads, rows = 3, 70
    x = torch.randn(rows, heads * d, generator=g)
    size = torch.where(torch.arange(rows) % 3 == 0, torch.tensor(1.0), torch.tensor(scale))   # beside ordinary rows
    x = (x.double() * size.double()[:, None]).to(dtype).cuda()
    gamma = torch.randn(d, generator=g).cuda()
    positions = torch.randn(rows, 3, generator=g).cuda()
    frequencies = torch.randn(d // 2, 3, generator=g).cuda()
    turn = dict(positions=positions, frequencies=frequencies)
    y = ops.head_norm(x, heads, gamma, eps=eps, **turn)
    A.check(y, *A.head_norm(x, heads, gamma, positions, frequencies, eps), "y")
    # gradients as small as the inputs are large: their product with 1 / |x| stays within the type
    gy = torch.randn(rows, heads * d, generator=g)
    gy = (gy.double() * size.double()[:, None] * 0.5).to(dtype).cuda()
    gx, gg = ops.head_norm_backward(gy, x, heads, gamma, eps=eps, **turn)
    (dx, bound), (dg, gbound) = A.head_norm_backward(gy, x, heads, gamma, positions, frequencies, eps)
    A.check(gx, dx, bound, "grad_x")
    A.check(gg, dg, gbound, "grad_gamma")
