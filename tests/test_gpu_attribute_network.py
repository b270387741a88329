"""The attribute network: its gradients against 64-bit automatic differentiation of the same formula, and a scene
recoloured through it."""
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu


def reference(net, weights, vectors, features):
    """The network's formula in 64 bits on leaf copies of its parameters."""
    m = len(weights)
    sizes = [w.shape[0] for w in weights] + [weights[0].shape[0]] * (2 * (net.blocks + 1))
    v = vectors.split(sizes)
    norms = list(zip(v[m::2], v[m + 1::2]))

    def norm(h, gamma, beta):
        mean = h.mean(1, keepdim=True)
        return (h - mean) / torch.sqrt(((h - mean) ** 2).mean(1, keepdim=True) + net.eps) * gamma + beta

    def act(z):
        return 0.5 * z * (1.0 + torch.tanh((2.0 / torch.pi) ** 0.5 * (z + 0.044715 * z ** 3)))

    h = features @ weights[0].t() + v[0]
    for k in range(net.blocks):
        a = act(norm(h, *norms[k]) @ weights[1 + 2 * k].t() + v[1 + 2 * k])
        h = h + a @ weights[2 + 2 * k].t() + v[2 + 2 * k]
    return norm(h, *norms[-1]) @ weights[-1].t() + v[m - 1]


@pytest.mark.parametrize("dtype,bound", [(torch.float32, 1e-5), (torch.float16, 1e-2), (torch.bfloat16, 6e-2)],
                         ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 777])
def test_gradients(hip, dtype, bound, rows):
    """Normwise: float errors of a dozen operators, or about as many roundings to the type (2^-11, 2^-8)."""
    from tinygs_amd.network import AttributeNetwork
    net = AttributeNetwork(39, 59, width=96, hidden=136, blocks=2, dtype=dtype, seed=3)
    g = torch.Generator().manual_seed(1)
    net.weights[-1].copy_(0.1 * torch.randn(net.weights[-1].shape, generator=g).cuda())
    if net.copies is not None:
        net.copies[-1].copy_(net.weights[-1])
    net.vectors.add_(0.1 * torch.randn(net.vectors.shape, generator=g).cuda())
    features = torch.randn(rows, 39, generator=g).cuda().to(dtype)
    grad = torch.randn(rows, 59, generator=g).cuda().to(dtype)
    y = net.forward(features)
    gx = net.backward(grad, need_features=True)
    weights = [w.double().requires_grad_() for w in net.matrices()]
    vectors = net.vectors.double().requires_grad_()
    x = features.double().requires_grad_()
    want = reference(net, weights, vectors, x)
    want.backward(grad.double())

    def near(a, b, what):
        assert float((a.double() - b).norm()) <= bound * float(b.norm()), (what, float((a.double() - b).norm() / b.norm()))

    near(y, want.detach(), "attributes")
    near(gx, x.grad, "features")
    near(net.vector_grads, vectors.grad, "vectors")
    for k, (a, b) in enumerate(zip(net.grads, weights)):
        near(a, b.grad, f"matrix {k}")
    assert torch.equal(net.forward(features, keep=False), y)
    with pytest.raises(RuntimeError, match="no forward"):
        net.backward(grad)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_recolour_example(hip, dtype):
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
    from recolour import recolour
    losses = recolour(gaussians=4000, steps=40, width=64, blocks=1, dtype=dtype, image=128,
                      log=lambda s: print(s, flush=True))
    assert losses[-1] < 0.5 * losses[0], (losses[0], losses[-1])


def test_refusals(hip):
    from tinygs_amd.network import AttributeNetwork
    with pytest.raises(RuntimeError, match="unknown activation"):
        AttributeNetwork(4, 3, activation="tanh")
    with pytest.raises(RuntimeError, match="positive"):
        AttributeNetwork(0, 3)
    with pytest.raises(RuntimeError, match="float32, float16 and bfloat16"):
        AttributeNetwork(4, 3, dtype=torch.float64)
