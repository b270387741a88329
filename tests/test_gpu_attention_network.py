"""An attribute network that attends to an encoder's states: its gradients against 64-bit automatic differentiation of
the same formula; clipping; a training step of Gaussians with a bound on the gradients' norm; the C++ interface; the
example."""
import math
import os
import subprocess
import sys

import pytest
import torch

from tinygs_amd import build as hb

pytestmark = pytest.mark.gpu


def reference(net, weights, vectors, features, context, mask, batch, positions, context_positions):
    """The network's formula in 64 bits on leaf copies of its parameters."""
    blocks, last, width = net.blocks, net.last, weights[0].shape[0]
    d = width // net.heads
    base, more = weights[:last + 1], weights[last + 1:]
    sizes = ([w.shape[0] for w in base] + [width, width] * (blocks + 1) + [w.shape[0] for w in more] +
             [width, width, d, d] * blocks)
    v = vectors.split(sizes)
    m, n = last + 1, last + 1 + 2 * (blocks + 1)
    norms = list(zip(v[m:n:2], v[m + 1:n:2]))
    biases, own = v[n:n + 4 * blocks], v[n + 4 * blocks:]

    def norm(h, gamma, beta):
        mean = h.mean(1, keepdim=True)
        return (h - mean) / torch.sqrt(((h - mean) ** 2).mean(1, keepdim=True) + net.eps) * gamma + beta

    def act(z):
        return 0.5 * z * (1.0 + torch.tanh((2.0 / torch.pi) ** 0.5 * (z + 0.044715 * z ** 3)))

    def head_norm(x, heads, gamma, at):
        x = x.reshape(x.shape[0], heads, d)
        x = x / torch.sqrt((x * x).mean(2, keepdim=True) + 1e-6) * gamma
        if net.axes:
            angle = (at.double() @ net.frequencies.double().t())[:, None, :]
            z = torch.view_as_complex(x.reshape(*x.shape[:2], d // 2, 2).contiguous()) * torch.polar(torch.ones_like(angle),
                                                                                                angle)
            x = torch.view_as_real(z).reshape(*x.shape[:2], d)
        return x

    def attend(h, k):
        w, b = more[4 * k:4 * k + 4], biases[4 * k:4 * k + 4]
        gamma, beta, gamma_q, gamma_k = own[4 * k:4 * k + 4]
        q = head_norm(norm(h, gamma, beta) @ w[0].t() + b[0], net.heads, gamma_q, positions)
        key = head_norm(context @ w[1].t() + b[1], net.kv_heads, gamma_k, context_positions)
        val = (context @ w[2].t() + b[2]).reshape(context.shape[0], net.kv_heads, d)
        t = net.heads // net.kv_heads
        q, key, val = (x.reshape(batch, -1, x.shape[1], d).transpose(1, 2) for x in (q, key, val))
        key, val = key.repeat_interleave(t, 1), val.repeat_interleave(t, 1)
        s = (q @ key.transpose(2, 3).contiguous() / math.sqrt(d)).masked_fill(~mask[:, None, None, :], -math.inf)
        a = (torch.softmax(s, 3) @ val).transpose(1, 2).reshape(h.shape)
        return h + a @ w[3].t() + b[3]

    h = features @ base[0].t() + v[0]
    for k in range(blocks):
        h = attend(h, k)
        a = act(norm(h, *norms[k]) @ base[1 + 2 * k].t() + v[1 + 2 * k])
        h = h + a @ base[2 + 2 * k].t() + v[2 + 2 * k]
    return norm(h, *norms[-1]) @ base[last].t() + v[last]


@pytest.mark.parametrize("dtype,bound", [(torch.float32, 2e-5), (torch.float16, 2e-2), (torch.bfloat16, 1.2e-1)],
                         ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("axes,kv_heads", [(0, 4), (3, 2)])
def test_gradients(hip, dtype, bound, axes, kv_heads):
    """Normwise: float errors of two dozen operators, or about as many roundings to the type (2^-11, 2^-8)."""
    from tinygs_amd.network import AttributeNetwork
    batch, rows, states = 2, 333, 75
    net = AttributeNetwork(39, 59, width=96, hidden=136, blocks=2, dtype=dtype, seed=3, context=50, heads=4,
                           kv_heads=kv_heads, axes=axes, extent=3.0)
    g = torch.Generator().manual_seed(1)
    net.weights[net.last].copy_(0.1 * torch.randn(net.weights[net.last].shape, generator=g).cuda())
    if net.copies is not None:
        net.copies[net.last].copy_(net.weights[net.last])
    net.vectors.add_(0.1 * torch.randn(net.vectors.shape, generator=g).cuda())
    features = torch.randn(batch * rows, 39, generator=g).cuda().to(dtype)
    context = torch.randn(batch * states, 50, generator=g).cuda().to(dtype)
    grad = torch.randn(batch * rows, 59, generator=g).cuda().to(dtype)
    mask = (torch.rand(batch, states, generator=g) < 0.7).cuda()
    at, where = (3 * torch.randn(batch * n, max(axes, 1), generator=g).cuda() for n in (rows, states))
    args = dict(context=context, mask=mask, batch=batch)
    if axes:
        args.update(positions=at, context_positions=where)
    y = net.forward(features, **args)
    gx, gc = net.backward(grad, need_features=True, need_context=True)
    weights = [w.double().requires_grad_() for w in net.matrices()]
    vectors = net.vectors.double().requires_grad_()
    x, c = features.double().requires_grad_(), context.double().requires_grad_()
    want = reference(net, weights, vectors, x, c, mask, batch, at, where)
    want.backward(grad.double())

    def near(a, b, what):
        assert float((a.double() - b).norm()) <= bound * float(b.norm()), (what, float((a.double() - b).norm() / b.norm()))

    near(y, want.detach(), "attributes")
    near(gx, x.grad, "features")
    near(gc, c.grad, "context")
    near(net.vector_grads, vectors.grad, "vectors")
    for k, (a, b) in enumerate(zip(net.grads, weights)):
        near(a, b.grad, f"matrix {k}")
    assert torch.equal(net.forward(features, keep=False, **args), y)
    # the bound takes all of them along
    before = [t.clone() for t in net.grads + [net.vector_grads]]
    total = math.sqrt(sum(float((t.double() ** 2).sum()) for t in before))
    norm = net.clip(0.5 * total)
    assert abs(float(norm) - total) <= 1e-6 * total
    unit = torch.finfo(dtype).eps
    for a, b in zip(net.grads + [net.vector_grads], before):
        assert float((a.double() - 0.5 * b.double()).norm()) <= (unit + 1e-6) * float(b.double().norm())
    net.optimizer().step(1.0)


def test_network_without_context_is_as_before(hip):
    """The same weights for the same seed, with and without attention."""
    from tinygs_amd.network import AttributeNetwork
    a, b = AttributeNetwork(20, 3, width=64, seed=5), AttributeNetwork(20, 3, width=64, seed=5, context=16)
    assert all(torch.equal(x, y) for x, y in zip(a.weights, b.weights))
    x = torch.randn(30, 20, device="cuda")
    with pytest.raises(RuntimeError, match="network with context"):
        a.forward(x, context=torch.randn(9, 16, device="cuda"))
    with pytest.raises(RuntimeError, match="network with context"):
        b.forward(x)
    a.forward(x)
    with pytest.raises(RuntimeError, match="without context"):
        a.backward(torch.randn(30, 3, device="cuda"), need_context=True)
    for more, words in ((dict(heads=5), "divide"), (dict(kv_heads=3), "divide"), (dict(axes=5), "axes"),
                        (dict(width=512, heads=2), "128"), (dict(context=0), "divide"), (dict(extent=0.0, axes=1), "extent")):
        with pytest.raises(RuntimeError, match=words):
            AttributeNetwork(20, 3, **dict(dict(width=64, context=16), **more))
    with pytest.raises(RuntimeError, match="positions"):
        AttributeNetwork(20, 3, width=64, context=16, axes=3).forward(x, context=torch.randn(9, 16, device="cuda"))


def test_a_run_captured_and_replayed(hip):
    """Norm, projections, head norms, attention, backward, clipping and Muon's step as one graph, against eager steps."""
    from tinygs_amd.network import AttributeNetwork
    s = torch.cuda.Stream()
    g = torch.Generator().manual_seed(2)
    features, context, grad = (torch.randn(n, c, generator=g).cuda() for n, c in ((500, 20), (40, 16), (500, 3)))
    at, where = torch.randn(500, 3, generator=g).cuda(), torch.randn(40, 3, generator=g).cuda()
    nets = [AttributeNetwork(20, 3, width=64, blocks=1, seed=5, context=16, axes=3) for _ in range(2)]
    for n in nets:
        n.weights[n.last].fill_(0.05)
    optimizers = [n.optimizer() for n in nets]
    torch.cuda.synchronize()

    def step(n, o):
        y = n.forward(features, context=context, positions=at, context_positions=where, stream=s)
        n.backward(grad, stream=s)
        n.clip(0.5, stream=s)
        o.step(1.0, stream=s)
        return y

    for n, o in zip(nets, optimizers):
        step(n, o)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        held = step(nets[0], optimizers[0])
    for _ in range(3):
        graph.replay()
        y = step(nets[1], optimizers[1])
        torch.cuda.synchronize()
        assert torch.equal(held, y)
        assert all(torch.equal(a, b) for a, b in zip(nets[0].weights + nets[0].grads, nets[1].weights + nets[1].grads))
        assert torch.equal(nets[0].vector_grads, nets[1].vector_grads)


def test_gaussians_step_with_a_bound(hip):
    """TrainStep's bound: the gradients' norm as summed in 64 bits, and Adam's step on clipped gradients."""
    from tinygs_amd import scenes
    from tinygs_amd.train import TrainStep
    scene = scenes.config3(seed=3, n=3000, width=128, height=96)
    with pytest.raises(ValueError, match="sparse_grads"):
        TrainStep(scene, max_grad_norm=1.0)
    free, bounded = (TrainStep(scene, sparse_grads=False, grad_scaler=2.0, max_grad_norm=m) for m in (math.inf, 1e-5))
    for ts in (free, bounded):
        ts.step()
    torch.cuda.synchronize()
    total = math.sqrt(sum(float((t.double() ** 2).sum()) for t in free.grads.tensors()))
    for ts in (free, bounded):
        assert abs(float(ts.grad_norm) - total) <= 1e-6 * total
    assert total > 2e-5
    after = math.sqrt(sum(float((t.double() ** 2).sum()) for t in bounded.grads.tensors()))
    # epsilon is 1e-6 next to the norm
    assert abs(after - 2e-5 * total / (total + 1e-6)) <= 1e-5 * after
    for a, b in zip(free.grads.tensors(), bounded.grads.tensors()):
        f = 2e-5 / (total + 1e-6)
        assert float((b.double() - f * a.double()).norm()) <= 1e-6 * f * float(a.double().norm()) + 1e-30


def test_cpp_attention_step(hip):
    exe = hb.cpp_test_bin("attention_step")
    if not os.path.exists(exe):
        hb.build_cpp_test(verbose=False)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "attention ok" in r.stdout


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_recolour_example_attends(hip, dtype):
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
    from recolour import recolour
    losses = recolour(gaussians=4000, steps=6, width=64, blocks=1, dtype=dtype, image=128, states=64, max_grad_norm=0.01,
                      log=lambda s: print(s, flush=True))
    assert len(losses) == 6 and all(math.isfinite(x) for x in losses)
