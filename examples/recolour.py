"""Recolours a scene through an attribute network: the network maps encoded positions to a change of every Gaussian's
base colour (SH degree 0) and is trained through the rasteriser, with Muon on its matrices and Adam on its vectors.

    python examples/recolour.py [--gaussians N] [--steps K] [--dtype float32|float16|bfloat16]

The target is the same scene with its colours shifted along x; each step renders, evaluates L1 + SSIM and steps."""
import argparse
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))


def recolour(gaussians: int = 20000, steps: int = 60, width: int = 128, blocks: int = 2, dtype: str = "bfloat16",
             image: int = 256, log=print):
    """The losses of the steps (mean of the loss image)."""
    import torch
    from tinygs_amd import scenes
    from tinygs_amd.network import AttributeNetwork, encode_positions
    from tinygs_amd.train import TrainStep

    scene = scenes.config3(seed=7, n=gaussians, width=image, height=image)
    ts = TrainStep(scene, l1_weight=0.8, ssim_weight=0.2, sparse_grads=False)
    base = ts.gaussians.sh_coefficient_0().clone()
    means = ts.gaussians.means()

    # the target image: colours shifted by a smooth function of the position
    shift = torch.stack([torch.sin(means[:, 0]), torch.cos(means[:, 0]), -torch.sin(means[:, 0])], dim=1)
    ts.gaussians.sh_coefficient_0().copy_(base + 0.8 * shift)
    ts.forward()
    ts.target.data.copy_(ts.pred.data)

    t = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}[dtype]
    features = encode_positions(means, octaves=6, dtype=t)
    net = AttributeNetwork(features.shape[1], 3, width=width, blocks=blocks, dtype=t)
    muon = net.optimizer()
    muon.set_params({"lr": 0.02, "weight_decay": 0.0})
    net.vectors.grad = net.vector_grads
    adam = torch.optim.Adam([net.vectors], lr=2e-3)
    # the loss gradients of an image are about 1 / pixels: halves get them scaled
    scale = 4096.0 if t == torch.float16 else 1.0
    losses = []
    for step in range(steps):
        change = net.forward(features)
        ts.gaussians.sh_coefficient_0().copy_(base + change.float())
        ts.zero()
        ts.forward()
        ts.losses_and_grad()
        ts.backward()
        net.backward((ts.grads.sh_coefficient_0() * scale).to(t))
        muon.step(1.0)
        if scale != 1.0:
            net.vector_grads.mul_(1.0 / scale)
        adam.step()
        losses.append(ts.loss_img.data.float().mean())
        if step % 10 == 0 or step == steps - 1:
            log(f"step {step}: loss {float(losses[-1]):.4e}")
    return [float(v) for v in losses]


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--gaussians", type=int, default=20000)
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--dtype", default="bfloat16", choices=["float32", "float16", "bfloat16"])
    a = ap.parse_args()
    recolour(a.gaussians, a.steps, dtype=a.dtype)
