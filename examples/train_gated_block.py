"""A few training steps and a rollout of a small Swin emulator with gated feed-forward networks and sandwich
norms, in 16-bit parameters with a plain PyTorch optimizer.

    python examples/train_gated_block.py [--steps 20] [--dim 256] [--depth 4] [--grid 72x144]

The model is the framework's own (``mlp_type="swiglu"``, ``block_norm="sandwich"``).  Its blocks run
``ops.gated_mlp`` and ``ops.norm_gate_residual``; each step clips the gradients, which here are separate bf16
tensors and not views of the trainer's flat buffer, with ``ops.clip_grad_norm``.  Synthetic data: the target is
the input field advected by one patch.  Needs a GPU with the built extension, or runs the plain operators on a
CPU.
"""

import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from neural_scaling_weather_b200 import ops  # noqa: E402
from neural_scaling_weather_b200.models.swin import SwinTransformer  # noqa: E402
from neural_scaling_weather_b200.utils.misc import get_spatial_coords  # noqa: E402


def build(dim: int, depth: int, grid, channels: int, device, dtype) -> SwinTransformer:
    h, w = grid
    lat = torch.linspace(90, -90, h + 1)[:-1].numpy()
    lon = (torch.arange(w) * 360.0 / w).numpy()
    metadata = {"sp_shapes": [[h], [w]], "n_channels": channels, "coords": get_spatial_coords((lat, lon)).float()}
    model = SwinTransformer(window_size=(9, 9), patch_size=4, in_chans=channels, out_chans=channels, embed_dim=dim,
                            depth=depth, num_heads=dim // 64, mlp_ratio=8 / 3, domain_metadata=metadata,
                            mlp_type="swiglu", block_norm="sandwich")
    return model.to(device=device, dtype=dtype)


def train(model, steps: int, grid, channels: int, max_norm: float = 1.0, lr: float = 0.05, seed: int = 0):
    """``steps`` SGD steps; returns the losses and the gradient norms before clipping."""
    param = next(model.parameters())
    gen = torch.Generator(device=param.device).manual_seed(seed)
    opt = torch.optim.SGD(model.parameters(), lr=lr, momentum=0.9)
    losses, norms = [], []
    for _ in range(steps):
        x = torch.randn(2, 1, channels, *grid, generator=gen, device=param.device).to(param.dtype)
        y = torch.roll(x, 4, dims=-1)
        loss = (model(x) - y).float().square().mean()
        loss.backward()
        norms.append(ops.clip_grad_norm([p.grad for p in model.parameters()], max_norm))
        opt.step()
        opt.zero_grad(set_to_none=True)
        losses.append(loss.detach())
    return torch.stack(losses).cpu(), torch.stack(norms).cpu()


@torch.no_grad()
def rollout(model, x, steps: int):
    for _ in range(steps):
        x = model(x)
    return x


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--dim", type=int, default=256)
    ap.add_argument("--depth", type=int, default=4)
    ap.add_argument("--grid", default="72x144")
    ap.add_argument("--channels", type=int, default=8)
    a = ap.parse_args()
    grid = tuple(int(v) for v in a.grid.split("x"))
    cuda = torch.cuda.is_available()
    device, dtype = ("cuda", torch.bfloat16) if cuda else ("cpu", torch.float32)
    torch.manual_seed(0)
    model = build(a.dim, a.depth, grid, a.channels, device, dtype)
    t = time.perf_counter()
    losses, norms = train(model, a.steps, grid, a.channels)
    t = time.perf_counter() - t
    for i in range(0, a.steps, max(1, a.steps // 10)):
        print(f"step {i:4d}  loss {losses[i]:.4f}  gradient norm {norms[i]:.3f}")
    print(f"{a.steps} steps in {t:.2f} s; loss {losses[0]:.4f} -> {losses[-1]:.4f}")
    x = torch.randn(1, 1, a.channels, *grid, device=device).to(dtype)
    print(f"rollout of 4 steps: output std {rollout(model, x, 4).float().std():.3f}")


if __name__ == "__main__":
    main()
