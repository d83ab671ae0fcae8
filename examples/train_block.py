"""Fit encoder blocks to a target with the training operators: a windowed block and a global one in bf16, f32 master
weights, gradients clipped into f32 buffers, plain SGD with momentum.

    python examples/train_block.py --steps 20 --dim 256 --heads 4 --side 28

Each step is one forward pass (fused attention that keeps its softmax sums, LayerNorm), one backward pass (the
attention's and LayerNorm's gradient kernels) and one clip_grad_norm; the projections are library matrix products.
"""
import argparse
import importlib
import pathlib
import sys

import torch

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parents[1]))
samrs = importlib.import_module("sam-rs_b200")


def block_params(dim, heads, span, gen):
    """Random parameters of one block whose attention spans span x span tokens."""
    shapes = {"norm1_w": (dim,), "norm1_b": (dim,), "qkv_w": (3 * dim, dim), "qkv_b": (3 * dim,), "proj_w": (dim, dim),
              "proj_b": (dim,), "rel_pos_h": (2 * span - 1, dim // heads), "rel_pos_w": (2 * span - 1, dim // heads),
              "norm2_w": (dim,), "norm2_b": (dim,), "lin1_w": (4 * dim, dim), "lin1_b": (4 * dim,),
              "lin2_w": (dim, 4 * dim), "lin2_b": (dim,)}
    params = {k: torch.randn(*s, generator=gen, device="cuda") * s[-1] ** -0.5 for k, s in shapes.items()}
    params["norm1_w"], params["norm2_w"] = (torch.ones(dim, device="cuda") for _ in range(2))
    return params


def train(steps=20, dim=256, heads=4, side=28, window=14, images=1, lr=0.5, max_norm=1.0, seed=0):
    """Returns the losses and the gradient norms before clipping, one of each per step."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    masters = [block_params(dim, heads, window or side, gen), block_params(dim, heads, side, gen)]
    blocks = [samrs.train.TrainBlock({k: v.bfloat16() for k, v in m.items()}, heads, ws)
              for m, ws in zip(masters, (window, 0))]
    params = [p for b in blocks for p in b.parameters()]
    master = [v for m in masters for v in m.values()]
    clipped = [torch.empty_like(v) for v in master]  # f32
    momentum = [torch.zeros_like(v) for v in master]
    x = torch.randn(images, side, side, dim, generator=gen, device="cuda").bfloat16()
    target = torch.randn(images, side, side, dim, generator=gen, device="cuda")
    losses, norms = [], []
    for _ in range(steps):
        y = x
        for b in blocks:
            y = b(y)
        loss = (y.float() - target).square().mean()
        loss.backward()
        norms.append(samrs.clip_grad_norm([p.grad for p in params], max_norm, out=clipped))
        torch._foreach_mul_(momentum, 0.9)
        torch._foreach_add_(momentum, clipped)
        torch._foreach_add_(master, momentum, alpha=-lr * 0.1)
        with torch.no_grad():
            torch._foreach_copy_(params, master)
        for p in params:
            p.grad = None
        losses.append(loss.detach())
    if samrs.device_status():
        raise RuntimeError("a kernel reported a fault")
    return [float(v) for v in losses], [float(v) for v in norms]


def main():
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, default in (("steps", 20), ("dim", 256), ("heads", 4), ("side", 28), ("window", 14), ("images", 1)):
        p.add_argument(f"--{name}", type=int, default=default)
    p.add_argument("--lr", type=float, default=0.5)
    p.add_argument("--max-norm", type=float, default=1.0)
    for k, (loss, norm) in enumerate(zip(*train(**vars(p.parse_args())))):
        print(f"step {k:3d}  loss {loss:.4f}  gradient norm {norm:.4f}")


if __name__ == "__main__":
    main()
