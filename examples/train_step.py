"""A small language model's training loop on the library's operators: an embedding, blocks of layer norm, gated
projection and down projection with a residual, a last norm, and the output projection with its loss.

    python examples/train_step.py [--steps 20] [--dtype f32|bf16] [--tokens 2048] [--width 512] [--classes 8192]

Learns to continue a fixed random cycle over the classes; prints the loss as it falls, and the time of a step.  The
down projections are PyTorch's own linears: run under LD_PRELOAD=vkblas_amd/libvkblas_hipblas.so, they and their
gradients are the library's GEMMs too.
"""
import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from vkblas_amd import torch_nn as vnn  # noqa: E402


class Block(torch.nn.Module):
    def __init__(self, width, hidden, dtype):
        super().__init__()
        self.norm_w = torch.nn.Parameter(torch.ones(width))
        self.norm_b = torch.nn.Parameter(torch.zeros(width))
        self.gate_up = torch.nn.Parameter((torch.randn(2 * hidden, width) * width ** -0.5).to(dtype))
        self.down = torch.nn.Parameter((torch.randn(width, hidden) * hidden ** -0.5).to(dtype))

    def forward(self, x):
        h = vnn.gated_linear(vnn.layer_norm(x, self.norm_w, self.norm_b), self.gate_up)
        return x + torch.nn.functional.linear(h, self.down)


class Model(torch.nn.Module):
    def __init__(self, width, hidden, layers, classes, dtype):
        super().__init__()
        self.embed = torch.nn.Parameter(torch.randn(classes, width).to(dtype))
        self.blocks = torch.nn.ModuleList(Block(width, hidden, dtype) for _ in range(layers))
        self.norm_w = torch.nn.Parameter(torch.ones(width))
        self.head = torch.nn.Parameter((torch.randn(classes, width) * width ** -0.5).to(dtype))

    def forward(self, tokens, target):
        x = self.embed[tokens]
        for b in self.blocks:
            x = b(x)
        return vnn.linear_cross_entropy(vnn.layer_norm(x, self.norm_w), self.head, target)


def train(steps=20, dtype=torch.bfloat16, tokens=2048, width=512, hidden=1408, layers=2, classes=8192, lr=1e-3, log=print):
    torch.manual_seed(0)
    model = Model(width, hidden, layers, classes, dtype).cuda()
    opt = torch.optim.AdamW(model.parameters(), lr=lr)
    successor = torch.randperm(classes, device="cuda")
    losses, start = [], time.time()
    for step in range(steps):
        t = torch.randint(0, min(classes, 256), (4, tokens // 4), device="cuda")
        loss = model(t, successor[t])
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(loss.item())
        if step == 0 or step == steps - 1 or step % 10 == 9:
            log(f"step {step + 1}: loss {losses[-1]:.3f}", flush=True)
        if step == 0:
            start = time.time()
    if steps > 1:
        log(f"{(time.time() - start) / (steps - 1) * 1e3:.2f} ms a step", flush=True)
    return losses


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--dtype", choices=["f32", "bf16"], default="bf16")
    for name, value in (("tokens", 2048), ("width", 512), ("hidden", 1408), ("layers", 2), ("classes", 8192)):
        ap.add_argument("--" + name, type=int, default=value)
    a = vars(ap.parse_args())
    a["dtype"] = {"f32": torch.float32, "bf16": torch.bfloat16}[a["dtype"]]
    train(**a)
