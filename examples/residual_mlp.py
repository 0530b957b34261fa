"""A residual stack of ReLU^2 MLP blocks, trained on synthetic data.

What stands around the blocks runs as one kernel a step: the first block's
norm (``block_norm``), and from each block's output to the next one's input
the norm after the block, its gate, the scaled residual and the norm before
the next block (``block_join``).  The blocks keep their activations compressed
(``FFNRelu2``), and their weight matrices are updated by orthogonalised steps
(``Muon``); the vectors take a plain gradient step.

    python examples/residual_mlp.py --steps 50
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from bitsparse_amd.bitsparse import TensorBuffer  # noqa: E402
from bitsparse_amd.layers import FFNRelu2  # noqa: E402
from bitsparse_amd.muon import Muon  # noqa: E402
from bitsparse_amd.residual import RowNorm, block_join, block_norm  # noqa: E402


class ResidualMLP(torch.nn.Module):
    """x [tokens, width] -> the last norm of the stream, [tokens, width]"""

    def __init__(self, width: int, hidden: int, depth: int, device="cuda", dtype=torch.bfloat16):
        super().__init__()
        new = lambda *shape, std: torch.nn.Parameter(torch.randn(shape, device=device).mul_(std).to(dtype))  # noqa: E731
        vector = lambda value: torch.nn.Parameter(torch.full((width,), value, device=device, dtype=dtype))  # noqa: E731
        self.up = torch.nn.ParameterList(new(hidden, width, std=width ** -0.5) for _ in range(depth))
        self.down = torch.nn.ParameterList(new(width, hidden, std=hidden ** -0.5) for _ in range(depth))
        self.pre = torch.nn.ParameterList(vector(1.0) for _ in range(depth + 1))
        self.post = torch.nn.ParameterList(vector(1.0) for _ in range(depth))
        self.gate = torch.nn.ParameterList(vector(0.5) for _ in range(depth))
        self.scale = torch.nn.ParameterList(vector(1.0) for _ in range(depth))

    def matrices(self) -> list[torch.nn.Parameter]:
        return [*self.up, *self.down]

    def vectors(self) -> list[torch.nn.Parameter]:
        return [*self.pre, *self.post, *self.gate, *self.scale]

    def forward(self, x: torch.Tensor, buf: TensorBuffer) -> torch.Tensor:
        buf.reset_buffer()
        h = block_norm(x, RowNorm(self.pre[0]))
        for i in range(len(self.up)):
            y = FFNRelu2.apply(h, self.up[i], self.down[i], sparse_data=buf)
            x, h = block_join(x, y, post=RowNorm(self.post[i]), gate=self.gate[i], scale=self.scale[i],
                              pre=RowNorm(self.pre[i + 1]))
        return h


def train(width=256, hidden=1024, depth=4, tokens=512, steps=50, lr=0.02, seed=0) -> list[float]:
    """Losses of `steps` steps on one batch of a fixed random map."""
    torch.manual_seed(seed)
    model = ResidualMLP(width, hidden, depth)
    buf = TensorBuffer(2 * depth * tokens * hidden, device="cuda")
    x = torch.randn(tokens, width, device="cuda").bfloat16()
    target = torch.tanh(x.float() @ torch.randn(width, width, device="cuda") / width ** 0.5)
    muon, sgd = Muon(model.matrices(), lr=lr), torch.optim.SGD(model.vectors(), lr=lr)
    losses = []
    for _ in range(steps):
        loss = (model(x, buf).float() - target).square().mean()
        loss.backward()
        for opt in (muon, sgd):
            opt.step()
            opt.zero_grad()
        losses.append(loss.detach())
    return [v.item() for v in losses]


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("width", 256), ("hidden", 1024), ("depth", 4), ("tokens", 512), ("steps", 50)):
        ap.add_argument(f"--{name}", type=int, default=value)
    ap.add_argument("--lr", type=float, default=0.02)
    a = ap.parse_args()
    for i, v in enumerate(train(a.width, a.hidden, a.depth, a.tokens, a.steps, a.lr)):
        if i % 10 == 0 or i == a.steps - 1:
            print(f"step {i}: loss {v:.4f}", flush=True)
