"""Training with the feed-forward block, the gradient clipping and SCAO together.

A residual stack of gated feed-forward blocks whose weights have been disturbed
learns the outputs of the undisturbed one.  Each step sums the gradients of a few micro-batches, averages and clips
them by their global norm in one call, and takes an SCAO step:

    python examples/train_ffn.py [--steps 60] [--dtype bf16]
"""

from __future__ import annotations

import argparse
import os
import sys

import torch
from torch import nn

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import scao_amd  # noqa: E402

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


class Stack(nn.Module):
    def __init__(self, layers: int, d_model: int, d_ff: int, **kw) -> None:
        super().__init__()
        self.blocks = nn.ModuleList(scao_amd.GatedFFN(d_model, d_ff, "silu", packed=i % 2 == 1, **kw)
                                    for i in range(layers))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        for block in self.blocks:
            x = x + block(x)
        return x


def train(steps: int = 60, layers: int = 2, d_model: int = 256, d_ff: int = 704, tokens: int = 512,
          micro_batches: int = 4, max_norm: float = 1.0, lr: float = 4e-3, dtype: str = "bf16",
          log=print) -> list:
    """(loss, gradient norm) of every step"""
    kw = dict(device="cuda", dtype=DTYPES[dtype])
    torch.manual_seed(0)
    teacher, model = Stack(layers, d_model, d_ff, **kw), Stack(layers, d_model, d_ff, **kw)
    with torch.no_grad():
        for p, q in zip(model.parameters(), teacher.parameters()):
            q *= 2.0
            p.copy_(q + 0.5 * q.std() * torch.randn_like(q))
    opt = scao_amd.SCAO(model.parameters(), lr=lr, weight_decay=0.0, k_min=32, k_max=32,
                        max_precond_dim=1024, warmup_steps=20, precond_freq=10,
                        min_precond_updates=1, sparsity=0.0, noise_std_init=0.0, lars_coeff=0.0)
    history = []
    for step in range(steps):
        opt.zero_grad()
        loss = 0.0
        for _ in range(micro_batches):
            x = torch.randn(4, tokens // 4, d_model, device="cuda").to(DTYPES[dtype])
            with torch.no_grad():
                target = teacher(x)
            part = (model(x) - target).float().square().mean()
            part.backward()
            loss += part.detach() / micro_batches
        norm = scao_amd.clip_grad_norm_(model.parameters(), max_norm, scale=1.0 / micro_batches)
        opt.step()
        history.append((float(loss), float(norm)))
        if step % 10 == 0 or step == steps - 1:
            log(f"step {step:3d}  loss {history[-1][0]:.5f}  gradient norm {history[-1][1]:.4f}")
    return history


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--dtype", choices=sorted(DTYPES), default="bf16")
    a = ap.parse_args()
    train(a.steps, dtype=a.dtype)


if __name__ == "__main__":
    main()
