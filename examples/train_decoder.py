"""Training a small decoder with the operators together.

Every layer: queries, keys and values in one projection, the norms of queries and
keys with their rotation (``QKNormRope``), attention, the gated feed-forward block
(``GatedFFN``).  Each step averages the gradients of a few micro-batches and clips
them by their global norm, then ``Muon`` steps the matrices of the layers and
``SCAO`` what is left (norms' weights and the embedding):

    python examples/train_decoder.py [--steps 40] [--dtype bf16]

The model learns to continue sequences that repeat themselves.
"""

from __future__ import annotations

import argparse
import math
import os
import sys

import torch
from torch import nn

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import scao_amd  # noqa: E402

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


class Layer(nn.Module):
    def __init__(self, d_model: int, heads: int, kv_heads: int, d_ff: int, length: int, **kw) -> None:
        super().__init__()
        self.heads, self.kv_heads, self.dim = heads, kv_heads, d_model // heads
        self.norms = nn.ModuleList(nn.RMSNorm(d_model, **kw) for _ in range(2))
        self.qkv = nn.Linear(d_model, (heads + 2 * kv_heads) * self.dim, bias=False, **kw)
        self.rope = scao_amd.QKNormRope(self.dim, length, **kw)
        self.out = nn.Linear(d_model, d_model, bias=False, **kw)
        self.ffn = scao_amd.GatedFFN(d_model, d_ff, packed=True, **kw)

    def attention(self, x: torch.Tensor) -> torch.Tensor:
        rows = self.qkv(x).unflatten(-1, (-1, self.dim))
        q, k, v = rows.split([self.heads, self.kv_heads, self.kv_heads], -2)
        q, k = self.rope(q, k)
        share = self.heads // self.kv_heads
        q, k, v = (t.transpose(1, 2) for t in (q, k.repeat_interleave(share, -2),
                                               v.repeat_interleave(share, -2)))
        logits = (q.float() @ k.float().mT) / math.sqrt(self.dim)
        later = torch.ones(x.shape[1], x.shape[1], dtype=torch.bool, device=x.device).triu(1)
        weights = logits.masked_fill(later, -math.inf).softmax(-1)
        mixed = (weights @ v.float()).to(x.dtype)
        return self.out(mixed.transpose(1, 2).flatten(2))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        x = x + self.attention(self.norms[0](x))
        return x + self.ffn(self.norms[1](x))


class Decoder(nn.Module):
    def __init__(self, vocabulary: int = 64, layers: int = 2, d_model: int = 128, heads: int = 4,
                 kv_heads: int = 2, d_ff: int = 352, length: int = 64, **kw) -> None:
        super().__init__()
        self.embedding = nn.Embedding(vocabulary, d_model, **kw)
        nn.init.normal_(self.embedding.weight, std=d_model ** -0.5)
        self.layers = nn.ModuleList(Layer(d_model, heads, kv_heads, d_ff, length, **kw)
                                    for _ in range(layers))
        self.norm = nn.RMSNorm(d_model, **kw)

    def forward(self, tokens: torch.Tensor) -> torch.Tensor:
        x = self.embedding(tokens)
        for layer in self.layers:
            x = layer(x)
        return self.norm(x) @ self.embedding.weight.t()


def optimizers(model: Decoder, lr: float) -> list:
    """Muon for the layers' matrices, SCAO for the rest."""
    matrices = [p for p in model.layers.parameters() if p.ndim == 2]
    chosen = {id(p) for p in matrices}
    rest = [p for p in model.parameters() if id(p) not in chosen]
    return [scao_amd.Muon(matrices, lr=lr, weight_decay=0.01),
            scao_amd.SCAO(rest, lr=lr / 4, weight_decay=0.0, warmup_steps=10, sparsity=0.0,
                          noise_std_init=0.0, lars_coeff=0.0)]


def train(steps: int = 40, batch: int = 16, micro_batches: int = 2, lr: float = 0.02,
          dtype: str = "bf16", log=print, **sizes) -> list:
    """(loss, gradient norm) of every step"""
    torch.manual_seed(0)
    model = Decoder(device="cuda", dtype=DTYPES[dtype], **sizes)
    vocabulary, length = model.embedding.num_embeddings, model.layers[0].rope.cos.shape[0]
    opts, history = optimizers(model, lr), []
    for step in range(steps):
        model.zero_grad()
        loss = 0.0
        for _ in range(micro_batches):
            period = torch.randint(vocabulary, (batch, length // 4), device="cuda")
            tokens = period.repeat(1, 5)[:, :length + 1]
            logits = model(tokens[:, :-1])
            part = nn.functional.cross_entropy(logits.float().flatten(0, 1), tokens[:, 1:].flatten())
            part.backward()
            loss += part.detach() / micro_batches
        norm = scao_amd.clip_grad_norm_(model.parameters(), 1.0, scale=1.0 / micro_batches)
        for opt in opts:
            opt.step()
        history.append((float(loss), float(norm)))
        if step % 10 == 0 or step == steps - 1:
            log(f"step {step:3d}  loss {history[-1][0]:.4f}  gradient norm {history[-1][1]:.4f}")
    return history


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=40)
    ap.add_argument("--dtype", choices=sorted(DTYPES), default="bf16")
    a = ap.parse_args()
    train(a.steps, dtype=a.dtype)


if __name__ == "__main__":
    main()
