"""Trains a small decoder whose projections keep their inputs compressed.

    python examples/train_gated_block.py [--steps N]

Each block: a fused query / key / value projection (STACRLinear), rotary positions on a part of the head,
causal attention, an output projection, a gated feed-forward block whose two projections share one
compressed input (STACRGatedFeedForward) and its down projection; gradients are clipped to a global
norm before every optimizer step.  The task is synthetic: the second half of every sequence repeats the
first.  Runs on an MI355X.
"""
from __future__ import annotations

import argparse
import os
import sys

import torch
from torch import nn
from torch.nn import functional as F

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "stac-r_amd"))

import stacr_amd  # noqa: E402


class Block(nn.Module):
    def __init__(self, width: int, heads: int, inner: int, **stacr):
        super().__init__()
        self.heads, self.head = heads, width // heads
        self.norm1, self.norm2 = nn.LayerNorm(width), nn.LayerNorm(width)
        self.query_key_value = stacr_amd.STACRLinear.from_linear(nn.Linear(width, 3 * width), **stacr)
        self.dense = stacr_amd.STACRLinear.from_linear(nn.Linear(width, width), **stacr)
        self.feed_forward = stacr_amd.STACRGatedFeedForward.from_linears(
            nn.Linear(width, inner, bias=False), nn.Linear(width, inner, bias=False), activation="silu", **stacr)
        self.down_proj = stacr_amd.STACRLinear.from_linear(nn.Linear(inner, width, bias=False), **stacr)

    def forward(self, x, cos, sin):
        batch, seq, width = x.shape
        qkv = self.query_key_value(self.norm1(x)).view(batch, seq, 3, self.heads, self.head)
        q, k = stacr_amd.rotary(qkv[:, :, 0], qkv[:, :, 1], cos, sin)
        mixed = F.scaled_dot_product_attention(q.transpose(1, 2), k.transpose(1, 2), qkv[:, :, 2].transpose(1, 2),
                                               is_causal=True)
        x = x + self.dense(mixed.transpose(1, 2).reshape(batch, seq, width))
        return x + self.down_proj(self.feed_forward(self.norm2(x)))


class Decoder(nn.Module):
    def __init__(self, vocab: int = 64, width: int = 256, heads: int = 4, inner: int = 680, layers: int = 2,
                 length: int = 64, **stacr):
        super().__init__()
        self.embed = nn.Embedding(vocab, width)
        self.blocks = nn.ModuleList(Block(width, heads, inner, **stacr) for _ in range(layers))
        self.norm, self.head = nn.LayerNorm(width), nn.Linear(width, vocab, bias=False)
        self.rot, self.length = width // heads // 2, length

    def forward(self, tokens):
        cos, sin = stacr_amd.rotary_tables(self.length, self.rot, device=tokens.device)
        x = self.embed(tokens)
        for block in self.blocks:
            x = block(x, cos, sin)
        return self.head(self.norm(x))


def train(steps: int = 200, batch: int = 64, length: int = 64, vocab: int = 64, dtype=torch.bfloat16, seed: int = 0,
          report: int = 50):
    """The losses and gradient norms of ``steps`` steps."""
    torch.manual_seed(seed)
    device = torch.device("cuda")
    model = Decoder(vocab=vocab, length=length, rank=8, residual_budget=0.02, turbo_after_step=None).to(device)
    optimizer = torch.optim.AdamW(model.parameters(), lr=2e-3, betas=(0.9, 0.95))
    losses, norms = [], []
    for step in range(steps):
        half = torch.randint(vocab, (batch, length // 2 + 1), device=device)
        tokens = torch.cat((half, half), 1)[:, :length + 1]
        stacr_amd.set_step(model, step)
        with torch.autocast("cuda", dtype=dtype):
            logits = model(tokens[:, :-1])
        # the first half cannot be known
        loss = F.cross_entropy(logits[:, length // 2:].float().reshape(-1, vocab), tokens[:, length // 2 + 1:].reshape(-1))
        optimizer.zero_grad()
        loss.backward()
        norms.append(stacr_amd.clip_grad_norm(model.parameters(), 1.0))
        optimizer.step()
        losses.append(loss.detach())
        if report and (step + 1) % report == 0:
            print(f"step {step + 1}: loss {float(losses[-1]):.3f}, gradient norm {float(norms[-1]):.3f}", flush=True)
    return [float(v) for v in losses], [float(v) for v in norms]


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--steps", type=int, default=200)
    train(parser.parse_args().steps)
