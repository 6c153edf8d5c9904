"""A few training steps of one transformer block on the package's training operators.

The block normalises before and after its attention, adds the attention's output to the residual stream
through a gate and a residual scale, and is trained to follow a teacher of which only the top logits of
each position were kept. Projections are torch.matmul; everything between them is this package:

    rms_norm -> q, k, v -> attention -> o projection -> gated_residual_norm -> vocabulary projection
    -> distill_loss, and the backward pass of each through autograd

    python examples/train_block.py [--steps 20]

Prints the loss of every step; with the defaults it falls from about 7 to about 0.1.
"""
from __future__ import annotations

import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import neptune_opt_b200 as NB  # noqa: E402


class Block(torch.nn.Module):
    def __init__(self, width, heads, kv_heads, vocab, dtype):
        super().__init__()
        self.heads, self.kv_heads = heads, kv_heads

        def weight(rows, cols):
            return torch.nn.Parameter((torch.randn(rows, cols, device="cuda") / math.sqrt(cols)).to(dtype))

        self.embed = weight(vocab, width)
        self.qkv = weight((heads + 2 * kv_heads) * 128, width)
        self.out = weight(width, heads * 128)
        self.gate = torch.nn.Parameter(torch.zeros(width, device="cuda", dtype=dtype))
        self.post = torch.nn.Parameter(torch.ones(width, device="cuda", dtype=dtype))
        self.pre = torch.nn.Parameter(torch.ones(width, device="cuda", dtype=dtype))
        self.head = weight(vocab, width)
        self.first = torch.ones(width, device="cuda", dtype=dtype)

    def forward(self, tokens, seq_lens):
        x = self.embed[tokens] * math.sqrt(self.embed.shape[1])
        # The norm before the block: a gated norm whose block output is zero.
        _, h = NB.gated_residual_norm(torch.zeros_like(x), x, pre_weight=self.first)
        b, n, _ = h.shape
        qkv = (h @ self.qkv.t()).view(b, n, self.heads + 2 * self.kv_heads, 128).transpose(1, 2)
        q, k, v = qkv.split([self.heads, self.kv_heads, self.kv_heads], dim=1)
        o = NB.attention(q, k, v, causal=True, seq_lens=seq_lens)
        y = o.transpose(1, 2).reshape(b, n, -1) @ self.out.t()
        _, h = NB.gated_residual_norm(y, x, self.gate, post_weight=self.post, pre_weight=self.pre, gate_act="sigmoid")
        return h @ self.head.t()


def train(steps=20, batch=4, seq=200, width=512, heads=4, kv_heads=2, vocab=4001, top=16, seed=0, dtype=torch.bfloat16,
          verbose=True):
    """Losses of each step."""
    torch.manual_seed(seed)
    model = Block(width, heads, kv_heads, vocab, dtype)
    optimiser = torch.optim.AdamW(model.parameters(), lr=3e-3, weight_decay=0.0)
    tokens = torch.randint(0, vocab, (batch, seq), device="cuda")
    # A right-padded batch: padding positions have no teacher entries.
    seq_lens = torch.tensor([seq] + [1 + seq * (i + 1) // (batch + 1) for i in range(batch - 1)], dtype=torch.int32,
                            device="cuda")
    padding = torch.arange(seq, device="cuda")[None] >= seq_lens[:, None]
    first = torch.randint(0, vocab, (batch, seq, 1), device="cuda")
    index = (first + 7 * torch.arange(top, device="cuda")) % vocab
    index = index.masked_fill(padding[..., None], -1)
    teacher = torch.randn(batch, seq, top, device="cuda").sort(-1, descending=True).values * 2
    count = (~padding).sum()
    losses = []
    for step in range(steps):
        logits = model(tokens, seq_lens)
        loss = NB.distill_loss(logits, teacher, index, temperature=1.0).sum() / count
        optimiser.zero_grad(set_to_none=True)
        loss.backward()
        optimiser.step()
        losses.append(loss.item())
        if verbose:
            print(f"step {step:3d}  loss {losses[-1]:.4f}")
    return losses


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--steps", type=int, default=20)
    train(parser.parse_args().steps)
