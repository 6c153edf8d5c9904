"""A batch of conversations that share a long prompt, decoded token by token on the package's serving operators.

One transformer block with random weights. The shared prompt's keys and values are computed once (`attention`); then every
step takes each sequence's last token through

    quantized_rms_norm -> q, k, v -> prefix_attention (shared prompt + own cache) -> output projection
    -> quantized_rms_norm with the residual's addition -> vocabulary projection -> penalize_logits -> softmax -> a token

as one CUDA graph that is replayed for every token: caches, lengths and histories are updated on the device. The products
are torch.matmul on the values that the 8-bit outputs stand for.

    python examples/decode_batch.py [--steps 32]

Prints the sequences' tokens.
"""
from __future__ import annotations

import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import neptune_opt_b200 as NB  # noqa: E402


class Decoder:
    """Weights, caches and the state of a batch. `tokens` is [batch, room]: each row's history, `lens` how much of it is
    there; the shared prompt is no part of it."""

    def __init__(self, batch=4, width=256, heads=4, kv_heads=2, vocab=1003, prompt=200, room=64, dim=128, seed=0,
                 dtype=torch.bfloat16):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.heads, self.kv_heads, self.dim, self.vocab = heads, kv_heads, dim, vocab

        def weight(rows, cols):
            return (torch.randn(rows, cols, device="cuda", generator=gen) / math.sqrt(cols)).to(dtype)

        self.embed, self.qkv = weight(vocab, width), weight((heads + 2 * kv_heads) * dim, width)
        self.out, self.head = weight(width, heads * dim), weight(vocab, width)
        self.first, self.second = torch.ones(width, device="cuda", dtype=dtype), torch.ones(width, device="cuda", dtype=dtype)
        # The shared prompt, once.
        tokens = torch.randint(0, vocab, (1, prompt), device="cuda", generator=gen)
        _, k, v = self.project(NB.rms_norm(self.stream(tokens[0]), self.first))
        self.prefix_k, self.prefix_v = k.transpose(0, 1).contiguous(), v.transpose(0, 1).contiguous()
        self.k = torch.zeros(batch, kv_heads, room, dim, device="cuda", dtype=dtype)
        self.v = torch.zeros_like(self.k)
        self.tokens = torch.full((batch, room + 1), -1, device="cuda")
        self.tokens[:, 0] = torch.randint(0, vocab, (batch,), device="cuda", generator=gen)
        self.lens = torch.ones(batch, dtype=torch.int32, device="cuda")
        self.prompt_lens = torch.ones_like(self.lens)
        self.repetition = torch.full((batch,), 1.2, device="cuda")
        self.frequency = torch.full((batch,), 0.3, device="cuda")
        self.temperature = torch.full((batch,), 0.8, device="cuda")
        # Every other sequence may only use the first half of the vocabulary.
        bit = torch.arange(32 * -(-vocab // 32), device="cuda").view(-1, 32)
        half = torch.where(bit < vocab // 2, 1 << (bit % 32), 0).sum(-1).to(torch.int32)
        row = torch.arange(batch, device="cuda")[:, None]
        self.allowed = torch.where(row % 2 == 0, -1, half[None]).to(torch.int32).contiguous()

    def stream(self, tokens):
        return self.embed[tokens] * math.sqrt(self.embed.shape[1])

    def project(self, h):
        qkv = (h @ self.qkv.t()).view(-1, self.heads + 2 * self.kv_heads, self.dim)
        return qkv.split([self.heads, self.kv_heads, self.kv_heads], dim=1)

    def step(self):
        """One token for every sequence: (the penalised logits, their softmax). Updates the state in place."""
        rows = torch.arange(self.tokens.shape[0], device="cuda")
        last = (self.lens - 1).long()
        x = self.stream(self.tokens[rows, last])
        q8, scale, _ = NB.quantized_rms_norm(x, self.first)
        q, k, v = self.project((q8.float() * scale).to(x.dtype))
        self.k[rows, :, last], self.v[rows, :, last] = k, v
        o = NB.prefix_attention(q[:, :, None], self.prefix_k, self.prefix_v, self.k, self.v, self.lens)
        y = o.reshape(o.shape[0], -1) @ self.out.t()
        q8, scale, _ = NB.quantized_rms_norm(y, self.second, x)
        logits = ((q8.float() * scale).to(x.dtype) @ self.head.t()).float()
        logits = NB.penalize_logits(logits, self.tokens, self.lens, self.prompt_lens, repetition=self.repetition,
                                    frequency=self.frequency, temperature=self.temperature, allowed=self.allowed)
        p = NB.softmax(logits)
        self.tokens[rows, last + 1] = p.argmax(-1)
        self.lens += 1
        return logits, p


@torch.no_grad()
def decode(steps=32, **sizes):
    """Tokens of every sequence, [batch, steps + 1]."""
    model = Decoder(room=steps, **sizes)
    state = [t.clone() for t in (model.k, model.v, model.tokens, model.lens)]
    warm = torch.cuda.Stream()
    with torch.cuda.stream(warm):
        model.step()  # loads the library and the products' kernels before the capture
    warm.synchronize()
    for t, s in zip((model.k, model.v, model.tokens, model.lens), state):
        t.copy_(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        model.step()
    for _ in range(steps):
        graph.replay()
    return model.tokens


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--steps", type=int, default=32)
    for row in decode(parser.parse_args().steps).tolist():
        print(" ".join(str(t) for t in row))
