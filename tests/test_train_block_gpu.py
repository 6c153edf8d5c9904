"""The training operators together: examples/train_block.py learns, and its gradients agree with the same block
written in torch operations (float32 on the same bf16 parameters)."""
from __future__ import annotations

import importlib.util
import math
import os

import pytest

from conftest import ROOT, cuda_available

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_available(), reason="needs a CUDA device")]


def _example():
    spec = importlib.util.spec_from_file_location("train_block", os.path.join(ROOT, "examples", "train_block.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_the_example_learns():
    losses = _example().train(steps=20, verbose=False)
    assert all(math.isfinite(v) for v in losses)
    assert losses[-1] < 0.5 * losses[0], losses


def test_gradients_of_the_block_agree_with_torch():
    """Direction and length of every parameter's gradient. The block rounds to bf16 between its operators
    (2^-8 each, a dozen of them on the longest path, in independent directions), which moves a gradient by
    about sqrt(12) 2^-8 = 1.4% of its norm; 6% bounds it."""
    import torch

    import neptune_opt_b200 as NB

    torch.manual_seed(3)
    width, heads, kv, vocab, b, n, top = 256, 4, 2, 701, 3, 70, 8
    model = _example().Block(width, heads, kv, vocab, torch.bfloat16)
    with torch.no_grad():
        model.gate.normal_()
    tokens = torch.randint(0, vocab, (b, n), device="cuda")
    lens = torch.tensor([n, 33, 0], dtype=torch.int32, device="cuda")
    live = torch.arange(n, device="cuda")[None] < lens[:, None]
    index = torch.randint(0, vocab, (b, n, top), device="cuda").masked_fill(~live[..., None], -1)
    teacher = torch.randn(b, n, top, device="cuda")
    NB.distill_loss(model(tokens, lens), teacher, index).sum().backward()

    w = {k: p.detach().float().requires_grad_() for k, p in model.named_parameters()}

    def norm(x, weight):
        return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight

    x = w["embed"][tokens] * math.sqrt(width)
    h = norm(x, 1.0)
    q, k, v = (h @ w["qkv"].t()).view(b, n, heads + 2 * kv, 128).transpose(1, 2).split([heads, kv, kv], 1)
    k, v = (t.repeat_interleave(heads // kv, 1) for t in (k, v))
    pos = torch.arange(n, device="cuda")
    ok = (pos[None] <= pos[:, None])[None, None] & live[:, None, None, :] & live[:, None, :, None]
    s = (q @ k.transpose(-1, -2) / math.sqrt(128)).masked_fill(~ok, -1e30)
    p = torch.softmax(s, -1).masked_fill(~ok, 0.0)
    y = (p @ v).transpose(1, 2).reshape(b, n, -1) @ w["out"].t()
    z = x + torch.sigmoid(w["gate"]) * norm(y, w["post"])
    logits = norm(z, w["pre"]) @ w["head"].t()
    logq = torch.log_softmax(logits, -1).gather(-1, index.clamp(min=0))
    t = torch.softmax(teacher, -1)
    ((t * (t.log() - logq)).sum(-1) * live).sum().backward()
    for name, param in model.named_parameters():
        got, ref = param.grad.float(), w[name].grad
        rel = (got - ref).norm() / ref.norm()
        assert rel < 0.06, (name, rel.item())


def test_operators_replay_from_a_graph():
    """Every operator captured into one CUDA graph; replays on new inputs equal the eager calls bit for bit."""
    import torch

    import neptune_opt_b200 as NB

    gen = torch.Generator(device="cuda").manual_seed(1)

    def normal(*shape, dtype=torch.bfloat16):
        return torch.randn(*shape, device="cuda", generator=gen).to(dtype)

    q, k, v, g = normal(2, 8, 300, 128), normal(2, 1, 300, 128), normal(2, 1, 300, 128), normal(2, 8, 300, 128)
    x, r, gate, w, gh = normal(4, 50, 333), normal(4, 50, 333), normal(4, 1, 333), normal(333), normal(4, 50, 333)
    logits, teacher = normal(9, 70001), normal(9, 16)
    index = torch.randint(0, 70001, (9, 16), device="cuda", generator=gen)
    weight = torch.rand(9, device="cuda", generator=gen)

    def everything():
        o, lse = NB.attention(q, k, v, causal=True, return_lse=True)
        y, h, rstd = NB.run_gated_residual_norm(x, r, gate, post_weight=w, pre_weight=w, gate_act="tanh")
        loss, stats = NB.run_distill_loss(logits, teacher, index)
        return (o, lse, *NB.attention_backward(q, k, v, o, lse, g, causal=True), y, h,
                *NB.gated_residual_norm_backward(y, gh, x, r, gate, rstd, post_weight=w, pre_weight=w, gate_act="tanh"),
                loss, NB.distill_loss_backward(weight, logits, teacher, index, stats))

    everything()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = everything()
    for t in (q, k, v, g, x, r, gate, gh, logits, teacher):
        t.copy_(normal(*t.shape))
    graph.replay()
    torch.cuda.synchronize()
    got = [t.clone() for t in out]
    assert all(torch.equal(a, b) for a, b in zip(got, everything()))
