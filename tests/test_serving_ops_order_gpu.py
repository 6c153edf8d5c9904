"""Serving operators whose inputs are rewritten by the kernel just ahead of them, again and again at the same addresses: each
call sees what was written last, though the operators' kernels start while the ones ahead of them drain."""
from __future__ import annotations

import pytest

from conftest import cuda_available

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_available(), reason="needs a CUDA device")]

STEPS = 24


def in_turn(state, versions, call):
    """The outputs of `call` for each version of the state's tensors: eager with a wait after every one, then back to back, then
    captured as one graph and replayed twice."""
    import torch

    def write(version):
        for t, v in zip(state, version):
            t.copy_(v)

    want = []
    for version in versions:
        write(version)
        torch.cuda.synchronize()
        want.append([t.clone() for t in call()])
        torch.cuda.synchronize()
    got = []
    for version in versions:
        write(version)
        got.append(call())
    torch.cuda.synchronize()
    yield want, got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = []
        for version in versions:
            write(version)
            got.append(call())
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        yield want, got


def same(runs):
    import torch

    for want, got in runs:
        for i, (a, b) in enumerate(zip(want, got)):
            assert all(torch.equal(x, y) for x, y in zip(a, b)), f"call {i}"


@pytest.mark.parametrize("batch,heads,kv_heads,dim,prefix,cache", [
    (32, 32, 8, 128, 2048, 300), (64, 8, 1, 64, 1500, 90), (3, 48, 2, 128, 100, 400), (2, 8, 2, 128, 200, 64)])
def test_attention_sees_the_last_lengths_queries_and_keys(batch, heads, kv_heads, dim, prefix, cache):
    import torch

    import neptune_opt_b200 as NB

    gen = torch.Generator(device="cuda").manual_seed(batch)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=gen).to(torch.bfloat16)

    pk, pv = normal(kv_heads, prefix, dim), normal(kv_heads, prefix, dim)
    shapes = ((batch, heads, 1, dim), (batch, kv_heads, cache, dim), (batch, kv_heads, cache, dim))
    versions = [(torch.randint(0, cache + 1, (batch,), device="cuda", generator=gen).int(), *(normal(*s) for s in shapes))
                for _ in range(STEPS)]
    state = [torch.empty_like(t) for t in versions[0]]
    same(in_turn(state, versions, lambda: NB.prefix_attention(state[1], pk, pv, state[2], state[3], state[0], return_lse=True)))


@pytest.mark.parametrize("rows,vocab,history", [(64, 70001, 300), (3, 200000, 9000), (8, 32000, 300), (40, 50000, 0)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_logits_see_the_last_history_and_temperature(rows, vocab, history, dtype):
    import torch

    import neptune_opt_b200 as NB

    gen = torch.Generator(device="cuda").manual_seed(rows)
    versions = [((torch.randn(rows, vocab, device="cuda", generator=gen) * 3).to(getattr(torch, dtype)),
                 torch.randint(0, vocab, (rows, max(history, 1)), device="cuda", generator=gen),
                 torch.rand(rows, device="cuda", generator=gen) + 0.5,
                 torch.randint(-2 ** 31, 2 ** 31, (rows, -(-vocab // 32)), device="cuda", generator=gen).int()) for _ in range(8)]
    state = [torch.empty_like(t) for t in versions[0]]

    def call():
        names = {"tokens": state[1], "frequency": state[2]} if history else {}
        return [NB.penalize_logits(state[0], **names, temperature=state[2], allowed=state[3])]

    same(in_turn(state, versions, call))


def test_norms_see_the_last_rows():
    import torch

    import neptune_opt_b200 as NB

    gen = torch.Generator(device="cuda").manual_seed(0)
    versions = [tuple(torch.randn(*s, device="cuda", generator=gen) for s in ((300, 1001), (1001,), (300, 1001)))
                for _ in range(STEPS)]
    state = [torch.empty_like(t) for t in versions[0]]
    same(in_turn(state, versions, lambda: [t.view(torch.uint8) for t in NB.quantized_rms_norm(*state)]))
