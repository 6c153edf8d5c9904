"""GPU parity of attention behind a shared prefix where every score of a row is far from 0.

Each score is one product of a power of two and a value with no more bits than the type has, so it is exact in any order; the
64-bit softmax of the exact scores is the reference. Tolerances as in test_prefix_attention_gpu.py without the error of a
score, with u = half a step of the type, A = sum p |v| / sum p: (2 u + parts 2^-21) A, the probabilities' own error 2^-19 A
twice, fp16's smallest probability 2^-31 max |v| for each key; lse 2^-20 (1 + |lse|).
"""
from __future__ import annotations

import pytest

from conftest import cuda_available

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_available(), reason="needs a CUDA device")]

HALF_STEP = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
# (batch, heads, kv_heads, tokens, prefix, cache): the single kernel; parts of the stream; the prefix on the tensor cores in
# alternating streams, in paired ones, and in both.
CALLS = [(2, 8, 2, 1, 200, 64), (2, 8, 2, 2, 300, 2100), (40, 8, 2, 1, 1000, 64), (20, 48, 2, 1, 700, 30),
         (33, 36, 2, 1, 1025, 90)]


def make(call, dim, dtype, far, small=0.0):
    """q reads the first column alone; scores are `far` (times a little where `small` is not 0) but for every third head,
    whose are within +-4."""
    import torch

    batch, heads, kv_heads, tokens, prefix, cache = call
    gen = torch.Generator(device="cuda").manual_seed(dim + prefix)
    dt = getattr(torch, dtype)
    q = torch.zeros(batch, heads, tokens, dim, device="cuda", dtype=dt)
    q[..., 0] = 1.0
    q[:, ::3, :, 0], q[:, ::3, :, 1] = 0.0, 1.0

    def keys(*shape):
        k = torch.randn(*shape, dim, device="cuda", generator=gen).to(dt)
        k[..., 0] = far
        if small:
            k[..., 0] = torch.where(torch.rand(*shape, device="cuda", generator=gen) < 0.4, far, far * (1 + small))
        return k

    def values(*shape):
        return torch.randn(*shape, dim, device="cuda", generator=gen).to(dt)

    lens = torch.tensor([cache if i % 3 else max(tokens, cache // (i + 1)) for i in range(batch)], dtype=torch.int32, device="cuda")
    return (q, keys(kv_heads, prefix), values(kv_heads, prefix), keys(batch, kv_heads, cache),
            values(batch, kv_heads, cache), lens)


def check(args, scale, parts):
    import torch

    import neptune_opt_b200 as NB

    q, pk, pv, k, v, lens = args
    o, lse = NB.prefix_attention(*args, scale=scale, return_lse=True)
    b, h, t, d = q.shape
    hk, u = k.shape[1], HALF_STEP[str(q.dtype)[6:]]
    for i in range(b):
        for j in range(t):
            own = int(lens[i]) - t + j + 1
            kk, vv = (torch.cat([x, y[i, :, :own]], 1).double() for x, y in ((pk, k), (pv, v)))
            s = torch.einsum("gpd,gkd->gpk", q[i, :, j].double().view(hk, h // hk, d), kk) * scale
            p = torch.softmax(s, -1)
            mean = torch.matmul(p, vv.abs())
            tol = (2 * u + parts * 2.0 ** -21 + 2.0 ** -18) * mean + kk.shape[1] * 2.0 ** -31 * vv.abs().amax()
            off = (o[i, :, j].double() - torch.matmul(p, vv).view(h, d)).abs()
            assert bool((off <= tol.view(h, d)).all()), f"sequence {i}, token {j}: o off by up to {off.amax():.3e}"
            want = torch.logsumexp(s, -1).view(h)
            off = (lse[i, :, j].double() - want).abs()
            assert bool((off <= 2.0 ** -20 * (1 + want.abs())).all()), f"sequence {i}, token {j}: lse off by up to {off.amax():.3e}"


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("far", [-2.0 ** 9, 2.0 ** 14, -2.0 ** 34, 2.0 ** 66, -2.0 ** 123, 2.0 ** 127])
def test_scores_alike_and_far_from_zero(call, dim, far):
    """As behind a mask that adds the same large number everywhere: the weights are those without it."""
    check(make(call, dim, "bfloat16", far), dim ** -0.5, 2048)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("far,scale", [(-2.0 ** 15, 0.125), (2.0 ** 15, 2.0 ** 20)])
def test_scores_alike_and_far_from_zero_in_fp16(call, dim, far, scale):
    check(make(call, dim, "float16", far), scale if scale < 1 else 1.0, 2048)
    if scale > 1:  # scores of 2^35, beside which those of the other heads would be far apart, too
        args = make(call, dim, "float16", far)
        args[0][:, ::3] = args[0][:, 1:2]
        check(args, scale, 2048)


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("far", [-2.0 ** 20, 2.0 ** 40, -2.0 ** 100])
def test_a_step_of_the_type_apart(call, far):
    """Two scores, one step of bf16 apart, which is so much that only the higher one has weight."""
    check(make(call, 128, "bfloat16", far, 2.0 ** -7), 128 ** -0.5, 2048)


def test_the_lowest_values_of_the_type():
    """Keys at finfo.min are as good as masked beside others, and all alike where there are no others."""
    import torch

    for call in CALLS:
        args = make(call, 128, "bfloat16", torch.finfo(torch.bfloat16).min)
        check(args, 128 ** -0.5, 2048)
        args[1][:, ::2, 0] = 1.0
        check(args, 128 ** -0.5, 2048)
