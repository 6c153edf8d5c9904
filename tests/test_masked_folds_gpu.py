"""logsumexp and softmax of rows masked with large finite values, in part and whole, on every path (a warp, a CTA or a
cluster a row, the split plan; 16-bit and fp32), against float64.

A sum of exponentials is one of terms of one sign in fp32, in chains of at most 1024 and a tree: 2^-13 with the
exponentials' own error. A result is rounded once to its type, and where a row's maximum is the mask, to fp32 before."""
from __future__ import annotations

import math

import pytest

from conftest import cuda_available

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_available(), reason="needs a CUDA device")]

MASKS = (-1e4, -1e9, -1e10, -7e11, -1e15, -1e20, -1e30, -1e37, -2.3e38, -3.3e38)
UNIT = {"float32": 2.0 ** -23, "bfloat16": 2.0 ** -8}
SHAPES = [(12, 100), (12, 3001), (12, 2048), (400, 2048), (400, 4096), (12, 20000), (12, 65536), (40, 131072), (320, 40960)]


def _check(got, want, dtype, label):
    over = (got.double() - want).abs() - (2.0 ** -13 + UNIT[dtype] * want.abs())
    assert not got.isnan().any() and over.max().item() <= 0, (label, over.argmax().item(), over.max().item())


def _masked(shape, dtype, whole):
    import torch

    gen = torch.Generator(device="cuda").manual_seed(shape[1])
    x = torch.randn(*shape, device="cuda", generator=gen).to(getattr(torch, dtype))
    for i, mask in enumerate(MASKS):
        if whole:
            x[i] = mask
        else:
            x[i, shape[1] // 5:] = mask
            x[i, 1:shape[1] // 5:3] = mask
    if not whole:
        x[len(MASKS), shape[1] // 2:] = torch.finfo(x.dtype).min
    return x


@pytest.mark.parametrize("whole", [False, True])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_logsumexp(shape, dtype, whole):
    import torch

    import neptune_opt_b200 as NB

    x = _masked(shape, dtype, whole)
    want = torch.logsumexp(x.double(), -1)
    _check(NB.logsumexp(x), want, dtype, "serial")
    for block in (None, 1024, 4096):
        _check(NB.run("logsumexp", x, plan="split", block=block), want, dtype, f"split {block}")
    wide = NB.run("lse_scaled", x, T=2.0)
    _check(wide, torch.logsumexp(x.double() / 2, -1), dtype, "scaled")
    assert NB._lib.stream_fault() == 0


@pytest.mark.parametrize("whole", [False, True])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_softmax(shape, dtype, whole):
    import torch

    import neptune_opt_b200 as NB

    x = _masked(shape, dtype, whole)
    want = torch.softmax(x.double(), -1)
    got = NB.softmax(x).double()
    assert ((got - want).abs() <= (2.0 ** -12 + UNIT[dtype]) * want + 1e-30).all()
    got, want = NB.log_softmax(x), torch.log_softmax(x.double(), -1)
    over = (got.double() - want).abs() - (2.0 ** -12 + UNIT[dtype] * want.abs())
    assert not got.isnan().any() and over.max().item() <= 0
    assert not math.isnan(NB.run_softmax_lse(x)[1].double().sum().item())
