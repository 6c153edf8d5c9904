"""The distillation loss on logits masked with large finite values: what a mask adds or writes differs from program to
program (-1e4, -1e9, -1e30, the type's lowest value, ...)."""
from __future__ import annotations

import pytest

from conftest import cuda_available
from test_distill_gpu import _make, _run_and_check

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_available(), reason="needs a CUDA device")]

MASKS = (-1e4, -3e4, -1e9, -1e10, -7e11, -1e15, -1e20, -1e30, -1e37, -2.5e38, -3e38)


@pytest.mark.parametrize("temperature", [0.7, 1.0, 1.7, 2.0, 4.0])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("shape", [(len(MASKS) + 1, 3001, 8), (900, 300, 8), (len(MASKS) + 1, 70001, 8)])
def test_part_of_the_vocabulary_masked(shape, dtype, temperature):
    """Runs of a masked row longer than a thread's share of it, and single masked logits, a CTA, a warp and a cluster
    to a row."""
    import torch

    x, t, index, grad = _make(*shape, dtype, 12)
    info, vocab = torch.finfo(x.dtype), shape[1]
    for i, mask in enumerate((*MASKS, info.min)):
        # What a temperature below 1 takes past fp32's range is not finite in the plain form either.
        mask = max(mask, info.min, -3e38 * min(temperature, 1.0))
        x[i, vocab // 5:] = mask
        x[i, 1:vocab // 5:3] = mask
        index[i] = torch.arange(8, device="cuda") * 3
        index[i, 7] = vocab - 1 if i % 2 else -1
        t[i, 7] = t[i].min() - 1
    _run_and_check(x, t, index, grad, dtype, temperature, label=f"{shape} {dtype} {temperature}")
