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


@pytest.mark.parametrize("temperature", [1.0, 1.7, 2.0])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("rows,vocab", [(len(MASKS) + 8, 900), (900, 300), (len(MASKS) + 8, 70001)])
def test_rows_that_a_mask_leaves_nothing(rows, vocab, dtype, temperature):
    """All logits of a row are the mask (or its largest value): the student is uniform there, so the loss is
    sum p log p + log of how many are level. That logarithm comes from an fp32 sum of equal terms, in chains of up to
    1024 (2^-14); where no other path is taken, up to 2^20 in base 2, the logits themselves are held to 2^-24 of their
    size, twice."""
    import math

    import torch

    import neptune_opt_b200 as NB

    x, t, index, _ = _make(rows, vocab, 8, dtype, 5)
    info = torch.finfo(x.dtype)
    want, wstats = NB.run_distill_loss(x, t, index, temperature=temperature)
    masks = [m for m in MASKS if m >= info.min] + [info.min, info.max, 1e4]
    for i, mask in enumerate(masks):
        x[i] = mask
    n = len(masks)
    x[n] = -math.inf
    x[n, :100] = info.min
    index[n] = torch.arange(8, device="cuda")
    x[n + 1] = -math.inf
    x[n + 2] = -math.inf
    x[n + 2, 5] = math.nan
    x[n + 3, 5] = math.inf
    loss, stats = NB.run_distill_loss(x, t, index, temperature=temperature)
    p = torch.softmax(t.double() / temperature, -1)
    for i in range(n + 1):
        size = x[i, 0].abs().double().item() / temperature
        ref = (p[i] * p[i].log()).sum().item() + math.log(100 if i == n else vocab)
        tol = 2.0 ** -13 + (2.0 ** -22 * size if size * 1.45 < 2.0 ** 20 else 0.0)
        assert abs(loss[i].item() - ref) <= tol, (i, x[i, 0].item(), loss[i].item(), ref, tol)
        lse = x[i, 0].double().item() / temperature + math.log(100 if i == n else vocab)
        assert abs(stats[i, 0].double().item() - lse) <= 2.0 ** -21 * abs(lse) + 2.0 ** -13, (i, x[i, 0].item())
    assert stats[n + 1, 0] == -math.inf and stats[n + 2:n + 4, 0].isnan().all() and loss[n + 2:n + 4].isnan().all()
    assert torch.equal(loss[n + 4:], want[n + 4:]) and torch.equal(stats[n + 4:], wstats[n + 4:])


@pytest.mark.parametrize("temperature", [0.9, 1.0, 1.7, 3.0])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,vocab", [(len(MASKS), 900), (900, 300)])
def test_gradients_of_rows_that_a_mask_leaves_nothing(rows, vocab, dtype, temperature):
    """The fp32 log-sum-exp of such a row says no more than the logits' size, so q is anything up to 1 there, and the
    gradient at most grad / T (mass + sum p) = 2 grad / T."""
    import torch

    import neptune_opt_b200 as NB

    x, t, index, grad = _make(rows, vocab, 8, dtype, 5)
    plain = x.clone()
    for i, mask in enumerate(MASKS):
        x[i] = max(mask, -3e38 * min(temperature, 1.0))
    _, stats = NB.run_distill_loss(x, t, index, temperature=temperature)
    dx = NB.distill_loss_backward(grad, x, t, index, stats, temperature=temperature)
    assert (dx.double().abs() <= 2.01 * grad.double().abs()[:, None] / temperature).all()
    _, stats = NB.run_distill_loss(plain, t, index, temperature=temperature)
    want = NB.distill_loss_backward(grad, plain, t, index, stats, temperature=temperature)
    assert torch.equal(dx[len(MASKS):], want[len(MASKS):])
