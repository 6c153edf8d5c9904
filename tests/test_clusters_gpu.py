"""Kernels whose CTAs meet through distributed shared memory, launched back to back: clusters start while others of
the same and the previous launch drain, and every launch gives the same bits."""
from __future__ import annotations

import pytest

from conftest import cuda_available
from test_distill_gpu import _make, _run_and_check

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_available(), reason="needs a CUDA device")]


@pytest.mark.parametrize("rows", [1, 40, 80, 150, 300, 600])
def test_distillation_rows_shared_by_16_to_1_ctas(rows):
    import torch

    import neptune_opt_b200 as NB

    x, t, index, grad = (a.repeat(rows, *[1] * (a.dim() - 1)) for a in _make(1, 70001, 24, "bfloat16", rows))
    x[:, 5] += torch.arange(rows, device="cuda") % 7  # not every row alike
    loss, _ = _run_and_check(x, t, index, grad, "bfloat16", label=f"{rows}")
    runs = [NB.run_distill_loss(x, t, index)[0] for _ in range(64)]
    assert all(torch.equal(r, loss) for r in runs)


@pytest.mark.parametrize("rows", [1, 30, 100, 256])
def test_wide_rows_shared_by_16_to_2_ctas(rows):
    """The folds and RMSNorm of few, very wide rows."""
    import torch

    import neptune_opt_b200 as NB

    gen = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.randn(rows, 20480, device="cuda", generator=gen)
    gamma = torch.randn(20480, device="cuda", generator=gen)
    lse, y = NB.logsumexp(x), NB.rms_norm(x, gamma)
    runs = [(NB.logsumexp(x), NB.rms_norm(x, gamma)) for _ in range(64)]
    assert all(torch.equal(a, lse) and torch.equal(b, y) for a, b in runs)
    xd = x.double()
    # fp32 sums of 20480 terms of one sign: off by less than 20480 2^-24 = 2^-9.6 in any order, which logsumexp takes
    # as it is and the norm halves; the rest is a few roundings.
    assert ((lse.double() - torch.logsumexp(xd, -1)).abs() <= 2.0 ** -9).all()
    want = xd * torch.rsqrt(xd.square().mean(-1, keepdim=True) + 1e-6) * gamma.double()
    assert ((y.double() - want).abs() <= 2.0 ** -9 * want.abs()).all()
