"""Training operators at the edges of their contracts, on CUDA tensors."""
from __future__ import annotations

import pytest

from conftest import cuda_available

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_available(), reason="needs a CUDA device")]


def _ops():
    import neptune_opt_b200.aot as aot
    import torch

    aot.load()
    return torch.ops.nb200


@pytest.mark.parametrize("shape,gate", [((0, 64), (64,)), ((3, 0, 64), (3, 1, 64)), ((0, 5, 64), (0, 1, 64)),
                                        ((0, 5, 64), (0, 5, 64)), ((0, 64), None)])
def test_gated_norm_ops_without_rows(shape, gate):
    import torch

    x, w = torch.empty(shape, device="cuda"), torch.ones(64, device="cuda")
    g = None if gate is None else torch.ones(gate, device="cuda")
    y, h, rstd = _ops().gated_norm(x, x, g, w, w, 1, 0.5, 1e-6)
    assert y.shape == h.shape == x.shape and rstd.shape == (*shape[:-1], 2)
    grads = _ops().gated_norm_bwd(y, h, x, x, g, rstd, w, w, 1, 0.5)
    assert [None if t is None else t.shape for t in grads] == [x.shape, x.shape, None if g is None else g.shape, w.shape, w.shape]
    assert all(t is None or not t.any() for t in grads)


def test_attention_and_distillation_ops_without_elements():
    import torch

    for shape in ((2, 0, 9, 128), (0, 4, 9, 128), (2, 4, 0, 128)):
        q = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
        grads = _ops().attention_bwd(q, q, q, q, torch.empty(shape[:3], device="cuda"), q, None, True, 0.1)
        assert [t.shape for t in grads] == [q.shape] * 3
    for rows, top in ((0, 4), (0, 0), (3, 0)):
        x, t = torch.randn(rows, 50, device="cuda"), torch.empty(rows, top, device="cuda")
        index = torch.empty(rows, top, dtype=torch.int64, device="cuda")
        loss, stats = _ops().distill_loss(x, t, index, 1.0, None)
        assert loss.shape == (rows,) and stats.shape == (rows, 3) and not loss.any()
        dx = _ops().distill_loss_bwd(torch.ones(rows, device="cuda"), x, t, index, stats, 1.0)
        assert dx.shape == x.shape and not dx.any()
