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
    assert [t.shape for t in grads] == [x.shape, x.shape, (0,) if g is None else g.shape, w.shape, w.shape]
    assert not any(t.any() for t in grads)


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


@pytest.mark.parametrize("z", [False, True])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("rows,vocab", [(6, 500), (900, 300), (3, 70001)])
def test_rows_whose_kept_teacher_logits_are_all_minus_infinity(rows, vocab, dtype, z):
    """Rows padded with logits of -inf in place of index -1: loss and gradient are 0, whatever the student's logits
    hold, and neighbouring rows are what they are without them. A CTA a row, a warp a row and a cluster a row."""
    import math

    import torch

    import neptune_opt_b200 as NB
    from test_distill_gpu import _make

    x, t, index, grad = _make(rows, vocab, 8, dtype, 5)
    lse = torch.logsumexp(t.float(), -1) + 0.2 if z else None
    want, stats = NB.run_distill_loss(x, t, index, teacher_lse=lse)
    dwant = NB.distill_loss_backward(grad, x, t, index, stats)
    t[1::3] = -math.inf
    index[1::3, 4:] = 0  # the usual padding: one column named again and again
    x[1, 7] = math.nan
    loss, stats = NB.run_distill_loss(x, t, index, teacher_lse=lse)
    dx = NB.distill_loss_backward(grad, x, t, index, stats)
    assert not loss[1::3].any() and not stats[1::3, 2].any() and not dx[1::3].any()
    for first in (0, 2):
        assert torch.equal(loss[first::3], want[first::3]) and torch.equal(dx[first::3], dwant[first::3])


def test_tensors_of_a_subclass_give_what_plain_ones_give():
    import torch

    import neptune_opt_b200 as NB

    class Tagged(torch.Tensor):
        pass

    gen = torch.Generator(device="cuda").manual_seed(5)

    def normal(*shape, dtype=torch.bfloat16):
        return torch.randn(*shape, device="cuda", generator=gen).to(dtype)

    def plain(t):
        return t.as_subclass(torch.Tensor) if isinstance(t, torch.Tensor) else t

    q, k, g = normal(2, 4, 90, 128), normal(2, 2, 90, 128), normal(2, 4, 90, 128)
    x, r, gate, w, gy = normal(6, 9, 200), normal(6, 9, 200), normal(6, 1, 200), normal(200), normal(6, 9, 200)
    logits, teacher = normal(9, 3001), normal(9, 8)
    index = torch.randint(0, 3001, (9, 8), device="cuda", generator=gen)
    weight = torch.rand(9, device="cuda", generator=gen)

    def everything(kind):
        def leaf(t):
            return t.clone().as_subclass(kind).requires_grad_()

        q_, k_, x_, r_, gate_, w_, l_ = (leaf(t) for t in (q, k, x, r, gate, w, logits))
        o, lse = NB.attention(q_, k_, k_, causal=True, return_lse=True)
        y, h = NB.gated_residual_norm(x_, r_, gate_, post_weight=w_, pre_weight=w_, gate_act="tanh")
        loss = NB.distill_loss(l_, teacher.as_subclass(kind), index)
        torch.autograd.backward([o, y, h, loss], [t.as_subclass(kind) for t in (g, gy, gy, weight)])
        a = [t.as_subclass(kind) for t in (x, r, gate, w, logits, q, k, teacher)]
        with torch.no_grad():
            ys, hs, rstd = NB.run_gated_residual_norm(*a[:3], post_weight=a[3], pre_weight=a[3])
            ls, stats = NB.run_distill_loss(a[4], a[7], index)
            direct = (*NB.attention_backward(a[5], a[6], a[6], o, lse, g, causal=True),
                      *NB.gated_residual_norm_backward(gy, None, *a[:3], rstd, post_weight=a[3], pre_weight=a[3]),
                      NB.distill_loss_backward(weight, a[4], a[7], index, stats))
        return [plain(t) for t in (o, lse, y, h, loss, q_.grad, k_.grad, x_.grad, r_.grad, gate_.grad, w_.grad, l_.grad,
                                   ys, hs, rstd, ls, stats, *direct)]

    want, got = everything(torch.Tensor), everything(Tagged)
    assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("frozen", ["gate", "post", "pre", "gate post pre"])
@pytest.mark.parametrize("gate", ["channel", "sequence", "full"])
def test_frozen_weights_leave_the_other_gradients_what_they_are(gate, frozen):
    import torch

    import neptune_opt_b200 as NB
    from test_block_norm_gpu import _make

    s = _make((5, 70, 384), "bfloat16", gate, 8)
    names = ("x", "residual", "gate", "post", "pre")

    def grads(frozen):
        leaves = {n: s[n].clone().requires_grad_(n not in frozen) for n in names}
        y, h = NB.gated_residual_norm(leaves["x"], leaves["residual"], leaves["gate"], post_weight=leaves["post"],
                                      pre_weight=leaves["pre"], gate_act="tanh")
        torch.cuda.synchronize()
        before = NB.launch_count()
        torch.autograd.backward([y, h], [s["gy"], s["gh"]])
        return {n: leaf.grad for n, leaf in leaves.items()}, NB.launch_count() - before

    want, launches = grads(())
    got, fewer = grads(frozen.split())
    for n in names:
        assert got[n] is None if n in frozen.split() else torch.equal(got[n], want[n]), n
    assert launches == 2 and fewer == (1 if len(frozen.split()) == 3 else 2)
