"""Training operators at the edges of their contracts, without a GPU."""
from __future__ import annotations

import ctypes

import pytest

import neptune_opt_b200._lib as L


@pytest.mark.parametrize("batch,heads,kv,seq", [(0, 8, 2, 16), (2, 0, 0, 16), (2, 8, 2, 0), (0, 0, 0, 0), (2, 0, 3, 16)])
def test_attention_backward_needs_no_work_memory_for_an_empty_call(batch, heads, kv, seq):
    a = L.NB200AttnArgs(batch, heads, kv, seq, 128, None, 0, 0.1)
    lib = L.load()
    assert lib.nb200_attention_bwd_work_bytes(ctypes.byref(a)) == 0
    s = (L.NB200AttnStrides * 8)()
    null = ctypes.c_void_p(0)
    assert lib.nb200_attention_bwd(ctypes.byref(a), s, *[null] * 10, 0, null) == L.NB200_OK


class _Reached(Exception):
    """An op of the library was dispatched."""


def _wrapper(*shape, dtype):
    """A tensor of a subclass of its own that says it is on a CUDA device; its ops go to the subclass."""
    import torch

    class Wrapper(torch.Tensor):
        @staticmethod
        def __new__(cls):
            return torch.Tensor._make_wrapper_subclass(cls, shape, dtype=dtype, device="cuda")

        @classmethod
        def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
            if func.namespace == "nb200":
                raise _Reached(func)
            raise NotImplementedError(func)

    return Wrapper()


def test_tensor_subclasses_reach_the_ops():
    """A CUDA tensor is one whatever its Python type: its results come from the library, or its type refuses."""
    import torch

    import neptune_opt_b200 as NB

    bf, f32 = torch.bfloat16, torch.float32
    q, lse = _wrapper(1, 2, 8, 128, dtype=bf), _wrapper(1, 2, 8, dtype=f32)
    x, w, rstd = _wrapper(4, 64, dtype=bf), _wrapper(64, dtype=bf), _wrapper(4, 2, dtype=f32)
    t, i = _wrapper(4, 8, dtype=bf), _wrapper(4, 8, dtype=torch.int64)
    loss, stats = _wrapper(4, dtype=f32), _wrapper(4, 3, dtype=f32)
    for call in (lambda: NB.attention_backward(q, q, q, q, lse, q),
                 lambda: NB.run_gated_residual_norm(x, x, pre_weight=w),
                 lambda: NB.gated_residual_norm(x, x, post_weight=w),
                 lambda: NB.gated_residual_norm_backward(x, None, x, x, None, rstd, post_weight=w),
                 lambda: NB.run_distill_loss(x, t, i), lambda: NB.distill_loss(x, t, i),
                 lambda: NB.distill_loss_backward(loss, x, t, i, stats)):
        with pytest.raises(_Reached):
            call()


def test_forward_mode_is_refused():
    """The operators have no tangents; a dual tensor is refused, not stripped of its own."""
    import torch
    import torch.autograd.forward_ad as forward

    import neptune_opt_b200 as NB

    def meta(*shape, dtype=torch.bfloat16):
        return torch.empty(*shape, dtype=dtype, device="meta")

    q, lse = meta(1, 2, 8, 128), meta(1, 2, 8, dtype=torch.float32)
    x, w, rstd, t, i = meta(4, 64), meta(64), meta(4, 2, dtype=torch.float32), meta(4, 8), meta(4, 8, dtype=torch.int64)
    row, stats = meta(4, dtype=torch.float32), meta(4, 3, dtype=torch.float32)
    calls = [(q, lambda d: NB.attention(d, q, q)), (q, lambda d: NB.attention(q, q, d)),
             (q, lambda d: NB.attention_backward(q, q, q, q, lse, d)),
             (x, lambda d: NB.gated_residual_norm(d, x, pre_weight=w)), (w, lambda d: NB.gated_residual_norm(x, x, d, pre_weight=w)),
             (x, lambda d: NB.run_gated_residual_norm(x, d, post_weight=w)),
             (x, lambda d: NB.gated_residual_norm_backward(d, None, x, x, None, rstd, post_weight=w)),
             (x, lambda d: NB.distill_loss(d, t, i)), (t, lambda d: NB.run_distill_loss(x, d, i)),
             (row, lambda d: NB.distill_loss_backward(d, x, t, i, stats))]
    for a, call in calls:
        call(a)
        for leaf in (a, a.clone().requires_grad_()):
            with forward.dual_level(), pytest.raises((NotImplementedError, RuntimeError)):
                call(forward.make_dual(leaf, torch.ones_like(a)))


def test_gradients_nobody_wants_are_not_made():
    """Frozen weights and a constant gate: the backward pass asks for no sums, and makes no tensor of them."""
    import torch

    import neptune_opt_b200 as NB
    from torch.fx.experimental.proxy_tensor import make_fx

    def step(x, gate, w, train):
        leaf = x.detach().requires_grad_()
        w = w.detach().requires_grad_(train)
        y, h = NB.gated_residual_norm(leaf, x, gate, post_weight=w, pre_weight=w.detach())
        return torch.autograd.grad(h.sum() + y.sum(), [leaf, w] if train else [leaf])

    x, w = torch.empty(4, 64, device="meta"), torch.empty(64, device="meta")
    for train in (False, True):
        graph = make_fx(lambda a, b, c: step(a, b, c, train))(x, x, w).graph
        node = next(n for n in graph.nodes if "gated_norm_bwd" in str(n.target))
        wanted = (list(node.args[10:]) + [True] * 3)[:3]
        assert wanted == [False, train, False]
        assert [tuple(v.shape) for v in node.meta["val"]] == [(4, 64), (4, 64), (0,), (64,) if train else (0,), (0,)]
