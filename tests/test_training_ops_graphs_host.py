"""Graphs traced through the training operators hold the library's ops (no GPU: fake CUDA tensors and meta tensors)."""
from __future__ import annotations

import pytest


def _fakes():
    import torch
    from torch._subclasses.fake_tensor import FakeTensorMode

    mode = FakeTensorMode()

    def empty(*shape, dtype=torch.bfloat16):
        with mode:
            return torch.empty(*shape, dtype=dtype, device="cuda")

    return mode, empty


def _ops(graph):
    """Names of what a graph calls, tuple access apart."""
    return [str(n.target) for n in graph.nodes if n.op == "call_function" and "getitem" not in str(n.target)]


def test_exported_graphs_hold_the_ops():
    import torch

    import neptune_opt_b200 as NB

    _, e = _fakes()
    x, w, gate, rstd = e(2, 5, 64), e(64), e(2, 1, 64), e(2, 5, 2, dtype=torch.float32)
    logits, t, i = e(3, 100), e(3, 8), e(3, 8, dtype=torch.int64)
    row, stats = e(3, dtype=torch.float32), e(3, 3, dtype=torch.float32)
    q, k, lse, lens = e(2, 4, 9, 128), e(2, 2, 9, 128), e(2, 4, 9, dtype=torch.float32), e(2, dtype=torch.int32)
    cases = [
        (lambda x, w: NB.gated_residual_norm(x, x, post_weight=w)[0], (x, w), "gated_norm", [x.shape]),
        (lambda x, w: NB.run_gated_residual_norm(x, x, pre_weight=w), (x, w), "gated_norm", [x.shape, x.shape, rstd.shape]),
        (lambda x, w, g, r: NB.gated_residual_norm_backward(x, None, x, x, g, r, post_weight=w)[:4], (x, w, gate, rstd),
         "gated_norm_bwd", [x.shape, x.shape, gate.shape, w.shape]),
        (lambda *a: NB.distill_loss(*a), (logits, t, i), "distill_loss", [row.shape]),
        (lambda *a: NB.run_distill_loss(*a), (logits, t, i), "distill_loss", [row.shape, stats.shape]),
        (lambda *a: NB.distill_loss_backward(*a), (row, logits, t, i, stats), "distill_loss_bwd", [logits.shape]),
        (lambda q, k, lse, n: NB.attention_backward(q, k, k, q, lse, q, seq_lens=n), (q, k, lse, lens), "attention_bwd",
         [q.shape, k.shape, k.shape]),
    ]
    for call, args, op, shapes in cases:
        class Module(torch.nn.Module):
            def forward(self, *a):
                return call(*a)

        ep = torch.export.export(Module(), args, strict=False)
        assert _ops(ep.graph) == [f"nb200.{op}.default"]
        outputs = [n.meta["val"] for n in next(n for n in ep.graph.nodes if n.op == "output").args[0]]
        assert [o.shape for o in outputs] == shapes and all(o.device.type == "cuda" for o in outputs)


def test_a_batch_size_stays_symbolic():
    import torch

    import neptune_opt_b200 as NB

    _, e = _fakes()

    class Loss(torch.nn.Module):
        def forward(self, logits, t, i):
            loss, stats = NB.run_distill_loss(logits, t, i)
            return loss, NB.distill_loss_backward(loss, logits, t, i, stats)

    class Norm(torch.nn.Module):
        def forward(self, x, w):
            return NB.gated_residual_norm(x, x, w, post_weight=w, pre_weight=w)

    rows = torch.export.Dim("rows", min=2, max=64)
    args = (e(3, 100), e(3, 8), e(3, 8, dtype=torch.int64))
    ep = torch.export.export(Loss(), args, strict=False, dynamic_shapes=[{0: rows}] * 3)
    assert _ops(ep.graph) == ["nb200.distill_loss.default", "nb200.distill_loss_bwd.default"]
    ep = torch.export.export(Norm(), (e(3, 64), e(64)), strict=False, dynamic_shapes=[{0: rows}, None])
    assert _ops(ep.graph) == ["nb200.gated_norm.default"]
    outs = [n.meta["val"] for n in next(n for n in ep.graph.nodes if n.op == "output").args[0]]
    assert all(isinstance(o.shape[0], torch.SymInt) for o in outs)


def test_a_traced_training_step_holds_both_directions():
    import torch

    import neptune_opt_b200 as NB
    from torch.fx.experimental.proxy_tensor import make_fx

    def step(x, w, t, i):
        leaves = [a.detach().requires_grad_() for a in (x, w)]
        _, h = NB.gated_residual_norm(leaves[0], x, post_weight=leaves[1], pre_weight=w)
        return torch.autograd.grad(NB.distill_loss(h, t, i).sum(), leaves)

    def meta(*shape, dtype=torch.bfloat16):
        return torch.empty(*shape, dtype=dtype, device="meta")

    graph = make_fx(step)(meta(3, 100), meta(100), meta(3, 8), meta(3, 8, dtype=torch.int64)).graph
    ours = [n for n in _ops(graph) if n.startswith("nb200.")]
    assert ours == ["nb200.gated_norm.default", "nb200.distill_loss.default", "nb200.distill_loss_bwd.default",
                    "nb200.gated_norm_bwd.default"]
    assert not any("empty" in n for n in _ops(graph))


def test_gradients_of_attention_have_the_layout_the_kernel_gives_them():
    import torch

    import neptune_opt_b200 as NB

    def meta(*shape, dtype=torch.bfloat16):
        return torch.empty(*shape, dtype=dtype, device="meta")

    packed = meta(2, 9, 8, 128).transpose(1, 2)  # [batch, seq, heads, 128] as a projection leaves it
    q, k, v = packed[:, :4], packed[:, 4:6], packed[:, 6:]
    lse = meta(2, 4, 9, dtype=torch.float32)
    dq, dk, dv = NB.attention_backward(q, k, v, q, lse, q)
    assert dq.stride() == (9 * 4 * 128, 128, 4 * 128, 1) and dk.stride() == dv.stride() == (9 * 2 * 128, 128, 2 * 128, 1)
    turned = meta(2, 2, 128, 9).transpose(2, 3)
    assert NB.attention_backward(q, turned, turned, q, lse, q)[1].is_contiguous()
    one = meta(1, 2, 9, 128).expand(2, 2, 9, 128)
    assert NB.attention_backward(q, one, one, q, lse, q)[2].is_contiguous()


def test_real_tensors_of_other_devices_are_still_refused():
    import torch

    import neptune_opt_b200 as NB

    x = torch.zeros(2, 8)
    with pytest.raises(ValueError):
        NB.run_gated_residual_norm(x, x, post_weight=torch.zeros(8))
    with pytest.raises(ValueError):
        NB.run_distill_loss(x, x, torch.zeros(2, 8, dtype=torch.int64))


def test_the_attention_op_sees_what_its_kernel_takes():
    """Shared key/value heads trace, and what no kernel takes is refused when it is traced, not when it runs."""
    import torch

    import neptune_opt_b200 as NB
    import neptune_opt_b200.aot as A

    A.load()

    def meta(*shape, dtype=torch.bfloat16):
        return torch.empty(*shape, dtype=dtype, device="meta")

    q, k = meta(2, 8, 30, 128), meta(2, 2, 30, 128)
    o, lse = NB.attention_op()(q, k, k, True, 0.1)
    assert o.shape == q.shape and lse.shape == (2, 8, 30)
    for bad in (meta(2, 3, 30, 128), meta(2, 2, 31, 128), meta(1, 2, 30, 128), meta(2, 30, 128), meta(2, 0, 30, 128)):
        with pytest.raises(ValueError):
            torch.ops.nb200.attention(q, bad, bad, True, 0.1)
    with pytest.raises(TypeError):
        torch.ops.nb200.attention(q, k.float(), k.float(), True, 0.1)


def test_attention_itself_exports():
    """With everything the function takes: shared heads, lengths, the log-sum-exp, a symbolic batch."""
    import torch

    import neptune_opt_b200 as NB

    _, e = _fakes()
    q, k, lens = e(2, 4, 9, 128), e(2, 2, 9, 128), e(2, dtype=torch.int32)

    class Plain(torch.nn.Module):
        def forward(self, q, k, lens):
            return NB.attention(q, k, k)

    class Whole(torch.nn.Module):
        def forward(self, q, k, lens):
            return NB.attention(q, k, k, causal=True, scale=0.2, return_lse=True, seq_lens=lens)

    batch = torch.export.Dim("batch", min=2, max=64)
    for module, shapes in ((Plain(), [q.shape]), (Whole(), [q.shape, (2, 4, 9)])):
        ep = torch.export.export(module, (q, k, lens), strict=False)
        assert _ops(ep.graph) == ["nb200.attention_fwd.default"]
        outputs = [n.meta["val"] for n in next(n for n in ep.graph.nodes if n.op == "output").args[0]]
        assert [tuple(o.shape) for o in outputs] == [tuple(s) for s in shapes]
        ep = torch.export.export(module, (q, k, lens), strict=False, dynamic_shapes=[{0: batch}] * 3)
        assert _ops(ep.graph) == ["nb200.attention_fwd.default"]
