"""The training operators inside torch.export, torch.compile and AOTInductor packages give what eager calls give."""
from __future__ import annotations

import pytest

from conftest import cuda_available

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_available(), reason="needs a CUDA device")]


def _inputs():
    import torch

    gen = torch.Generator(device="cuda").manual_seed(2)

    def normal(*shape, dtype=torch.bfloat16):
        return torch.randn(*shape, device="cuda", generator=gen).to(dtype)

    return {"x": normal(4, 9, 200), "r": normal(4, 9, 200), "gate": normal(4, 1, 200), "w": normal(200),
            "logits": normal(9, 3001), "t": normal(9, 8), "row": torch.rand(9, device="cuda", generator=gen),
            "i": torch.randint(0, 3001, (9, 8), device="cuda", generator=gen),
            "lens": torch.tensor([90, 33], dtype=torch.int32, device="cuda"), "q": normal(2, 4, 90, 128), "k": normal(2, 2, 90, 128), "v": normal(2, 2, 90, 128), "g": normal(2, 4, 90, 128)}


def _modules():
    import torch

    import neptune_opt_b200 as NB

    class Norm(torch.nn.Module):
        names = ("x", "r", "gate", "w")

        def forward(self, x, r, gate, w):
            y, h = NB.gated_residual_norm(x, r, gate, post_weight=w, pre_weight=w, gate_act="tanh")
            return y, h, NB.gated_residual_norm(h, y, post_weight=w)[0]

    class NormBackward(torch.nn.Module):
        names = ("x", "r", "gate", "w")

        def forward(self, x, r, gate, w):
            y, h, rstd = NB.run_gated_residual_norm(x, r, gate, post_weight=w, pre_weight=w)
            return NB.gated_residual_norm_backward(y, h, x, r, gate, rstd, post_weight=w, pre_weight=w)

    class Loss(torch.nn.Module):
        names = ("logits", "t", "i", "row")

        def forward(self, logits, t, i, row):
            loss, stats = NB.run_distill_loss(logits, t, i, temperature=2.0)
            return loss, NB.distill_loss_backward(row, logits, t, i, stats, temperature=2.0)

    class Attention(torch.nn.Module):
        names = ("q", "k", "v", "g", "lens")

        def forward(self, q, k, v, g, lens):
            o, lse = NB.attention(q, k, v, causal=True, return_lse=True, seq_lens=lens)
            return o, lse, NB.attention(q, q, q), *NB.attention_backward(q, k, v, o, lse, g, causal=True, seq_lens=lens)

    return [Norm(), NormBackward(), Loss(), Attention()]


def _same(a, b):
    import torch

    a, b = ([t for t in (u if isinstance(u, (tuple, list)) else (u,))] for u in (a, b))
    assert len(a) == len(b) and all(torch.equal(x, y) and x.stride() == y.stride() for x, y in zip(a, b))


@pytest.mark.parametrize("which", [0, 1, 2, 3])
def test_exported_compiled_and_packaged(which, tmp_path):
    import torch

    import neptune_opt_b200.aot as A

    module, data = _modules()[which], _inputs()
    args = tuple(data[n] for n in module.names)
    want = module(*args)
    with torch.no_grad():
        for strict in (False, True):
            ep = torch.export.export(module, args, strict=strict)
            _same(ep.module()(*args), want)
        for backend in ("eager", "inductor"):
            _same(torch.compile(module, fullgraph=True, backend=backend)(*args), want)
        package = A.compile_package(ep, str(tmp_path / "ops.pt2"))
        _same(torch._inductor.aoti_load_package(package)(*args), want)


def test_compiled_training_step():
    """Gradients through torch.compile are those of the eager autograd functions, one weight for both norms too."""
    import torch

    import neptune_opt_b200 as NB

    data = _inputs()

    def step(x, r, gate, w, t, i):
        y, h = NB.gated_residual_norm(x, r, gate, post_weight=w, pre_weight=w, gate_act="sigmoid")
        return (NB.distill_loss(h, t, i).sum() + y.float().sum()) * 2.0

    t, i = data["x"][..., :8].contiguous(), data["x"][..., :8].argsort(-1)

    def run(f):
        leaves = [data[n].clone().requires_grad_() for n in ("x", "r", "gate", "w")]
        loss = f(*leaves, t, i)
        loss.backward()
        return [loss.detach(), *(leaf.grad for leaf in leaves)]

    want, got = run(step), run(torch.compile(step, backend="aot_eager"))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_compiled_attention_step():
    """One projection as key and value: its gradient is the sum of both."""
    import torch

    import neptune_opt_b200 as NB

    data = _inputs()

    def run(f):
        leaves = [data[n].clone().requires_grad_() for n in ("q", "k")]
        o = f(*leaves)
        o.backward(data["g"])
        return [o.detach(), *(leaf.grad for leaf in leaves)]

    def step(q, k):
        return NB.attention(q, k, k, causal=True, seq_lens=data["lens"])

    want = run(step)  # the first call makes the autograd function, which no graph holds
    for backend in ("eager", "aot_eager"):
        assert all(torch.equal(a, b) for a, b in zip(run(torch.compile(step, fullgraph=True, backend=backend)), want))
        torch._dynamo.reset()


@pytest.mark.parametrize("layout", ["dense", "packed"])
def test_attention_op_with_shared_heads(layout, tmp_path):
    """The op a graph holds takes shared heads and strided tensors, eager, exported and packaged."""
    import torch

    import neptune_opt_b200 as NB
    import neptune_opt_b200.aot as A

    data = _inputs()
    q, k, v = (data[n] for n in ("q", "k", "v"))
    if layout == "packed":
        q, k, v = torch.cat([q, k, v], 1).transpose(1, 2).contiguous().transpose(1, 2).split([4, 2, 2], 1)
    op = NB.attention_op()

    class Module(torch.nn.Module):
        def forward(self, q, k, v):
            return op(q, k, v, True, 0.1)

    want = NB.attention(q, k, v, causal=True, scale=0.1, return_lse=True)
    _same(op(q, k, v, True, 0.1), want)
    ep = torch.export.export(Module(), (q, k, v))
    _same(ep.module()(q, k, v), want)
    for shims in (True, False):
        package = A.compile_package(ep, str(tmp_path / f"attention{shims}.pt2"), shims=shims)
        _same(torch._inductor.aoti_load_package(package)(q, k, v), want)
