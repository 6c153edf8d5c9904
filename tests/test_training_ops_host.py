"""Host-side contracts of the training operators (no GPU): exception types before any launch, shapes from
meta tensors, and the C entry points' refusals (none of these calls reaches a CUDA API)."""
from __future__ import annotations

import ctypes

import pytest
import torch

import neptune_opt_b200 as NB
import neptune_opt_b200._lib as L


def _meta(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="meta")


def test_attention_with_shared_heads_and_lengths():
    q, k = _meta(2, 8, 100, 128), _meta(2, 2, 100, 128)
    o, lse = NB.attention(q, k, k, return_lse=True, seq_lens=_meta(2, dtype=torch.int32))
    assert o.shape == q.shape and lse.shape == (2, 8, 100)
    grads = NB.attention_backward(q, k, k, o, lse, o)
    assert [t.shape for t in grads] == [q.shape, k.shape, k.shape]
    for bad in ({"k": _meta(2, 3, 100, 128)}, {"k": _meta(1, 2, 100, 128)}, {"k": _meta(2, 2, 99, 128)},
                {"seq_lens": _meta(3, dtype=torch.int32)}, {"scale": -1.0}, {"scale": float("nan")},
                {"lse": _meta(2, 8, 99, dtype=torch.float32)}, {"grad": _meta(2, 8, 99, 128)},
                {"seq_lens": _meta(4, dtype=torch.int32)[::2]}):
        args = {"k": k, "seq_lens": None, "scale": None, "lse": lse, "grad": o, **bad}
        with pytest.raises(ValueError):
            NB.attention_backward(q, args["k"], args["k"], o, args["lse"], args["grad"], scale=args["scale"],
                                  seq_lens=args["seq_lens"])
    for bad in ({"grad": o.float()}, {"lse": lse.double()}, {"seq_lens": _meta(2, dtype=torch.int64)}):
        args = {"seq_lens": None, "lse": lse, "grad": o, **bad}
        with pytest.raises(TypeError):
            NB.attention_backward(q, k, k, o, args["lse"], args["grad"], seq_lens=args["seq_lens"])
    with pytest.raises(NotImplementedError):
        NB.attention_backward(*[_meta(1, 1, 8, 64)] * 4, _meta(1, 1, 8, dtype=torch.float32), _meta(1, 1, 8, 64))


def test_gated_residual_norm_contract():
    x, w = _meta(2, 5, 64), _meta(64)
    y, h, rstd = NB.run_gated_residual_norm(x, x, _meta(2, 1, 64), post_weight=w, pre_weight=w)
    assert y.shape == h.shape == x.shape and rstd.shape == (2, 5, 2) and rstd.dtype == torch.float32
    assert NB.gated_residual_norm(x, x, post_weight=w)[1] is None
    grads = NB.gated_residual_norm_backward(y, None, x, x, w, rstd, post_weight=w)
    assert [None if g is None else tuple(g.shape) for g in grads] == [(2, 5, 64), (2, 5, 64), (64,), (64,), None]
    ok = {"residual": x, "gate": None, "post_weight": w, "pre_weight": w}
    for bad in ({"residual": _meta(2, 4, 64)}, {"post_weight": _meta(63)}, {"post_weight": None, "pre_weight": None},
                {"gate": _meta(5, 64)}, {"gate": _meta(1, 5, 64)}, {"gate": _meta(2, 5, 63)}, {"gate_act": "relu"},
                {"residual_scale": float("inf")}, {"eps": 0.0}, {"eps": float("nan")}):
        a = {**ok, **bad}
        with pytest.raises(ValueError):
            NB.run_gated_residual_norm(x, a.pop("residual"), a.pop("gate"), **a)
    with pytest.raises(TypeError):
        NB.gated_residual_norm(x, x.float(), post_weight=w)
    with pytest.raises(TypeError):
        NB.gated_residual_norm(x.double(), x.double(), post_weight=w.double())
    with pytest.raises(NotImplementedError):
        NB.gated_residual_norm(_meta(1, 16385), _meta(1, 16385), post_weight=_meta(16385))
    with pytest.raises(ValueError):
        NB.gated_residual_norm(*[torch.zeros(2, 8)] * 2, post_weight=torch.zeros(8))
    with pytest.raises(ValueError):
        NB.gated_residual_norm_backward(x, x, x, x, None, rstd, post_weight=w)
    with pytest.raises(TypeError):
        NB.gated_residual_norm_backward(x, x, x, x, None, rstd.double(), post_weight=w, pre_weight=w)
    with pytest.raises(ValueError):
        NB.gated_residual_norm_backward(x, x, x, x, None, rstd[:1], post_weight=w, pre_weight=w)


def test_distill_loss_contract():
    x, t, i = _meta(2, 3, 100), _meta(2, 3, 8), _meta(2, 3, 8, dtype=torch.int64)
    loss, stats = NB.run_distill_loss(x, t, i)
    assert loss.shape == (2, 3) and stats.shape == (2, 3, 3) and loss.dtype == torch.float32
    assert NB.distill_loss_backward(loss, x, t, i, stats).shape == x.shape
    with pytest.raises(TypeError):
        NB.distill_loss(x, t, i.float())
    with pytest.raises(TypeError):
        NB.distill_loss(x.double(), t, i)
    with pytest.raises(TypeError):
        NB.distill_loss(x, t, i, teacher_lse=_meta(2, 3))
    for bad in ((x, t[:, :2], i), (x, t, i[..., :7]), (x[0], t, i)):
        with pytest.raises(ValueError):
            NB.distill_loss(*bad)
    for temperature in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            NB.distill_loss(x, t, i, temperature=temperature)
    with pytest.raises(ValueError):
        NB.distill_loss(x, t, i, teacher_lse=loss[0])
    with pytest.raises(NotImplementedError):
        NB.distill_loss(x, _meta(2, 3, 257), _meta(2, 3, 257, dtype=torch.int32))
    with pytest.raises(ValueError):
        NB.distill_loss(torch.zeros(2, 9), torch.zeros(2, 1), torch.zeros(2, 1, dtype=torch.int64))
    with pytest.raises(TypeError):
        NB.distill_loss_backward(loss.double(), x, t, i, stats)
    with pytest.raises(ValueError):
        NB.distill_loss_backward(loss, x, t, i, stats[..., :2])


def test_c_entry_points_refuse_before_any_launch():
    lib, fake, null = L.load(), ctypes.c_void_p(1 << 20), ctypes.c_void_p(0)
    odd = ctypes.c_void_p((1 << 20) + 2)
    s = L.NB200AttnStrides(8 * 16 * 128, 16 * 128, 128)

    def attn(strides=None, seq=16, heads=8, kv=2, dim=128, scale=0.1, q=fake, lse=fake, work=fake, nbytes=1 << 20):
        a = L.NB200AttnArgs(2, heads, kv, seq, dim, None, 0, scale)
        st = (L.NB200AttnStrides * 8)(*(strides or [s] * 8))
        return lib.nb200_attention_bwd(ctypes.byref(a), st, q, fake, fake, fake, lse, fake, fake, fake, fake, work,
                                       nbytes, null)

    assert attn(seq=0) == L.NB200_OK
    assert attn(kv=3) == L.NB200_ERR_ARG and attn(kv=0) == L.NB200_ERR_ARG
    assert attn(dim=64) == L.NB200_ERR_UNSUPPORTED
    assert attn(scale=-0.5) == L.NB200_ERR_ARG and attn(scale=float("nan")) == L.NB200_ERR_ARG
    assert attn(seq=-1) == L.NB200_ERR_ARG and attn(seq=(1 << 30) + 1) == L.NB200_ERR_CAPACITY
    assert attn(q=null) == L.NB200_ERR_ARG and attn(q=odd) == L.NB200_ERR_ARG and attn(lse=null) == L.NB200_ERR_ARG
    assert attn(work=odd) == L.NB200_ERR_ARG and attn(nbytes=16) == L.NB200_ERR_ARG
    for bad in (L.NB200AttnStrides(0, 2048, 128), L.NB200AttnStrides(16384, 2049, 128),
                L.NB200AttnStrides(16384, 2048, -128), L.NB200AttnStrides(1 << 39, 2048, 128)):
        assert attn([s] * 5 + [bad] + [s] * 2) == L.NB200_ERR_ARG and "strides" in L.last_error()
    a = L.NB200AttnArgs(2, 8, 2, 16, 128, None, 0, 0.1)
    assert lib.nb200_attention_bwd_work_bytes(ctypes.byref(a)) >= 2 * 8 * 16 * 4

    def norm(rows=4, width=64, group=1, act=0, dtype=1, dgate=null, nbytes=1 << 20, gate=None, eps=1e-6):
        a = L.NB200NormArgs(1 << 20, 1 << 20, gate, 1 << 20, None, rows, width, width, width, width, width, width,
                            group, act, 1.0, eps)
        return lib.nb200_gated_norm_bwd(ctypes.byref(a), dtype, fake, fake, null, fake, fake, dgate, null, null, fake,
                                        nbytes, null)

    assert norm(rows=0) == L.NB200_OK
    assert norm(width=0) == L.NB200_ERR_ARG and norm(rows=-1) == L.NB200_ERR_ARG and norm(dtype=9) == L.NB200_ERR_ARG
    assert norm(gate=1 << 20, group=3) == L.NB200_ERR_ARG and norm(act=3) == L.NB200_ERR_ARG
    assert norm(dgate=fake) == L.NB200_ERR_ARG and "absent" in L.last_error()
    assert norm(nbytes=8) == L.NB200_ERR_ARG
    assert norm(width=20000, nbytes=1 << 40) == L.NB200_ERR_CAPACITY

    def distill(rows=2, vocab=100, top=8, dtype=1, index=1, temperature=1.0, x=1 << 20):
        a = L.NB200DistillArgs(x, 1 << 20, 1 << 20, rows, vocab, top, vocab, top, top, dtype, 0, index, temperature)
        return lib.nb200_distill_loss(ctypes.byref(a), null, fake, fake, null)

    assert distill(rows=0) == L.NB200_OK and distill(vocab=0) == L.NB200_ERR_ARG and distill(top=-1) == L.NB200_ERR_ARG
    assert distill(dtype=5) == L.NB200_ERR_ARG and distill(index=2) == L.NB200_ERR_ARG
    assert distill(temperature=0.0) == L.NB200_ERR_ARG and distill(x=None) == L.NB200_ERR_ARG
    assert distill(top=257) == L.NB200_ERR_CAPACITY
