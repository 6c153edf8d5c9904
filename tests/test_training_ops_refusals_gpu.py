"""The training operators refuse bad CUDA arguments with the backend's exception types, before any launch."""
from __future__ import annotations

import pytest

from conftest import cuda_available

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_available(), reason="needs a CUDA device")]


def _z(*shape, dtype="bfloat16"):
    import torch

    return torch.zeros(*shape, dtype=getattr(torch, dtype), device="cuda")


def _raises(error, call, *args, **kw):
    import neptune_opt_b200 as NB

    before = NB.launch_count()
    with pytest.raises(error):
        call(*args, **kw)
    assert NB.launch_count() == before


def test_attention_backward():
    import neptune_opt_b200 as NB

    q, k, lse = _z(2, 4, 9, 128), _z(2, 2, 9, 128), _z(2, 4, 9, dtype="float32")
    f = NB.attention_backward
    good = dict(q=q, k=k, v=k, o=q, lse=lse, grad_out=q)
    for error, bad in ((ValueError, {"k": _z(2, 3, 9, 128), "v": _z(2, 3, 9, 128)}), (ValueError, {"v": _z(2, 2, 8, 128)}),
                       (TypeError, {"q": q.float()}), (TypeError, {"grad_out": q.half()}), (ValueError, {"o": q[:, :2]}),
                       (TypeError, {"lse": lse.double()}), (ValueError, {"lse": lse[:, :, :8]}), (ValueError, {"k": k.cpu()}),
                       (ValueError, {"lse": lse.cpu()}), (ValueError, {"scale": 0.0}), (ValueError, {"scale": float("inf")}),
                       (TypeError, {"seq_lens": _z(2, dtype="int64")}), (ValueError, {"seq_lens": _z(3, dtype="int32")}),
                       (ValueError, {"seq_lens": _z(2, dtype="int32").cpu()}), (TypeError, {"o": None})):
        a = {**good, **bad}
        _raises(error, f, a.pop("q"), a.pop("k"), a.pop("v"), a.pop("o"), a.pop("lse"), a.pop("grad_out"), **a)
    small = _z(1, 1, 4, 64)
    _raises(NotImplementedError, f, small, small, small, small, _z(1, 1, 4, dtype="float32"), small)


def test_gated_residual_norm():
    import torch

    import neptune_opt_b200 as NB

    x, w, r = _z(2, 5, 64), _z(64), _z(2, 5, 2, dtype="float32")
    good = dict(x=x, residual=x, gate=None, post_weight=w, pre_weight=w)
    cases = ((ValueError, {"residual": _z(5, 2, 64)}), (ValueError, {"residual": _z(2, 5, 63)}), (TypeError, {"residual": x.half()}),
             (ValueError, {"post_weight": _z(63)}), (TypeError, {"pre_weight": w.float()}), (ValueError, {"pre_weight": w.cpu()}),
             (ValueError, {"post_weight": None, "pre_weight": None}), (ValueError, {"gate": _z(5, 64)}),
             (ValueError, {"gate": _z(1, 5, 64)}), (ValueError, {"gate": _z(2, 5, 1)}), (ValueError, {"gate_act": "relu"}),
             (ValueError, {"residual_scale": float("nan")}), (TypeError, {"x": x.to(torch.float64)}))
    for error, bad in cases + ((ValueError, {"eps": 0.0}), (ValueError, {"eps": float("inf")})):
        a = {**good, **bad}
        _raises(error, NB.run_gated_residual_norm, a.pop("x"), a.pop("residual"), a.pop("gate"), **a)
    good.update(grad_y=x, grad_h=x, rstd=r)
    for error, bad in cases + ((ValueError, {"grad_y": x[:1]}), (TypeError, {"grad_h": x.float()}), (TypeError, {"rstd": r.double()}),
                               (ValueError, {"rstd": r[..., :1]}), (ValueError, {"rstd": r.view(10, 2)}),
                               (ValueError, {"pre_weight": None})):
        a = {**good, **bad}
        _raises(error, NB.gated_residual_norm_backward, a.pop("grad_y"), a.pop("grad_h"), a.pop("x"), a.pop("residual"),
                a.pop("gate"), a.pop("rstd"), **a)
    wide = _z(1, 16385)
    _raises(NotImplementedError, NB.gated_residual_norm, wide, wide, post_weight=_z(16385))


def test_distill_loss():
    import neptune_opt_b200 as NB

    x, t, i, f = _z(2, 3, 50), _z(2, 3, 4), _z(2, 3, 4, dtype="int64"), _z(2, 3, dtype="float32")
    for error, args, kw in ((TypeError, (x.double(), t, i), {}), (TypeError, (x, t, i.float()), {}), (ValueError, (x, t[..., :3], i), {}),
                            (ValueError, (x.view(6, 50), t, i), {}), (ValueError, (x.view(3, 2, 50), t, i), {}), (ValueError, (x, t.cpu(), i), {}),
                            (ValueError, (x, t, i), {"temperature": 0.0}), (ValueError, (x, t, i), {"temperature": float("nan")}),
                            (TypeError, (x, t, i), {"teacher_lse": f.double()}), (ValueError, (x, t, i), {"teacher_lse": f[:1]}),
                            (NotImplementedError, (x, _z(2, 3, 257), _z(2, 3, 257, dtype="int32")), {}), (TypeError, (x, None, i), {})):
        _raises(error, NB.distill_loss, *args, **kw)
    s = _z(2, 3, 3, dtype="float32")
    for error, grad, stats in ((TypeError, f.double(), s), (ValueError, f.view(6), s), (ValueError, f, s[..., :2]), (TypeError, f, s.half()),
                               (ValueError, f.cpu(), s)):
        _raises(error, NB.distill_loss_backward, grad, x, t, i, stats)
