"""Host-side contracts of the serving operators (no GPU): exception types before any launch, shapes from meta
tensors, and the C entry points' refusals (none of these calls reaches a CUDA API)."""
from __future__ import annotations

import ctypes

import pytest
import torch

import neptune_opt_b200 as NB
import neptune_opt_b200._lib as L

I32, I64, F32 = torch.int32, torch.int64, torch.float32


def _meta(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="meta")


# ------------------------------------------------------------------ prefix_attention
def _attention(**changes):
    a = {"q": _meta(3, 8, 2, 128), "pk": _meta(2, 100, 128), "pv": _meta(2, 100, 128), "k": _meta(3, 2, 50, 128),
         "v": _meta(3, 2, 50, 128), "lens": _meta(3, dtype=I32), "scale": None, **changes}
    return NB.prefix_attention(a["q"], a["pk"], a["pv"], a["k"], a["v"], a["lens"], scale=a["scale"], return_lse=True)


def test_prefix_attention_shapes():
    o, lse = _attention()
    assert o.shape == (3, 8, 2, 128) and o.dtype == torch.bfloat16 and lse.shape == (3, 8, 2) and lse.dtype == F32
    q, pk, k = _meta(1, 4, 1, 64, dtype=torch.float16), _meta(4, 0, 64, dtype=torch.float16), _meta(1, 4, 0, 64, dtype=torch.float16)
    assert NB.prefix_attention(q, pk, pk, k, k).shape == q.shape
    empty = _meta(0, 4, 1, 64), _meta(4, 9, 64), _meta(4, 9, 64), _meta(0, 4, 5, 64), _meta(0, 4, 5, 64)
    assert NB.prefix_attention(*empty).shape == (0, 4, 1, 64)


@pytest.mark.parametrize("bad", [
    {"pv": _meta(2, 99, 128)}, {"v": _meta(3, 2, 49, 128)}, {"pk": _meta(4, 100, 128), "pv": _meta(4, 100, 128)},
    {"k": _meta(2, 2, 50, 128), "v": _meta(2, 2, 50, 128)}, {"q": _meta(3, 8, 2, 64)}, {"q": _meta(3, 7, 2, 128)},
    {"q": _meta(8, 2, 128)}, {"pk": _meta(1, 2, 100, 128)}, {"lens": _meta(2, dtype=I32)},
    {"lens": _meta(6, dtype=I32)[::2]}, {"scale": 0.0}, {"scale": -1.0}, {"scale": float("nan")},
    {"scale": float("inf")}, {"pk": torch.zeros(2, 100, 128, dtype=torch.bfloat16)}])
def test_prefix_attention_refuses_shapes_and_scales(bad):
    with pytest.raises(ValueError):
        _attention(**bad)


@pytest.mark.parametrize("bad", [
    {"q": _meta(3, 8, 2, 128, dtype=F32)}, {"k": _meta(3, 2, 50, 128, dtype=torch.float16)}, {"pk": None},
    {"lens": _meta(3, dtype=I64)}, {"lens": [50, 50, 50]}, {"q": None}])
def test_prefix_attention_refuses_types(bad):
    with pytest.raises(TypeError):
        _attention(**bad)


def test_prefix_attention_refuses_head_dims_and_the_cpu():
    t = [_meta(1, 2, 1, 96), _meta(2, 4, 96), _meta(2, 4, 96), _meta(1, 2, 4, 96), _meta(1, 2, 4, 96)]
    with pytest.raises(NotImplementedError):
        NB.prefix_attention(*t)
    with pytest.raises(ValueError):
        NB.prefix_attention(*[torch.zeros(s.shape, dtype=s.dtype) for s in t])


# ------------------------------------------------------------------ quantized_rms_norm
@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.float8_e5m2, torch.int8])
def test_quantized_norm_shapes(dtype):
    x, w = _meta(2, 5, 256), _meta(256)
    q, scale, y = NB.quantized_rms_norm(x, w, x, dtype=dtype)
    assert q.shape == x.shape and q.dtype == dtype and scale.shape == (2, 5, 1) and scale.dtype == F32
    assert y.shape == x.shape and y.dtype == x.dtype
    q, scale, y = NB.quantized_rms_norm(x, w, group=64, dtype=dtype)
    assert scale.shape == (2, 5, 4) and y is None
    q, scale, y = NB.quantized_rms_norm(_meta(0, 256), w, _meta(0, 256))
    assert q.shape == (0, 256) and q.dtype == torch.float8_e4m3fn and scale.shape == (0, 1) and y.shape == (0, 256)


def test_quantized_norm_refuses():
    x, w = _meta(4, 96), _meta(96)
    for bad in ({"weight": _meta(95)}, {"weight": _meta(1, 96)}, {"residual": _meta(3, 96)}, {"group": 64}, {"group": 24},
                {"group": 0}, {"group": -32}, {"group": 256}, {"eps": 0.0}, {"eps": -1.0}, {"eps": float("nan")},
                {"eps": 1e-50}, {"eps": 1e60}):
        a = {"weight": w, "residual": x, **bad}
        with pytest.raises(ValueError):
            NB.quantized_rms_norm(x, a.pop("weight"), a.pop("residual"), **a)
    for bad in ({"weight": w.float()}, {"residual": x.float()}, {"dtype": torch.float16}, {"dtype": torch.uint8},
                {"weight": None}):
        a = {"weight": w, "residual": x, **bad}
        with pytest.raises(TypeError):
            NB.quantized_rms_norm(x, a.pop("weight"), a.pop("residual"), **a)
    with pytest.raises(TypeError):
        NB.quantized_rms_norm(x.double(), w.double())
    with pytest.raises(NotImplementedError):
        NB.quantized_rms_norm(_meta(1, 16385), _meta(16385))
    with pytest.raises(ValueError):
        NB.quantized_rms_norm(torch.zeros(2, 8), torch.zeros(8))
    with pytest.raises(ValueError):
        NB.quantized_rms_norm(_meta(2, 0), _meta(0))


# ------------------------------------------------------------------ penalize_logits
def _logits(**changes):
    a = {"logits": _meta(4, 100), "tokens": _meta(4, 7, dtype=I64), "token_lens": _meta(4, dtype=I32),
         "prompt_lens": _meta(4, dtype=I32), "repetition": _meta(4, dtype=F32), "presence": _meta(4, dtype=F32),
         "frequency": _meta(4, dtype=F32), "bias_index": _meta(4, 3, dtype=I32), "bias_value": _meta(4, 3, dtype=F32),
         "allowed": _meta(4, 4, dtype=I32), "temperature": _meta(4, dtype=F32), **changes}
    return NB.penalize_logits(a.pop("logits"), a.pop("tokens"), a.pop("token_lens"), a.pop("prompt_lens"), **a)


def test_logits_shapes():
    out = _logits()
    assert out.shape == (4, 100) and out.dtype == torch.bfloat16
    assert NB.penalize_logits(_meta(4, 100, dtype=F32)).dtype == F32
    assert NB.penalize_logits(_meta(0, 100), allowed=_meta(0, 4, dtype=I32)).shape == (0, 100)


@pytest.mark.parametrize("bad", [
    {"logits": _meta(100)}, {"logits": _meta(4, 0)}, {"tokens": _meta(3, 7, dtype=I64)}, {"tokens": _meta(7, dtype=I64)},
    {"token_lens": _meta(3, dtype=I32)}, {"prompt_lens": _meta(4, 1, dtype=I32)}, {"repetition": _meta(3, dtype=F32)},
    {"temperature": _meta(1, dtype=F32)}, {"bias_value": None}, {"bias_index": None}, {"bias_value": _meta(4, 2, dtype=F32)},
    {"allowed": _meta(4, 3, dtype=I32)}, {"allowed": _meta(4, 5, dtype=I32)}, {"tokens": None},
    {"allowed": torch.zeros(4, 4, dtype=I32)}])
def test_logits_refuses_shapes(bad):
    with pytest.raises(ValueError):
        _logits(**bad)


@pytest.mark.parametrize("bad", [
    {"logits": _meta(4, 100, dtype=torch.float64)}, {"tokens": _meta(4, 7, dtype=F32)}, {"token_lens": _meta(4, dtype=I64)},
    {"repetition": _meta(4)}, {"repetition": 1.2}, {"presence": _meta(4, dtype=torch.float64)},
    {"bias_index": _meta(4, 3, dtype=torch.int16)}, {"bias_value": _meta(4, 3)}, {"allowed": _meta(4, 4, dtype=torch.bool)},
    {"temperature": 1.0}])
def test_logits_refuses_types(bad):
    with pytest.raises(TypeError):
        _logits(**bad)


def test_logits_refuses_too_many_biases_and_the_cpu():
    with pytest.raises(NotImplementedError):
        _logits(bias_index=_meta(4, 1025, dtype=I32), bias_value=_meta(4, 1025, dtype=F32))
    with pytest.raises(ValueError):
        NB.penalize_logits(torch.zeros(2, 8))


# ------------------------------------------------------------------ what all of them refuse
def _calls():
    q, pk, k = _meta(1, 2, 1, 64), _meta(2, 4, 64), _meta(1, 2, 4, 64)
    x, w, z = _meta(4, 64), _meta(64), _meta(4, 100)
    return [(q, lambda d: NB.prefix_attention(d, pk, pk, k, k)), (pk, lambda d: NB.prefix_attention(q, pk, d, k, k)),
            (k, lambda d: NB.prefix_attention(q, pk, pk, d, k)), (x, lambda d: NB.quantized_rms_norm(d, w)),
            (x, lambda d: NB.quantized_rms_norm(x, w, d)), (w, lambda d: NB.quantized_rms_norm(x, d)),
            (z, lambda d: NB.penalize_logits(d))]


@pytest.mark.parametrize("which", range(7))
def test_gradients_are_refused(which):
    t, call = _calls()[which]
    leaf = t.clone().requires_grad_()
    with pytest.raises((NotImplementedError, RuntimeError), match="no gradient"):
        call(leaf)
    with torch.no_grad():
        call(leaf)
    call(t)


@pytest.mark.parametrize("which", range(7))
def test_forward_mode_is_refused(which):
    import torch.autograd.forward_ad as forward

    t, call = _calls()[which]
    with forward.dual_level(), pytest.raises((NotImplementedError, RuntimeError)):
        call(forward.make_dual(t, torch.ones_like(t)))


def test_traced_graphs_hold_the_ops():
    from torch.fx.experimental.proxy_tensor import make_fx

    def step(q, pk, k, x, w, z):
        return NB.prefix_attention(q, pk, pk, k, k), NB.quantized_rms_norm(x, w, x, group=32), NB.penalize_logits(z)

    names = {str(n.target) for n in make_fx(step)(_meta(1, 2, 1, 64), _meta(2, 4, 64), _meta(1, 2, 4, 64), _meta(4, 64),
                                                  _meta(64), _meta(4, 100)).graph.nodes}
    assert {"nb200.prefix_attention.default", "nb200.norm8.default", "nb200.penalize_logits.default"} <= names


def test_exported_with_dynamic_sizes():
    class Step(torch.nn.Module):
        def forward(self, q, pk, k, x, w, z):
            q8, scale, y = NB.quantized_rms_norm(x, w, x)
            return NB.prefix_attention(q, pk, pk, k, k), q8, scale, y, NB.penalize_logits(z)

    batch, own = torch.export.Dim("batch", min=2, max=64), torch.export.Dim("own", min=2, max=4096)
    args = (_meta(3, 4, 1, 128), _meta(2, 9, 128), _meta(3, 2, 17, 128), _meta(3, 64), _meta(64), _meta(3, 100))
    ep = torch.export.export(Step(), args, dynamic_shapes=({0: batch}, None, {0: batch, 2: own}, {0: batch}, None, {0: batch}),
                             strict=False)
    assert "nb200.prefix_attention" in str(ep.graph)


# ------------------------------------------------------------------ C entry points
FAKE, NULL, ODD = ctypes.c_void_p(1 << 20), ctypes.c_void_p(0), ctypes.c_void_p((1 << 20) + 2)


def _c_attention(strides=None, batch=2, heads=8, kv=2, tokens=1, dim=128, prefix=16, cache=16, dtype=1, scale=0.1, q=FAKE,
                 pk=FAKE, k=FAKE, lse=FAKE, work=FAKE, nbytes=1 << 40):
    s = L.NB200AttnStrides(8 * 16 * 128, 16 * 128, 128)
    a = L.NB200PrefixAttnArgs(batch, heads, kv, tokens, dim, prefix, cache, None, dtype, scale)
    st = (L.NB200AttnStrides * 5)(*(strides or [s] * 5))
    return L.load().nb200_prefix_attention(ctypes.byref(a), st, q, pk, FAKE, k, FAKE, FAKE, lse, work, nbytes, NULL)


def test_c_prefix_attention_refuses_before_any_launch():
    for empty in ({"batch": 0}, {"heads": 0}, {"tokens": 0}):
        assert _c_attention(**empty, q=NULL, work=NULL) == L.NB200_OK
    for bad in ({"kv": 3}, {"kv": 0}, {"dtype": 0}, {"dtype": 7}, {"scale": 0.0}, {"scale": float("nan")}, {"batch": -1},
                {"prefix": -1}, {"cache": -1}, {"tokens": -1}, {"q": NULL}, {"q": ODD}, {"pk": NULL}, {"k": ODD}, {"lse": ODD},
                {"work": ODD}, {"work": NULL}, {"nbytes": 8}, {"nbytes": 4096, "prefix": 4000}):
        assert _c_attention(**bad) == L.NB200_ERR_ARG, bad
    assert _c_attention(dim=96) == L.NB200_ERR_UNSUPPORTED and _c_attention(dim=0) == L.NB200_ERR_UNSUPPORTED
    for big in ({"prefix": (1 << 30) + 1}, {"cache": (1 << 30) + 1}, {"tokens": 1 << 28}, {"batch": 1 << 28},
                {"batch": 1 << 15, "cache": 1 << 20}, {"batch": 1 << 13, "cache": 1 << 20, "heads": 4096, "kv": 4096}):
        assert _c_attention(**big) == L.NB200_ERR_CAPACITY, big
    s = L.NB200AttnStrides(8 * 16 * 128, 16 * 128, 128)
    for bad in (L.NB200AttnStrides(16384, 2049, 128), L.NB200AttnStrides(16384, 0, 128), L.NB200AttnStrides(16384, 1 << 39, 128)):
        for i in range(5):
            assert _c_attention([s] * i + [bad] + [s] * (4 - i)) == L.NB200_ERR_ARG and "strides" in L.last_error()
    lib = L.load()
    for empty in ({"batch": 0, "heads": 8, "kv": 2}, {"batch": 2, "heads": 0, "kv": 0}):
        a = L.NB200PrefixAttnArgs(empty["batch"], empty["heads"], empty["kv"], 1, 128, 16, 16, None, 1, 0.1)
        assert lib.nb200_prefix_attention_work_bytes(ctypes.byref(a)) == 0
    assert lib.nb200_prefix_attention_work_bytes(None) == L.NB200_ERR_ARG


def test_c_norm8_refuses_before_any_launch():
    lib = L.load()

    def call(rows=4, width=64, group=0, dtype=1, kind=0, eps=1e-6, x=1 << 20, w=1 << 20, r=None, q=FAKE, scale=FAKE, y=NULL,
             stride=64):
        a = L.NB200Norm8Args(x, r, w, rows, width, group, stride, stride, dtype, kind, eps)
        return lib.nb200_norm8(ctypes.byref(a), q, scale, y, NULL)

    assert call(rows=0, x=None, q=NULL) == L.NB200_OK
    for bad in ({"rows": -1}, {"width": 0}, {"group": 8}, {"group": 128}, {"group": -16}, {"group": 16, "width": 40},
                {"dtype": 3}, {"kind": 3}, {"kind": -1}, {"eps": 0.0}, {"eps": float("inf")}, {"eps": 1e-60}, {"x": None},
                {"w": None}, {"q": NULL}, {"scale": NULL}, {"r": 1 << 20}, {"stride": -64}):
        assert call(**bad) == L.NB200_ERR_ARG, bad
    assert call(width=16385) == L.NB200_ERR_CAPACITY
    assert lib.nb200_norm8(None, FAKE, FAKE, NULL, NULL) == L.NB200_ERR_ARG


def test_c_logits_refuses_before_any_launch():
    lib = L.load()

    def call(rows=4, vocab=100, history=0, biases=0, dtype=1, tdt=1, bdt=1, logits=1 << 20, tokens=None, bi=None, bv=None,
             out=FAKE, stride=100, work=FAKE, nbytes=1 << 30):
        a = L.NB200LogitsArgs(logits, tokens, bi, bv, None, None, None, None, None, None, None, rows, vocab, history, biases,
                              stride, 0, 0, 0, 0, dtype, tdt, bdt)
        return lib.nb200_penalize_logits(ctypes.byref(a), out, work, nbytes, NULL)

    assert call(rows=0, logits=None) == L.NB200_OK
    for bad in ({"rows": -1}, {"vocab": 0}, {"history": -1}, {"biases": -1}, {"dtype": 4}, {"history": 5}, {"biases": 5},
                {"history": 5, "tokens": 1 << 20, "tdt": 2}, {"biases": 5, "bi": 1 << 20}, {"logits": None}, {"out": NULL},
                {"biases": 5, "bi": 1 << 20, "bv": 1 << 20, "bdt": 9}, {"stride": -100},
                {"history": 5000, "tokens": 1 << 20, "work": NULL}, {"history": 5000, "tokens": 1 << 20, "work": ODD},
                {"history": 5000, "tokens": 1 << 20, "nbytes": 64}):
        assert call(**bad) == L.NB200_ERR_ARG, bad
    assert call(biases=1025, bi=1 << 20, bv=1 << 20) == L.NB200_ERR_CAPACITY
    assert call(vocab=(1 << 30) + 1) == L.NB200_ERR_CAPACITY
    assert call(history=1 << 29) == L.NB200_ERR_CAPACITY
    assert lib.nb200_penalize_logits(None, FAKE, FAKE, 1 << 30, NULL) == L.NB200_ERR_ARG
    assert lib.nb200_penalize_logits_work_bytes(None) == L.NB200_ERR_ARG


def test_c_entries_refuse_tensors_off_their_elements():
    lib = L.load()
    base = 1 << 20

    def norm(dtype, x=base, w=base, r=base, scale=base, y=base):
        a = L.NB200Norm8Args(x, r, w, 4, 64, 0, 64, 64, dtype, 0, 1e-6)
        return lib.nb200_norm8(ctypes.byref(a), FAKE, ctypes.c_void_p(scale), ctypes.c_void_p(y), NULL)

    for dtype, off in ((0, 2), (1, 1), (2, 1)):
        for name in ("x", "w", "r", "y"):
            assert norm(dtype, **{name: base + off}) == L.NB200_ERR_ARG, (dtype, name)
    assert norm(1, scale=base + 2) == L.NB200_ERR_ARG

    pointers = ("logits", "tokens", "bias_index", "bias_value", "token_lens", "prompt_lens", "allowed", "repetition",
                "presence", "frequency", "temperature")

    def logits(dtype=0, index=1, out=1 << 28, history=8, work=FAKE, nbytes=1 << 30, **changes):
        a = L.NB200LogitsArgs(*(changes.get(name, base) for name in pointers), 4, 100, history, 8, 100, 8, 8, 8, 4, dtype, index,
                              index)
        return lib.nb200_penalize_logits(ctypes.byref(a), ctypes.c_void_p(out), work, nbytes, NULL)

    for name in pointers:
        assert logits(**{name: base + 2}) == L.NB200_ERR_ARG, name
    for name in ("tokens", "bias_index"):
        assert logits(**{name: base + 4}) == L.NB200_ERR_ARG, name
    assert logits(out=(1 << 28) + 2) == L.NB200_ERR_ARG
    for out in (base, base + 4 * 399, base - 4 * 399):  # in place, or over an end of the input
        assert logits(out=out) == L.NB200_ERR_ARG
    assert logits(dtype=1, logits=base + 1) == L.NB200_ERR_ARG and logits(dtype=2, out=(1 << 28) + 1) == L.NB200_ERR_ARG
    for bad in ({"work": NULL}, {"work": ODD}, {"nbytes": 64}):
        assert logits(history=5000, **bad) == L.NB200_ERR_ARG, bad
