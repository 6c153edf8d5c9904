"""Fused attention on the sm_100a tensor cores, forward (nb200_attention_fwd) and backward
(nb200_attention_bwd).

O = softmax(scale * Q K^T [+ masks]) V per (batch, head) with bf16 Q, O of shape [B, H, S, D] and
K, V of shape [B, H_kv, S, D] (H a multiple of H_kv: query head h reads key/value head
h // (H // H_kv)), fp32 scores and an fp32 online max/sum repair (the exp(c - s) rescale of the
repaired fold applied to attention rows), and optionally the fp32 natural log-sum-exp of each query
row's scaled scores, [B, H, S]. `seq_lens` [B] gives the tokens of each batch element: queries and
keys past them are masked, their rows of O and of the gradients are zero and their log-sum-exp is
-inf, whatever the tensors hold there. Graphs traced through the functions (export, torch.compile) hold
the C++ ops; forward-mode differentiation is refused.

The reference has no attention kernel (its roadmap declares one out of scope); the contract here
follows torch.nn.functional.scaled_dot_product_attention with is_causal (key index <= query
index) and its default scale 1/sqrt(D). Errors follow the backend's convention: TypeError for
dtypes, ValueError for devices, shapes and scale, NotImplementedError for head dimensions the
kernel is not built for.
"""
from __future__ import annotations

import ctypes
import math

from neptune_opt_b200 import _lib
from neptune_opt_b200.template import _on_device, current_stream
from neptune_opt_b200.torch_op import cxx_op, distinct, run_cxx

HEAD_DIMS = (128,)
OP_NAME = "neptune_b200::attention"


def validate_attention_inputs(q, k, v, scale, seq_lens=None):
    import torch

    for name, t in (("q", q), ("k", k), ("v", v)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"attention: {name} must be a tensor")
        if t.dtype != torch.bfloat16:
            raise TypeError(f"attention: {name} must be bfloat16, got {t.dtype}")
        if t.dim() != 4:
            raise ValueError(f"attention: {name} must be [batch, heads, seq, head_dim], got {tuple(t.shape)}")
    if k.shape != v.shape or q.shape[0] != k.shape[0] or q.shape[2:] != k.shape[2:]:
        raise ValueError(f"attention: q, k, v shapes differ: {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if q.shape[1] != k.shape[1] and (k.shape[1] == 0 or q.shape[1] % k.shape[1]):
        raise ValueError(f"attention: {q.shape[1]} query heads cannot share {k.shape[1]} key/value heads")
    if q.device != k.device or q.device != v.device:
        raise ValueError("attention: q, k, v must be on one device")
    if q.device.type != "cuda" and q.device.type != "meta":
        raise ValueError(f"attention: inputs must be CUDA tensors, got {q.device}")
    d = q.shape[-1]
    if d not in HEAD_DIMS:
        raise NotImplementedError(f"attention: head_dim {d} is not supported (built for {HEAD_DIMS})")
    if seq_lens is not None:
        if not isinstance(seq_lens, torch.Tensor) or seq_lens.dtype != torch.int32:
            raise TypeError("attention: seq_lens must be an int32 tensor")
        if tuple(seq_lens.shape) != (q.shape[0],) or seq_lens.device != q.device or not seq_lens.is_contiguous():
            raise ValueError("attention: seq_lens must be a contiguous [batch] tensor on the device of q")
    s = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if not (math.isfinite(s) and s > 0.0):
        raise ValueError(f"attention: scale must be finite and positive, got {scale}")
    return s


def _scale(q, scale):
    """The scale of a call, 1/sqrt(D) by default; what q is remains to be checked."""
    return 1.0 / math.sqrt(max(q.shape[-1], 1)) if scale is None and getattr(q, "shape", ()) else scale


def _args(q, k, causal, scale, seq_lens):
    b, h, s, d = q.shape
    return _lib.NB200AttnArgs(b, h, k.shape[1], s, d, seq_lens.data_ptr() if seq_lens is not None else None,
                              1 if causal else 0, scale)


def _strides(*tensors):
    return (_lib.NB200AttnStrides * len(tensors))(*[t.stride()[:3] for t in tensors])


def launch_attention(q, k, v, o, lse, *, causal: bool, scale: float, seq_lens=None) -> None:
    """One nb200_attention_fwd call into given tensors on the current stream of q's device (strides as the C entry
    asks for them)."""
    lib = _lib.load()
    with _on_device(q.device):
        rc = lib.nb200_attention_fwd(ctypes.byref(_args(q, k, causal, scale, seq_lens)), _strides(q, k, v, o),
                                     q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
                                     lse.data_ptr() if lse is not None else None, current_stream(q.device))
    _lib.check(rc, "nb200_attention")


def _forward(q, k, v, causal, scale, seq_lens, with_lse):
    """(O, LSE or None). A graph traced through it holds the op."""
    o, lse = cxx_op("attention_fwd")(q, k, v, seq_lens, causal, scale, with_lse)
    return o, lse if with_lse else None


def run_attention(q, k, v, *, causal: bool = False, scale=None, return_lse: bool = False, seq_lens=None):
    """Fresh contiguous O (and LSE when asked). With gradients enabled and wanted, O carries them (LSE
    does not)."""
    import torch

    sc = validate_attention_inputs(q, k, v, scale, seq_lens)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        o, lse = _function().apply(*distinct(q, k, v), causal, sc, seq_lens)
    else:
        o, lse = _forward(q, k, v, causal, sc, seq_lens, return_lse)
    return (o, lse) if return_lse else o


def attention_backward(q, k, v, o, lse, grad_out, *, causal: bool = False, scale=None, seq_lens=None):
    """(dq, dk, dv) of `run_attention`'s O for the gradient grad_out of it, from the saved O and LSE.

    The probabilities are recomputed; dk and dv of a shared key/value head sum over its query heads.
    The result does not depend on scheduling. Gradients keep the memory layout of their inputs."""
    return run_cxx("attention_bwd", q, (q, k, v, o, lse, grad_out, seq_lens, causal, _scale(q, scale)),
                   _validate_backward, q, k, v, o, lse, grad_out, scale, seq_lens)


def _validate_backward(q, k, v, o, lse, grad_out, scale, seq_lens):
    import torch

    validate_attention_inputs(q, k, v, scale, seq_lens)
    for name, t in (("o", o), ("grad_out", grad_out)):
        if not isinstance(t, torch.Tensor) or t.dtype != torch.bfloat16:
            raise TypeError(f"attention_backward: {name} must be a bfloat16 tensor")
        if t.shape != q.shape or t.device != q.device:
            raise ValueError(f"attention_backward: {name} must have the shape and device of q")
    if not isinstance(lse, torch.Tensor) or lse.dtype != torch.float32:
        raise TypeError("attention_backward: lse must be a float32 tensor")
    if lse.shape != q.shape[:-1] or lse.device != q.device:
        raise ValueError("attention_backward: lse must be [batch, heads, seq] on the device of q")


_FUNCTION = None


def _function():
    global _FUNCTION
    if _FUNCTION is not None:
        return _FUNCTION
    import torch

    class Attention(torch.autograd.Function):
        @staticmethod
        def forward(ctx, q, k, v, causal, scale, seq_lens):
            o, lse = _forward(q, k, v, causal, scale, seq_lens, True)
            ctx.save_for_backward(q, k, v, o, lse, seq_lens)
            ctx.causal, ctx.scale = causal, scale
            ctx.mark_non_differentiable(lse)
            return o, lse

        @staticmethod
        @torch.autograd.function.once_differentiable
        def backward(ctx, grad_out, _):
            q, k, v, o, lse, seq_lens = ctx.saved_tensors
            grads = attention_backward(q, k, v, o, lse, grad_out, causal=ctx.causal, scale=ctx.scale,
                                       seq_lens=seq_lens)
            return (*grads, None, None, None)

    _FUNCTION = Attention
    return _FUNCTION


_OP = None


def attention_op():
    """Op `neptune_b200::attention(q, k, v, causal, scale) -> (O, LSE)`. Like the region ops, its one
    kernel is a composite body that checks the contract and calls the C++-registered
    `nb200::attention`, so a graph holding it exports, and AOTInductor packages it as a call of the
    C++ op."""
    global _OP
    if _OP is not None:
        return _OP
    from neptune_opt_b200.torch_op import _nb200, _register

    def _body(q, k, v, causal, scale):
        sc = validate_attention_inputs(q, k, v, scale)
        return tuple(_nb200().attention(q, k, v, causal, sc))

    _OP = _register(OP_NAME, "(Tensor q, Tensor k, Tensor v, bool causal, float scale) -> (Tensor, Tensor)", _body)
    return _OP
