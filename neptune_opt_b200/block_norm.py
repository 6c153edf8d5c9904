"""The norms around a transformer block, fused with the block's gate and residual scale
(nb200_gated_norm, nb200_gated_norm_bwd).

    z = post_weight * x * rsqrt(mean(x^2) + eps)          x is the block's output (z = x without the weight)
    y = residual + residual_scale * a(gate) * z           a: identity, tanh or sigmoid (1 without a gate)
    h = pre_weight * y * rsqrt(mean(y^2) + eps)           the next block's input (None without the weight)

One pass over x and residual, everything in fp32, each result rounded once (h from the unrounded y).
Gradients are those of that function; weight and shared-gate gradients are fp32 column sums added in
a fixed order, and autograd asks only for those that are wanted. The reference's RMSNorm
(neptune_codegen/emitters.py:549-627) is the inner norm alone, forward only, with its own rounding
stages: `rms_norm` keeps those.

x and residual are [..., width] in float32, bfloat16 or float16, gate and weights of the same dtype.
gate is [width], or has x's rank with leading dimensions equal to x's followed by ones (one gate row
per sequence, or per token). Errors follow the backend's convention: TypeError for dtypes, ValueError
for devices, shapes and parameters, NotImplementedError past the kernels' width.
"""
from __future__ import annotations

import math

from neptune_opt_b200.torch_op import distinct, run_cxx

GATE_ACTS = {"none": 0, "tanh": 1, "sigmoid": 2}
MAX_WIDTH = 16384


def _broadcasts(x, gate) -> bool:
    """Whether the gate is one row, or x's leading dimensions followed by ones."""
    if gate.dim() == 1:
        return True
    if gate.dim() != x.dim():
        return False
    n = 0
    while n < x.dim() - 1 and gate.shape[n] == x.shape[n]:
        n += 1
    return all(s == 1 for s in gate.shape[n:-1])


def validate_gated_norm_inputs(x, residual, gate, post_weight, pre_weight, gate_act, residual_scale, eps=1.0):
    """Metadata-only contract."""
    import torch

    what = "gated_residual_norm"
    for name, t in (("x", x), ("residual", residual), ("gate", gate), ("post_weight", post_weight),
                    ("pre_weight", pre_weight)):
        if t is None and name not in ("x", "residual"):
            continue
        if not isinstance(t, torch.Tensor) or t.layout != torch.strided:
            raise TypeError(f"{what}: {name} must be a strided tensor")
        if t.dtype not in (torch.float32, torch.bfloat16, torch.float16) or t.dtype != x.dtype:
            raise TypeError(f"{what}: {name} must share x's float32/bfloat16/float16 dtype, got {t.dtype}")
        if t.device != x.device:
            raise ValueError(f"{what}: {name} must be on the device of x")
    if x.device.type not in ("cuda", "meta"):
        raise ValueError(f"{what}: inputs must be CUDA tensors, got {x.device}")
    if x.dim() < 1 or x.shape[-1] < 1 or x.shape != residual.shape:
        raise ValueError(f"{what}: x {tuple(x.shape)} and residual {tuple(residual.shape)} must be one [..., width]")
    for name, t in (("post_weight", post_weight), ("pre_weight", pre_weight)):
        if t is not None and tuple(t.shape) != (x.shape[-1],):
            raise ValueError(f"{what}: {name} must be [{x.shape[-1]}], got {tuple(t.shape)}")
    if post_weight is None and pre_weight is None:
        raise ValueError(f"{what}: neither post_weight nor pre_weight is given")
    if gate is not None and (gate.dim() < 1 or gate.shape[-1] != x.shape[-1]):
        raise ValueError(f"{what}: gate must be [..., {x.shape[-1]}], got {tuple(gate.shape)}")
    if gate is not None and not _broadcasts(x, gate):
        raise ValueError(f"{what}: gate {tuple(gate.shape)} does not broadcast over the rows of {tuple(x.shape)}")
    if gate_act not in GATE_ACTS:
        raise ValueError(f"{what}: gate_act must be one of {sorted(GATE_ACTS)}, got {gate_act!r}")
    if not math.isfinite(residual_scale):
        raise ValueError(f"{what}: residual_scale must be finite")
    if not (math.isfinite(eps) and eps > 0):
        raise ValueError(f"{what}: eps must be finite and positive")
    if x.shape[-1] > MAX_WIDTH:
        raise NotImplementedError(f"{what}: width {x.shape[-1]} exceeds {MAX_WIDTH}")


def run_gated_residual_norm(x, residual, gate=None, *, post_weight=None, pre_weight=None, gate_act: str = "none",
                            residual_scale: float = 1.0, eps: float = 1e-6):
    """(y, h, rstd): fresh contiguous results in x's dtype (h is None without pre_weight) and the fp32
    reciprocal norms [..., 2] that the backward pass takes."""
    y, h, rstd = run_cxx("gated_norm", x, (x, residual, gate, post_weight, pre_weight, GATE_ACTS.get(gate_act, -1),
                                           residual_scale, eps), validate_gated_norm_inputs,
                         x, residual, gate, post_weight, pre_weight, gate_act, residual_scale, eps)
    return y, None if pre_weight is None else h, rstd


def gated_residual_norm_backward(grad_y, grad_h, x, residual, gate, rstd, *, post_weight=None, pre_weight=None,
                                 gate_act: str = "none", residual_scale: float = 1.0):
    """(dx, dresidual, dgate, dpost_weight, dpre_weight) for the gradients of y and h (either may be
    None); None in the place of an input that is absent. dgate sums over the rows that share a gate row."""
    return _backward((True, True, True), grad_y, grad_h, x, residual, gate, rstd, post_weight, pre_weight, gate_act,
                     residual_scale)


def _backward(wanted, grad_y, grad_h, x, residual, gate, rstd, post_weight, pre_weight, gate_act, residual_scale):
    """The gradients; of gate, post_weight and pre_weight those that are wanted, None for the others."""
    dx, dresidual, *sums = run_cxx(
        "gated_norm_bwd", x, (grad_y, grad_h, x, residual, gate, rstd, post_weight, pre_weight,
                              GATE_ACTS.get(gate_act, -1), residual_scale, *wanted), _validate_backward,
        grad_y, grad_h, x, residual, gate, rstd, post_weight, pre_weight, gate_act, residual_scale)
    return (dx, dresidual, *(d if want and t is not None else None
                             for want, t, d in zip(wanted, (gate, post_weight, pre_weight), sums)))


def _validate_backward(grad_y, grad_h, x, residual, gate, rstd, post_weight, pre_weight, gate_act, residual_scale):
    import torch

    validate_gated_norm_inputs(x, residual, gate, post_weight, pre_weight, gate_act, residual_scale)
    if grad_h is not None and pre_weight is None:
        raise ValueError("gated_residual_norm_backward: grad_h without pre_weight")
    for name, t in (("grad_y", grad_y), ("grad_h", grad_h)):
        if t is None:
            continue
        if not isinstance(t, torch.Tensor) or t.dtype != x.dtype:
            raise TypeError(f"gated_residual_norm_backward: {name} must be a tensor of x's dtype")
        if t.shape != x.shape or t.device != x.device:
            raise ValueError(f"gated_residual_norm_backward: {name} must have the shape and device of x")
    if not isinstance(rstd, torch.Tensor) or rstd.dtype != torch.float32:
        raise TypeError("gated_residual_norm_backward: rstd must be a float32 tensor")
    if tuple(rstd.shape) != (*x.shape[:-1], 2) or rstd.device != x.device:
        raise ValueError("gated_residual_norm_backward: rstd must be [..., 2] on the device of x")


_FUNCTION = None


def _function():
    global _FUNCTION
    if _FUNCTION is not None:
        return _FUNCTION
    import torch

    class GatedResidualNorm(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, residual, gate, post_weight, pre_weight, gate_act, residual_scale, eps):
            y, h, rstd = run_gated_residual_norm(x, residual, gate, post_weight=post_weight, pre_weight=pre_weight,
                                                 gate_act=gate_act, residual_scale=residual_scale, eps=eps)
            ctx.save_for_backward(x, residual, gate, post_weight, pre_weight, rstd)
            ctx.gate_act, ctx.residual_scale = gate_act, residual_scale
            ctx.set_materialize_grads(False)
            return y, h

        @staticmethod
        @torch.autograd.function.once_differentiable
        def backward(ctx, grad_y, grad_h):
            x, residual, gate, post_weight, pre_weight, rstd = ctx.saved_tensors
            grads = _backward(ctx.needs_input_grad[2:5], grad_y, grad_h, x, residual, gate, rstd, post_weight,
                              pre_weight, ctx.gate_act, ctx.residual_scale)
            return (*grads, None, None, None)

    _FUNCTION = GatedResidualNorm
    return _FUNCTION


def gated_residual_norm(x, residual, gate=None, *, post_weight=None, pre_weight=None, gate_act: str = "none",
                        residual_scale: float = 1.0, eps: float = 1e-6):
    """(y, h): the residual stream after a block and the next block's normalised input (None without
    pre_weight). Differentiable in every tensor argument."""
    import torch

    tensors = (x, residual, gate, post_weight, pre_weight)
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in tensors):
        validate_gated_norm_inputs(*tensors, gate_act, residual_scale, eps)
        return _function().apply(*distinct(*tensors), gate_act, residual_scale, eps)
    return run_gated_residual_norm(x, residual, gate, post_weight=post_weight, pre_weight=pre_weight,
                                   gate_act=gate_act, residual_scale=residual_scale, eps=eps)[:2]
