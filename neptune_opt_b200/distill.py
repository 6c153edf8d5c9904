"""Distillation from a teacher of which only the top logits were kept (nb200_distill_loss,
nb200_distill_loss_bwd).

Per row of student logits x over the whole vocabulary, with kept teacher logits t_j at indices i_j:

    p_j  = exp(t_j / T - Z)     Z = logsumexp(t / T) over the kept entries, or teacher_lse
    q    = softmax(x / T)
    loss = sum_j p_j (log p_j - log q[i_j])
    dx   = grad / T * (mass * q - scatter(p)),   mass = sum_j p_j

An index outside [0, vocab), or a teacher logit of -inf, marks an entry that was not kept; a row without
kept entries (a prompt token) has loss 0 and gradient 0 whatever its logits hold. Entries that name one
column twice add.
The row's logsumexp is the reference's skeleton (neptune_codegen/library.py:19, :157); it has no loss
and no gradient. Everything is fp32 inside; the gradient is rounded once to the logits' dtype.

Errors follow the backend's convention: TypeError for dtypes, ValueError for devices, shapes and
parameters, NotImplementedError past the kernels' kept entries per row.
"""
from __future__ import annotations

import math

from neptune_opt_b200.torch_op import run_cxx

MAX_TOP = 256


def validate_distill_inputs(logits, teacher_logits, teacher_index, temperature, teacher_lse=None):
    """Metadata-only contract."""
    import torch

    what = "distill_loss"
    for name, t in (("logits", logits), ("teacher_logits", teacher_logits)):
        if not isinstance(t, torch.Tensor) or t.layout != torch.strided:
            raise TypeError(f"{what}: {name} must be a strided tensor")
        if t.dtype not in (torch.float32, torch.bfloat16, torch.float16):
            raise TypeError(f"{what}: {name} must be float32/bfloat16/float16, got {t.dtype}")
    if not isinstance(teacher_index, torch.Tensor) or teacher_index.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{what}: teacher_index must be an int32/int64 tensor")
    if teacher_lse is not None and (not isinstance(teacher_lse, torch.Tensor) or teacher_lse.dtype != torch.float32):
        raise TypeError(f"{what}: teacher_lse must be a float32 tensor")
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"{what}: logits must be [..., vocab], got {tuple(logits.shape)}")
    if (teacher_logits.shape != teacher_index.shape or teacher_logits.dim() != logits.dim()
            or teacher_logits.shape[:-1] != logits.shape[:-1]):
        raise ValueError(f"{what}: teacher_logits {tuple(teacher_logits.shape)} and teacher_index "
                         f"{tuple(teacher_index.shape)} must be [..., top] over the rows of {tuple(logits.shape)}")
    if teacher_lse is not None and teacher_lse.shape != logits.shape[:-1]:
        raise ValueError(f"{what}: teacher_lse must be {tuple(logits.shape[:-1])}, got {tuple(teacher_lse.shape)}")
    for name, t in (("teacher_logits", teacher_logits), ("teacher_index", teacher_index), ("teacher_lse", teacher_lse)):
        if t is not None and t.device != logits.device:
            raise ValueError(f"{what}: {name} must be on the device of logits")
    if logits.device.type not in ("cuda", "meta"):
        raise ValueError(f"{what}: inputs must be CUDA tensors, got {logits.device}")
    if not (math.isfinite(temperature) and temperature > 0):
        raise ValueError(f"{what}: temperature must be finite and positive, got {temperature}")
    if teacher_logits.shape[-1] > MAX_TOP:
        raise NotImplementedError(f"{what}: {teacher_logits.shape[-1]} kept logits per row exceed {MAX_TOP}")


def run_distill_loss(logits, teacher_logits, teacher_index, *, temperature: float = 1.0, teacher_lse=None):
    """(loss [...], stats [..., 3]) in fp32; stats holds each row's logsumexp(logits / T), teacher
    normaliser Z and kept mass, which the backward pass takes. teacher_lse [...] is the teacher's
    logsumexp(t / T) over its whole vocabulary; without it the kept entries are normalised to mass 1."""
    contract = (logits, teacher_logits, teacher_index, temperature, teacher_lse)
    return run_cxx("distill_loss", logits, contract, validate_distill_inputs, *contract)


def distill_loss_backward(grad, logits, teacher_logits, teacher_index, stats, *, temperature: float = 1.0):
    """Gradient of the logits (fresh, contiguous, their dtype) for the gradient of each row's loss, from
    the forward pass's stats."""
    contract = (grad, logits, teacher_logits, teacher_index, stats, temperature)
    return run_cxx("distill_loss_bwd", logits, contract, _validate_backward, *contract)


def _validate_backward(grad, logits, teacher_logits, teacher_index, stats, temperature):
    import torch

    validate_distill_inputs(logits, teacher_logits, teacher_index, temperature)
    for name, t, shape in (("grad", grad, logits.shape[:-1]), ("stats", stats, (*logits.shape[:-1], 3))):
        if not isinstance(t, torch.Tensor) or t.dtype != torch.float32:
            raise TypeError(f"distill_loss_backward: {name} must be a float32 tensor")
        if tuple(t.shape) != tuple(shape) or t.device != logits.device:
            raise ValueError(f"distill_loss_backward: {name} must be {tuple(shape)} on the device of logits")


_FUNCTION = None


def _function():
    global _FUNCTION
    if _FUNCTION is not None:
        return _FUNCTION
    import torch

    class DistillLoss(torch.autograd.Function):
        @staticmethod
        def forward(ctx, logits, teacher_logits, teacher_index, temperature, teacher_lse):
            loss, stats = run_distill_loss(logits, teacher_logits, teacher_index, temperature=temperature,
                                           teacher_lse=teacher_lse)
            ctx.save_for_backward(logits, teacher_logits, teacher_index, stats)
            ctx.temperature = temperature
            return loss

        @staticmethod
        @torch.autograd.function.once_differentiable
        def backward(ctx, grad):
            logits, teacher_logits, teacher_index, stats = ctx.saved_tensors
            return (distill_loss_backward(grad, logits, teacher_logits, teacher_index, stats,
                                          temperature=ctx.temperature), None, None, None, None)

    _FUNCTION = DistillLoss
    return _FUNCTION


def distill_loss(logits, teacher_logits, teacher_index, *, temperature: float = 1.0, teacher_lse=None):
    """Loss of each row, fp32 [...]. Differentiable in the logits; the teacher is a constant."""
    import torch

    if torch.is_grad_enabled() and isinstance(logits, torch.Tensor) and logits.requires_grad:
        return _function().apply(logits, teacher_logits, teacher_index, temperature, teacher_lse)
    return run_distill_loss(logits, teacher_logits, teacher_index, temperature=temperature, teacher_lse=teacher_lse)[0]
