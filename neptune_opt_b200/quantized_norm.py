"""RMSNorm with the residual's addition and an output in 8 bits with scales (nb200_norm8).

    y = x + residual                              (y = x without a residual)
    h = weight * y * rsqrt(mean(y^2) + eps)
    scale = max(max|h| / most, 2^-126)            per row, or per group of consecutive columns
    q = round(h / scale), saturating              so that q * scale stands for h

most is 448 for float8_e4m3fn, 57344 for float8_e5m2, 127 for int8. One pass over x and residual, everything
in fp32; y is rounded once to x's dtype, h is taken from the unrounded y. A NaN in a row makes its scales
NaN (and its float8 values; int8 ones are 0). The reference's RMSNorm (neptune_codegen/emitters.py:549-627)
has neither residual nor 8-bit output, and rounds between its stages: `rms_norm` keeps those.

x and residual are [..., width] in float32, bfloat16 or float16, weight [width] of the same dtype. No
gradient: one that is asked for is refused (NotImplementedError). Errors follow the backend's convention:
TypeError for dtypes, ValueError for devices, shapes and parameters, NotImplementedError past the kernels'
width.
"""
from __future__ import annotations

import math
import struct

from neptune_opt_b200.torch_op import run_cxx

GROUPS = (16, 32, 64, 128)
KINDS = {"float8_e4m3fn": 0, "float8_e5m2": 1, "int8": 2}
_KINDS = None
MAX_WIDTH = 16384


def _fp32_positive(value) -> bool:
    try:
        (value,) = struct.unpack("f", struct.pack("f", value))
    except OverflowError:
        return False
    return math.isfinite(value) and value > 0


def validate_quantized_norm_inputs(x, weight, residual, group, dtype, eps):
    """Metadata-only contract."""
    import torch

    what = "quantized_rms_norm"
    for name, t in (("x", x), ("weight", weight), ("residual", residual)):
        if t is None and name == "residual":
            continue
        if not isinstance(t, torch.Tensor) or t.layout != torch.strided:
            raise TypeError(f"{what}: {name} must be a strided tensor")
        if t.dtype not in (torch.float32, torch.bfloat16, torch.float16) or t.dtype != x.dtype:
            raise TypeError(f"{what}: {name} must share x's float32/bfloat16/float16 dtype, got {t.dtype}")
        if t.device != x.device:
            raise ValueError(f"{what}: {name} must be on the device of x")
    if dtype not in (None, torch.float8_e4m3fn, torch.float8_e5m2, torch.int8):
        raise TypeError(f"{what}: dtype must be float8_e4m3fn, float8_e5m2 or int8, got {dtype}")
    if x.device.type not in ("cuda", "meta"):
        raise ValueError(f"{what}: inputs must be CUDA tensors, got {x.device}")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"{what}: x must be [..., width], got {tuple(x.shape)}")
    if tuple(weight.shape) != (x.shape[-1],):
        raise ValueError(f"{what}: weight must be [{x.shape[-1]}], got {tuple(weight.shape)}")
    if residual is not None and residual.shape != x.shape:
        raise ValueError(f"{what}: residual {tuple(residual.shape)} must have the shape of x {tuple(x.shape)}")
    if group is not None and (group not in GROUPS or x.shape[-1] % group):
        raise ValueError(f"{what}: group must be one of {GROUPS} and divide the width {x.shape[-1]}, got {group}")
    if not _fp32_positive(eps):
        raise ValueError(f"{what}: eps must be finite and positive in fp32")
    if x.shape[-1] > MAX_WIDTH:
        raise NotImplementedError(f"{what}: width {x.shape[-1]} exceeds {MAX_WIDTH}")


def _kinds():
    """The op's number of each dtype; None stands for the default. Threads may meet here: the table is shown whole."""
    global _KINDS
    if _KINDS is None:
        import torch

        kinds = {getattr(torch, name): kind for name, kind in KINDS.items()}
        kinds[None] = KINDS["float8_e4m3fn"]
        _KINDS = kinds
    return _KINDS


def quantized_rms_norm(x, weight, residual=None, *, group=None, dtype=None, eps: float = 1e-6):
    """(q, scale, y): the normalised rows in 8 bits (dtype, float8_e4m3fn by default), their fp32 scales
    [..., 1] or [..., width / group], and the new residual stream in x's dtype (None without a residual).
    All fresh and contiguous."""
    q, scale, y = run_cxx("norm8", x, (x, weight, residual, 0 if group is None else group if group else -1,
                                       _kinds().get(dtype, -1), eps), validate_quantized_norm_inputs, x, weight, residual,
                          group, dtype, eps)
    return q, scale, None if residual is None else y
