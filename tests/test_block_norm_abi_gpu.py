"""nb200_gated_norm_bwd with pointers that torch never hands out."""
from __future__ import annotations

import ctypes

import pytest

from conftest import cuda_available
from test_block_norm_gpu import _backward_ref, _check, _make

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_available(), reason="needs a CUDA device")]


def _placed(t, at):
    """t's values `at` elements into a buffer of their own, with something else on either side."""
    import torch

    room = torch.full((t.numel() + at + 16,), 7.0, dtype=t.dtype, device="cuda")
    room[at:at + t.numel()] = t.reshape(-1)
    return room


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("rows_at,gate_at", [(0, 1), (0, 3), (1, 0), (3, 1), (0, 0)])
@pytest.mark.parametrize("shape", [(100, 20, 4096), (2000, 4, 256), (3000, 2, 64), (5, 700, 512)])
def test_gate_gradients_off_the_rows_boundary(shape, rows_at, gate_at, dtype):
    """Every row tensor starts `rows_at` elements off the 16-byte boundary, the gate's gradient `gate_at`: many whole
    gate groups for a CTA, whose gradients it writes itself, and one group over many CTAs."""
    import torch

    import neptune_opt_b200._lib as L

    s = _make(shape, dtype, "sequence", 3)
    batch, seq, width = shape
    rows, code = batch * seq, {"float32": 0, "bfloat16": 1, "float16": 2}[dtype]
    lib, esize = L.load(), s["x"].element_size()
    x = s["x"].double()
    r1 = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
    y = s["residual"].double() + 0.5 * torch.tanh(s["gate"].double()) * x * r1 * s["post"].double()
    rstd = torch.cat([r1, torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-6)], -1).float()
    room = {n: _placed(s[n], rows_at) for n in ("x", "residual", "gy", "gh")}
    out = {n: _placed(torch.zeros_like(s["x"]), rows_at) for n in ("x", "residual")}
    out["gate"] = _placed(torch.zeros_like(s["gate"]), gate_at)
    for n in ("post", "pre"):
        out[n] = torch.zeros_like(s[n])

    def ptr(t, at=0):
        return ctypes.c_void_p(t.data_ptr() + at * esize)

    a = L.NB200NormArgs(ptr(room["x"], rows_at), ptr(room["residual"], rows_at), s["gate"].data_ptr(), s["post"].data_ptr(),
                        s["pre"].data_ptr(), rows, width, width, width, width, width, width, seq, 1, 0.5, 1e-6)
    size = lib.nb200_gated_norm_bwd_work_bytes(ctypes.byref(a))
    assert size > 0
    work = torch.empty(size, dtype=torch.uint8, device="cuda")
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    L.check(lib.nb200_gated_norm_bwd(ctypes.byref(a), code, ptr(rstd), ptr(room["gy"], rows_at), ptr(room["gh"], rows_at),
                                     ptr(out["x"], rows_at), ptr(out["residual"], rows_at), ptr(out["gate"], gate_at),
                                     ptr(out["post"]), ptr(out["pre"]), ptr(work), size, stream), "gated_norm_bwd")
    torch.cuda.synchronize()
    n = 2.0 ** -24 * width + 2.0 ** -20
    for name, (ref, mag) in _backward_ref(s, rstd, "tanh", 0.5).items():
        at = rows_at if name in ("x", "residual") else gate_at if name == "gate" else 0
        got = out[name][at:at + s[name].numel()].view(s[name].shape)
        extra = 0.0 if name in ("x", "residual") else (rows + 8) * 2.0 ** -24
        _check(got, ref, mag, 4 * n + extra, dtype, f"{shape} {dtype} d{name}")
        assert (out[name][:at] == 7).all() and (name in ("post", "pre") or (out[name][at + s[name].numel():] == 7).all())
