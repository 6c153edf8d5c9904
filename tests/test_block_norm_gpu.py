"""GPU parity of the gated residual norm, forward and backward, against the formulas in float64.

Tolerances, elementwise: results are computed in fp32 and rounded once, so |got - ref| is at most half a
unit of the dtype (relative 2^-9 / 2^-12 / 2^-24, taken as one unit) plus the fp32 steps: a norm is off by
at most width 2^-24 / 2 (in any summation order, 2^-12 at width 4096; sums of one sign), every other
step by 2^-22 of the magnitudes it adds. Column sums over n rows add (n + 8) 2^-24 of the sum of
magnitudes. With N = 2^-24 width + 2^-20 as the bound on every row statistic:
  y, h: N (|residual| + |scale a z|) r2 w2      dY, dx: N of the sum of the magnitudes of its terms
"""
from __future__ import annotations

import math

import pytest

from conftest import cuda_available

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_available(), reason="needs a CUDA device")]

UNIT = {"float32": 2.0 ** -23, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
TINY = {"float32": 1e-38, "bfloat16": 1e-38, "float16": 2.0 ** -24}


def _make(shape, dtype, gate, seed):
    import torch

    gen = torch.Generator().manual_seed(seed)
    dt = getattr(torch, dtype)

    def one(*s, std=1.0, mean=0.0):
        return (torch.randn(*s, generator=gen) * std + mean).to(dt).cuda()

    c = shape[-1]
    g = {"none": None, "channel": (c,), "full": shape, "sequence": (shape[0],) + (1,) * (len(shape) - 2) + (c,)}[gate]
    return {"x": one(*shape), "residual": one(*shape, std=2.0), "gate": None if g is None else one(*g, mean=0.4),
            "post": one(c, mean=1.0, std=0.2), "pre": one(c, mean=1.0, std=0.2), "gy": one(*shape), "gh": one(*shape)}


def _act(g, kind):
    import torch

    if g is None:
        return 1.0, None
    if kind == "tanh":
        return torch.tanh(g), 1 - torch.tanh(g) ** 2
    if kind == "sigmoid":
        return torch.sigmoid(g), torch.sigmoid(g) * (1 - torch.sigmoid(g))
    return g, torch.ones_like(g)


def _forward_ref(s, act, scale, eps):
    import torch

    x, r = s["x"].double(), s["residual"].double()
    w1 = None if s["post"] is None else s["post"].double()
    w2 = None if s["pre"] is None else s["pre"].double()
    a, _ = _act(None if s["gate"] is None else s["gate"].double(), act)
    r1 = torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) if w1 is not None else torch.ones_like(x[..., :1])
    z = x * r1 * (w1 if w1 is not None else 1.0)
    y = r + scale * a * z
    r2 = torch.rsqrt((y * y).mean(-1, keepdim=True) + eps) if w2 is not None else torch.ones_like(x[..., :1])
    return y, None if w2 is None else y * r2 * w2, torch.cat([r1, r2], -1), r.abs() + (scale * a * z).abs()


def _backward_ref(s, rstd, act, scale):
    """{name: (value, magnitude of the terms it is built from)}."""
    import torch

    x, r = s["x"].double(), s["residual"].double()
    one = torch.ones(x.shape[-1], dtype=torch.float64, device="cuda")
    w1 = one if s["post"] is None else s["post"].double()
    w2 = one if s["pre"] is None else s["pre"].double()
    a, da = _act(None if s["gate"] is None else s["gate"].double(), act)
    r1, r2 = rstd.double()[..., :1], rstd.double()[..., 1:]
    xhat = x * r1
    z = xhat * w1
    yhat, ymag = (r + scale * a * z) * r2, (r.abs() + (scale * a * z).abs()) * r2
    zero = torch.zeros_like(x)
    gy = zero if s["gy"] is None else s["gy"].double()
    gh = zero if s["gh"] is None else s["gh"].double()
    t = gh * w2
    m2 = (t * yhat).mean(-1, keepdim=True) if s["pre"] is not None else 0.0
    m2mag = (t * ymag).abs().mean(-1, keepdim=True) if s["pre"] is not None else 0.0
    dy = gy + r2 * (t - yhat * m2)
    dymag = gy.abs() + r2 * (t.abs() + ymag * m2mag)
    u, umag = scale * a * dy * w1, (scale * a * w1).abs() * dymag if s["gate"] is not None else (scale * w1).abs() * dymag
    m1 = (u * xhat).mean(-1, keepdim=True) if s["post"] is not None else 0.0
    m1mag = (umag * xhat.abs()).mean(-1, keepdim=True) if s["post"] is not None else 0.0
    out = {"x": (r1 * (u - xhat * m1), r1 * (umag + xhat.abs() * m1mag)), "residual": (dy, dymag)}

    def columns(v, mag):
        return v.reshape(-1, x.shape[-1]).sum(0), mag.reshape(-1, x.shape[-1]).sum(0)

    if s["post"] is not None:
        out["post"] = columns(scale * a * dy * xhat, (scale * a * xhat if s["gate"] is not None else scale * xhat).abs() * dymag)
    if s["pre"] is not None:
        out["pre"] = columns(gh * yhat, gh.abs() * ymag)
    if s["gate"] is not None:
        v, mag = scale * da * z * dy, (scale * da * z).abs() * dymag
        if s["gate"].dim() == 1:
            out["gate"] = columns(v, mag)
        else:
            dims = [i for i in range(x.dim() - 1) if s["gate"].shape[i] == 1 and x.shape[i] != 1]
            out["gate"] = (v.sum(dims, keepdim=True), mag.sum(dims, keepdim=True)) if dims else (v, mag)
    return out


def _check(got, ref, mag, bound, dtype, label):
    err = (got.double() - ref).abs()
    over = err - (UNIT[dtype] * ref.abs() + bound * mag + TINY[dtype])
    assert over.max().item() <= 0, f"{label}: exceeds the bound by {over.max().item():.3g}"


def _run_and_check(s, dtype, act="none", scale=1.0, eps=1e-6, label=""):
    import torch

    import neptune_opt_b200 as NB

    kw = {"post_weight": s["post"], "pre_weight": s["pre"], "gate_act": act, "residual_scale": scale}
    y, h, rstd = NB.run_gated_residual_norm(s["x"], s["residual"], s["gate"], eps=eps, **kw)
    ry, rh, rr, mag = _forward_ref(s, act, scale, eps)
    width, rows = s["x"].shape[-1], s["x"].numel() // s["x"].shape[-1]
    n = 2.0 ** -24 * width + 2.0 ** -20
    _check(y, ry, mag, n, dtype, f"{label} y")
    assert ((rstd.double() - rr).abs() <= (n + n * mag.square().mean(-1, keepdim=True) * rr ** 2) * rr).all(), f"{label} rstd"
    if h is None:
        assert s["pre"] is None
    else:
        _check(h, rh, mag * rr[..., 1:] * s["pre"].double().abs(), 2 * n + n * 2, dtype, f"{label} h")
    grads = NB.gated_residual_norm_backward(s["gy"], s["gh"], s["x"], s["residual"], s["gate"], rstd, **kw)
    again = NB.gated_residual_norm_backward(s["gy"], s["gh"], s["x"], s["residual"], s["gate"], rstd, **kw)
    ref = _backward_ref(s, rstd, act, scale)
    for name, got, second in zip(("x", "residual", "gate", "post", "pre"), grads, again):
        if s[name] is None:
            assert got is None
            continue
        assert got.shape == s[name].shape and got.dtype == s[name].dtype and torch.equal(got, second)
        extra = 0.0 if name in ("x", "residual") else (rows + 8) * 2.0 ** -24
        _check(got, *ref[name], 4 * n + extra, dtype, f"{label} d{name}")
    return grads


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("width", [1, 7, 31, 64, 256, 264, 500, 512, 520, 1001, 2048, 4096, 4104, 5000, 8192, 8200, 16384])
def test_widths(width, dtype):
    _run_and_check(_make((3, 5, width), dtype, "sequence", width), dtype, "tanh", 0.5, label=f"{width} {dtype}")


@pytest.mark.parametrize("act", ["none", "tanh", "sigmoid"])
@pytest.mark.parametrize("gate", ["none", "channel", "sequence", "full"])
def test_gates(gate, act):
    for shape in ((2, 3, 96), (1, 1, 768), (5, 700, 200), (700, 5, 640)):
        _run_and_check(_make(shape, "float32", gate, 7), "float32", act, -1.5, label=f"{shape} {gate} {act}")


@pytest.mark.parametrize("without", ["post", "pre", "gy", "gh", "post gy", "pre gy"])
def test_absent_parts(without):
    s = _make((4, 33, 136), "bfloat16", "channel", 3)
    for name in without.split():
        s[name] = None
    if s["pre"] is None:
        s["gh"] = None
        if s["gy"] is None:
            s["gy"] = s["x"]
    _run_and_check(s, "bfloat16", label=without)


@pytest.mark.parametrize("without", ["", "post", "pre", "gy", "gh"])
@pytest.mark.parametrize("gate", ["none", "channel", "sequence", "full"])
@pytest.mark.parametrize("shape,dtype", [((2, 1000, 1024), "bfloat16"), ((3, 400, 768), "float32"),
                                         ((1, 701, 8192), "float16"), ((7, 200, 2056), "bfloat16")])
def test_rows_fetched_ahead(shape, dtype, gate, without):
    """Aligned rows, many for each CTA, so that every stage they pass through is used again."""
    s = _make(shape, dtype, gate, 17)
    if without:
        s[without] = None
    if s["pre"] is None:
        s["gh"] = None
    _run_and_check(s, dtype, "sigmoid" if gate == "full" else "tanh" if gate != "none" else "none", 0.7,
                   label=f"{shape} {gate} without {without}")


def test_many_rows_and_one_row():
    _run_and_check(_make((1, 128), "float32", "channel", 1), "float32", label="one row")
    _run_and_check(_make((40001, 72), "bfloat16", "channel", 2), "bfloat16", label="many rows")
    _run_and_check(_make((3, 3000, 1024), "bfloat16", "sequence", 2), "bfloat16", "sigmoid", label="chunks in groups")


def test_zero_and_extreme_rows():
    import torch

    import neptune_opt_b200 as NB

    s = _make((6, 640), "bfloat16", "channel", 5)
    s["x"][1] = 0.0
    s["residual"][1] = 0.0
    s["x"][2] *= 1e-20
    s["x"][3] = 3e4
    _run_and_check(s, "bfloat16", label="zero row")
    s["x"][4, 7] = math.nan
    y, h = NB.gated_residual_norm(s["x"], s["residual"], s["gate"], post_weight=s["post"], pre_weight=s["pre"])
    bad = torch.isnan(h.float()).any(-1)
    assert bad.tolist() == [False, False, False, False, True, False], "a NaN leaves its row"


def test_strided_rows_and_gates():
    import torch

    c = 384
    gen = torch.Generator().manual_seed(8)
    wide = torch.randn(4, 9, 3 * c, generator=gen).to(torch.bfloat16).cuda()
    s = _make((4, 9, c), "bfloat16", "sequence", 6)
    s["x"], s["residual"] = wide[..., :c], wide[..., c:2 * c]
    s["gate"] = wide[:, :1, 2 * c:]                      # a slice of a modulation vector
    s["gy"] = s["gy"][0, 0].expand(4, 9, c)              # broadcast gradient
    s["gh"] = wide.transpose(0, 1)[:, :, 1:c + 1].transpose(0, 1)  # rows off the 16-byte boundary
    _run_and_check(s, "bfloat16", "tanh", 2.0, label="strided")
    s["gy"] = torch.ones((), dtype=torch.bfloat16, device="cuda").expand(4, 9, c)
    _run_and_check(s, "bfloat16", "tanh", 2.0, label="gradient of a sum")


def test_autograd_and_differences():
    import torch

    import neptune_opt_b200 as NB

    s = _make((2, 3, 80), "float32", "sequence", 12)
    names = ("x", "residual", "gate", "post", "pre")
    leaves = [s[n].clone().requires_grad_() for n in names]
    y, h = NB.gated_residual_norm(*leaves[:3], post_weight=leaves[3], pre_weight=leaves[4], gate_act="sigmoid",
                                  residual_scale=0.7)
    torch.autograd.backward([y, h], [s["gy"], s["gh"]])
    direct = _run_and_check(s, "float32", "sigmoid", 0.7)
    assert all(torch.equal(t.grad, d) for t, d in zip(leaves, direct))
    y2, _ = NB.gated_residual_norm(*leaves[:3], post_weight=leaves[3], pre_weight=leaves[4])
    y2.sum().backward()  # only y is used

    def value(parts):
        y, h, _, _ = _forward_ref({**s, **dict(zip(names, parts))}, "sigmoid", 0.7, 1e-6)
        return (y * s["gy"].double()).sum() + (h * s["gh"].double()).sum()

    gen = torch.Generator(device="cuda").manual_seed(4)
    base = [s[n].double() for n in names]
    for i, grad in enumerate(direct):
        d = torch.randn(base[i].shape, dtype=torch.float64, device="cuda", generator=gen)
        up, down = list(base), list(base)
        up[i], down[i] = base[i] + 1e-6 * d, base[i] - 1e-6 * d
        slope = (value(up) - value(down)).item() / 2e-6
        got = (grad.double() * d).sum().item()
        assert abs(got - slope) <= 1e-5 * (grad.double() * d).abs().sum().item() + 1e-6, names[i]


def test_empty_and_other_stream():
    import torch

    import neptune_opt_b200 as NB

    s = _make((0, 64), "float32", "channel", 1)
    y, h, rstd = NB.run_gated_residual_norm(s["x"], s["residual"], s["gate"], post_weight=s["post"], pre_weight=s["pre"])
    assert y.shape == (0, 64) and rstd.shape == (0, 2)
    grads = NB.gated_residual_norm_backward(y, h, s["x"], s["residual"], s["gate"], rstd, post_weight=s["post"],
                                            pre_weight=s["pre"])
    assert not grads[2].any() and not grads[3].any()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        _run_and_check(_make((64, 640), "bfloat16", "full", 2), "bfloat16", label="stream")
    side.synchronize()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("gate", ["none", "channel", "sequence", "full"])
@pytest.mark.parametrize("shape", [(1, 1, 333), (2, 9, 1001), (3, 700, 77), (400, 3, 259), (2, 4, 4099), (1, 5, 8197),
                                   (600, 2, 514), (1, 3, 16383)])
def test_rows_off_the_vector_boundary(shape, gate, dtype):
    """Contiguous rows whose offsets repeat every 2 to 8 rows, alone and in groups that share a gate."""
    _run_and_check(_make(shape, dtype, gate, 31), dtype, "sigmoid", 0.8, label=f"{shape} {gate} {dtype}")


def test_slices_off_the_vector_boundary():
    """Rows with an aligned pitch and an unaligned start: tensors laid out alike, then each on its own."""
    import torch

    for same in (True, False):
        s = _make((6, 11, 520), "bfloat16", "sequence", 9)
        for i, name in enumerate(("x", "residual", "gy", "gh")):
            room = torch.zeros(6, 11, 528, dtype=torch.bfloat16, device="cuda")
            at = 3 if same else 1 + 2 * i
            room[..., at:at + 520] = s[name]
            s[name] = room[..., at:at + 520]
        _run_and_check(s, "bfloat16", "tanh", label=f"slices {same}")


def test_reciprocal_norms_off_their_boundary():
    import torch

    import neptune_opt_b200 as NB

    s = _make((5, 96), "float32", "channel", 4)
    kw = {"post_weight": s["post"], "pre_weight": s["pre"]}
    rstd = NB.run_gated_residual_norm(s["x"], s["residual"], s["gate"], **kw)[2]
    room = torch.empty(11, device="cuda")
    room[1:] = rstd.flatten()
    args = (s["gy"], s["gh"], s["x"], s["residual"], s["gate"])
    want = NB.gated_residual_norm_backward(*args, rstd, **kw)
    got = NB.gated_residual_norm_backward(*args, room[1:].view(5, 2), **kw)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
