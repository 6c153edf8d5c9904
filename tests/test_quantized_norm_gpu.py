"""GPU parity of RMSNorm to 8 bits against the formulas in float64.

Tolerances, elementwise: everything is fp32 and rounded once. A row's mean square is off by at most width 2^-24
relative (sums of one sign, any order), its reciprocal root by half of that, every other step by 2^-22 of the
magnitudes it adds; where a residual is added, y is off by 2^-24 (|x| + |r|), which weight and norm carry
along. With N = width 2^-24 + 2^-20 as the bound of every factor of a row:
  y: half a step of its type (2^-24, 2^-8, 2^-11 relative) and 2^-23 (|x| + |r|)
  scale: N relative
  q * scale: half a step of the 8-bit type (2^-4 e4m3, 2^-3 e5m2 of the value; 2^-10 and 2^-17 below their
    normal range; half a unit int8) of scale, N |h|, and 2^-22 rsqrt |weight| (|x| + |r|)
"""
from __future__ import annotations

import math

import pytest

from conftest import cuda_available

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_available(), reason="needs a CUDA device")]

HALF_STEP = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
KINDS = {"float8_e4m3fn": (448.0, 2.0 ** -4, 2.0 ** -10), "float8_e5m2": (57344.0, 2.0 ** -3, 2.0 ** -17),
         "int8": (127.0, 0.0, 0.5)}


def make(shape, dtype, seed=0, residual=True):
    import torch

    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = getattr(torch, dtype)

    def one(*s, std=1.0, mean=0.0):
        return (torch.randn(*s, device="cuda", generator=gen) * std + mean).to(dt)

    return one(*shape), one(shape[-1], mean=1.0, std=0.3), one(*shape, std=3.0) if residual else None


def check(x, weight, residual, group, kind, eps=1e-6, got=None):
    import torch

    import neptune_opt_b200 as NB

    width = x.shape[-1]
    q, scale, y = got if got is not None else NB.quantized_rms_norm(x, weight, residual, group=group,
                                                                    dtype=getattr(torch, kind), eps=eps)
    most, rel, least = KINDS[kind]
    n = width * 2.0 ** -24 + 2.0 ** -20
    mag = x.double().abs() + (residual.double().abs() if residual is not None else 0.0)
    ry = x.double() + (residual.double() if residual is not None else 0.0)
    r = torch.rsqrt(ry.square().mean(-1, keepdim=True) + eps)
    h = ry * r * weight.double()
    groups = h.view(*x.shape[:-1], -1, group or width)
    rs = (groups.abs().amax(-1) / most).clamp(min=2.0 ** -126)
    carried = 2.0 ** -22 * r * weight.double().abs() * mag
    assert scale.dtype == torch.float32 and scale.shape == rs.shape
    slack = carried.view(*x.shape[:-1], -1, group or width).amax(-1) / most
    assert bool(((scale.double() - rs).abs() <= n * rs + slack).all()), "scales"
    if residual is None:
        assert y is None
    else:
        assert y.dtype == x.dtype and y.shape == x.shape
        tol = HALF_STEP[str(x.dtype)[6:]] * ry.abs() + 2.0 ** -23 * mag + 2.0 ** -26
        assert bool(((y.double() - ry).abs() <= tol).all()), "y"
    assert q.dtype == getattr(torch, kind) and q.shape == x.shape
    each = scale.double().repeat_interleave(group or width, -1)
    off = (q.double() * each - h).abs()
    tol = torch.maximum(rel * h.abs(), least * each) + n * h.abs() + carried + 2.0 ** -140
    assert bool((off <= tol).all()), f"q off by up to {(off / tol).amax():.3f} of its bound"
    return q, scale, y


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("dtype", list(HALF_STEP))
@pytest.mark.parametrize("width,group", [(1, None), (7, None), (8, None), (64, 32), (96, 16), (255, None), (256, 64),
                                         (257, None), (1001, None), (1024, 128), (1025, None), (1152, 128)])
def test_against_the_formulas(kind, dtype, width, group):
    check(*make((37, width), dtype, width), group, kind)


@pytest.mark.parametrize("dtype", list(HALF_STEP))
@pytest.mark.parametrize("width", [2048, 2051, 4096, 4100, 4097, 8192, 8190, 16384, 16383])
@pytest.mark.parametrize("residual", [True, False])
def test_wide_rows(dtype, width, residual):
    check(*make((19, width), dtype, width, residual), None, "float8_e4m3fn")
    if width % 128 == 0:
        check(*make((19, width), dtype, width, residual), 128, "float8_e4m3fn")
        check(*make((19, width), dtype, width, residual), 16, "int8")


@pytest.mark.parametrize("rows", [1, 2, 3, 2999])
def test_row_counts(rows):
    check(*make((rows, 512), "bfloat16", rows), 64, "float8_e5m2")
    check(*make((rows, 2304), "bfloat16", rows), None, "float8_e4m3fn")


def test_leading_dimensions_and_no_rows():
    import torch

    import neptune_opt_b200 as NB

    x, w, r = make((2, 3, 5, 192), "float16")
    q, scale, y = check(x, w, r, 64, "float8_e4m3fn")
    assert scale.shape == (2, 3, 5, 3)
    q, scale, y = NB.quantized_rms_norm(x[:0], w, r[:0], dtype=torch.int8)
    assert q.shape == (0, 3, 5, 192) and scale.shape == (0, 3, 5, 1) and y.shape == (0, 3, 5, 192)
    check(x[0, 0, 0], w, r[0, 0, 0], None, "int8")


@pytest.mark.parametrize("dtype", list(HALF_STEP))
@pytest.mark.parametrize("group", [None, 32])
def test_layouts(dtype, group):
    """Slices of wider rows, bases off the 16-byte boundary, transposed and expanded rows, a strided weight."""
    import torch

    import neptune_opt_b200 as NB

    x, w, r = make((24, 320), dtype)
    wide = torch.zeros(24, 700, device="cuda", dtype=x.dtype)
    for at in (0, 1, 8, 13):
        a, b = wide.clone()[:, at:at + 320], wide.clone()[:, at:at + 320]
        a.copy_(x), b.copy_(r)
        check(a, w, b, group, "float8_e4m3fn")
        check(a, w, r, group, "float8_e4m3fn")
    check(x.t().contiguous().t(), w, r, group, "int8")
    check(x[:1].expand(24, -1), w, r, group, "int8")
    check(x, torch.stack([w, w], 1)[:, 0], r, group, "float8_e5m2")
    shifted = torch.empty(321, device="cuda", dtype=x.dtype)[1:]
    shifted.copy_(w)
    a, b = NB.quantized_rms_norm(x, shifted, r, group=group), NB.quantized_rms_norm(x, w, r, group=group)
    assert bool(((a[1] - b[1]).abs() <= 2.0 ** -20 * b[1]).all()) and torch.equal(a[2], b[2])


@pytest.mark.parametrize("dtype", list(HALF_STEP))
@pytest.mark.parametrize("rows,width", [(1, 3), (2, 3), (9, 1), (5, 5), (3, 9), (17, 33), (8, 4001)])
def test_rows_off_the_boundary_up_to_the_end_of_their_memory(dtype, rows, width):
    """Odd rows one behind the other, and overlapping ones: what lies around a row is neither read as part of it nor
    written. NaN on all sides of the inputs, sentinels around the outputs (through the C entry)."""
    import ctypes

    import torch

    import neptune_opt_b200._lib as L

    x, w, r = make((rows, width), dtype, rows * width)
    dt, n = x.dtype, rows * width
    pad = 64
    room = {k: torch.full((n + 2 * pad,), math.nan, device="cuda", dtype=dt) for k in ("x", "r")}
    for k, t in (("x", x), ("r", r)):
        room[k][pad:pad + n] = t.flatten()
    q = torch.full((n + 2 * pad,), 77, device="cuda", dtype=torch.uint8)
    y = torch.full((n + 2 * pad,), 3.0, device="cuda", dtype=dt)
    scale = torch.empty(rows, 1, device="cuda")
    at = lambda t: t.data_ptr() + pad * t.element_size()  # noqa: E731
    code = {"float32": 0, "bfloat16": 1, "float16": 2}[dtype]
    a = L.NB200Norm8Args(at(room["x"]), at(room["r"]), w.data_ptr(), rows, width, 0, width, width, code, 0, 1e-6)
    L.check(L.load().nb200_norm8(ctypes.byref(a), at(q), scale.data_ptr(), at(y),
                                 ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)), "norm8")
    got = q[pad:pad + n].view(torch.float8_e4m3fn).view(rows, width), scale, y[pad:pad + n].view(rows, width)
    check(x, w, r, None, "float8_e4m3fn", got=got)
    for t, v in ((q, 77), (y, 3.0)):
        assert bool((t[:pad] == v).all()) and bool((t[pad + n:] == v).all())
    windows = room["x"][pad:pad + n].as_strided((max(1, n - width), width), (1, 1))
    check(windows, w, None, None, "int8")


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("group", [None, 64])
@pytest.mark.parametrize("width", [256, 4096])
def test_rows_of_zeros_and_values_that_are_not_numbers(kind, group, width):
    import torch

    import neptune_opt_b200 as NB

    x, w, r = make((6, width), "float32")
    x[0] = r[0] = 0.0
    x[1, 70] = math.nan
    x[2, 70] = math.inf
    x[3, :64] = r[3, :64] = 0.0  # a group of zeros in an ordinary row
    x[4] *= 1e-30
    r[4] *= 1e-30
    q, scale, y = NB.quantized_rms_norm(x, w, r, group=group, dtype=getattr(torch, kind))
    assert not q[0].double().any() and bool((scale[0] == 2.0 ** -126).all()) and not y[0].any()
    for row in (1, 2):  # an infinity makes the norm's factor 0 and itself NaN
        if kind != "int8":
            assert bool(torch.isnan(q[row].float())[70])
        assert bool(torch.isnan(scale[row]).any())
    assert bool(torch.isnan(scale[1]).all())
    assert not q[3, :64].double().any()
    if group:
        assert float(scale[3, 0]) == 2.0 ** -126
    keep = torch.tensor([0, 3, 4, 5], device="cuda")
    check(x[keep], w, r[keep], group, kind, got=(q[keep], scale[keep], y[keep]))
    w[5] = math.nan
    q, scale, _ = NB.quantized_rms_norm(x[5:], w, r[5:], group=group, dtype=getattr(torch, kind))
    assert bool(torch.isnan(scale[0, 0])) and bool(torch.isnan(scale).all()) == (group is None)


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("group", [None, 64])
def test_values_take_the_byte_that_is_nearest(kind, group):
    """Without a residual a quotient is weight x / max |weight x| times the type's largest value: both products, the
    reciprocal, its factor and the last product round once, and once more the conversion of the 64-bit quotient here.
    With d = 6 2^-24 between the two, a byte is at most 2 d of the quotient further off than the nearest one."""
    import torch

    import neptune_opt_b200 as NB

    x, w, _ = make((501, 1024), "float32", 5, residual=False)
    q, _, _ = NB.quantized_rms_norm(x, w, group=group, dtype=getattr(torch, kind))
    h = (x.double() * w.double()).view(501, -1, group or 1024)
    quotient = (h / h.abs().amax(-1, keepdim=True) * KINDS[kind][0]).view_as(q)
    nearest = quotient.round() if kind == "int8" else quotient.to(q.dtype).double()
    further = (q.double() - quotient).abs() - (nearest - quotient).abs()
    assert bool((further <= 2 * 6 * 2.0 ** -24 * quotient.abs()).all())


@pytest.mark.parametrize("by,weight", [(1e-17, 1e-20), (1e-16, 1e-21), (1e17, 1e18)])
def test_products_whose_reciprocal_leaves_fp32(by, weight):
    """Where weight x is about 1e-37 or 1e35, its reciprocal times the largest value is not fp32's."""
    x, w, _ = make((33, 512), "float32", 6, residual=False)
    check(x * by, w * weight, None, None, "float8_e4m3fn", eps=1e-40)
    check(x * by, w * weight, None, 128, "int8", eps=1e-40)


def test_the_largest_value_fills_the_type():
    import torch

    x, w, r = make((50, 1000), "bfloat16")
    for kind, (most, _, _) in KINDS.items():
        q, _, _ = check(x, w, r, None, kind)
        assert bool((q.double().abs().amax(-1) == most).all())


def test_other_eps_and_runs_alike():
    import torch

    import neptune_opt_b200 as NB

    x, w, r = make((3000, 1024), "bfloat16")
    check(x, w, r, 128, "float8_e4m3fn", eps=10.0)
    check(x * 0, w, r * 0, 128, "float8_e4m3fn", eps=1e-30)
    first = NB.quantized_rms_norm(x, w, r, group=128)
    for _ in range(5):
        again = NB.quantized_rms_norm(x, w, r, group=128)
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(first, again))


def test_aliases_and_replays():
    """x as its own residual; a captured call whose inputs change between replays."""
    import torch

    import neptune_opt_b200 as NB

    x, w, r = make((65, 640), "bfloat16")
    check(x, w, x, None, "float8_e4m3fn")
    NB.quantized_rms_norm(x, w, r)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = NB.quantized_rms_norm(x, w, r, group=128)
    for factor in (1.0, -0.5, 3.0):
        x.mul_(factor)
        g.replay()
        check(x, w, r, 128, "float8_e4m3fn", got=out)
