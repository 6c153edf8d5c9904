"""GPU parity of the distillation loss and its gradient against the formulas in float64.

Tolerances. The row's sum of exponentials is an fp32 sum of terms of one sign whose chains hold at most
1024 terms, and the exponents are off by 2^-22 of the magnitudes they subtract, so logsumexp is off by at
most 2^-13 + 2^-21 |lse| (2^-14 from the chains, the rest from the exponentials); Z likewise (its sums
are shorter). Loss: sum_j p_j times the error of its logarithms, plus p's own relative error (2^-13) times
each term's magnitude. Gradient, from given stats: q and p have relative error
2^-22 (|x| / T + |lse| + 8) < 2^-14, and the result is rounded once (half a unit of the dtype, taken as one).
"""
from __future__ import annotations

import math

import pytest

from conftest import cuda_available

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_available(), reason="needs a CUDA device")]

UNIT = {"float32": 2.0 ** -23, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
TINY = {"float32": 1e-36, "bfloat16": 1e-36, "float16": 2.0 ** -24}


def _make(rows, vocab, top, dtype, seed, index_dtype="int64"):
    import torch

    gen = torch.Generator().manual_seed(seed)
    dt = getattr(torch, dtype)
    x = torch.randn(rows, vocab, generator=gen) * 3
    index = torch.stack([torch.randperm(vocab, generator=gen)[:top] for _ in range(rows)]) if rows else torch.empty(0, top)
    t = torch.randn(rows, top, generator=gen) * 2 + 6
    if top:
        x.scatter_(1, index.long(), t + torch.randn(rows, top, generator=gen))
    grad = torch.randn(rows, generator=gen) * (64.0 if dtype == "float16" else 1.0)
    return (x.to(dt).cuda(), t.to(dt).cuda(), index.to(getattr(torch, index_dtype)).cuda(), grad.cuda())


def _forward_ref(x, t, index, temperature, z=None):
    """loss, its bound, stats in float64."""
    import torch

    ok = (index >= 0) & (index < x.shape[-1])
    xd, td = x.double() / temperature, torch.where(ok, t.double() / temperature, -math.inf)
    lse = torch.logsumexp(xd, -1)
    z = torch.logsumexp(td, -1) if z is None else z.double()
    p = torch.where(ok, torch.exp(td - z[..., None]), 0.0)
    xi = torch.gather(xd, -1, torch.where(ok, index.long(), 0))
    live = p > 0
    zero = torch.zeros_like(p)
    term = torch.where(live, p * (td - z[..., None] - (xi - lse[..., None])), zero)
    mag = torch.where(live, td.abs() + z.abs()[..., None] + xi.abs() + lse.abs()[..., None], zero)
    bound = (torch.where(live, p * (2.0 ** -12 + 2.0 ** -20 * mag), zero) + 2.0 ** -13 * term.abs()).sum(-1) + 1e-30
    return term.sum(-1), bound, torch.stack([lse, z, p.sum(-1)], -1)


def _backward_ref(grad, x, t, index, stats, temperature):
    """dx and the magnitude of its terms."""
    import torch

    ok = (index >= 0) & (index < x.shape[-1])
    lse, z, mass = (s[..., None] for s in stats.double().unbind(-1))
    p = torch.where(ok, torch.exp(t.double() / temperature - z), 0.0)
    any_ = ok.any(-1, keepdim=True)
    w = grad.double()[..., None] / temperature
    q = torch.where(any_, torch.exp(x.double() / temperature - lse) * mass, 0.0)
    kept = torch.zeros_like(q).scatter_add_(-1, torch.where(ok, index.long(), 0), p)
    return w * (q - kept), w.abs() * (q + kept)


def _run_and_check(x, t, index, grad, dtype, temperature=1.0, z=None, label=""):
    import torch

    import neptune_opt_b200 as NB

    loss, stats = NB.run_distill_loss(x, t, index, temperature=temperature, teacher_lse=z)
    ref, bound, rstats = _forward_ref(x, t, index, temperature, z)
    assert loss.shape == x.shape[:-1] and stats.shape == (*x.shape[:-1], 3)
    over = (loss.double() - ref).abs() - bound
    assert over.max().item() <= 0, f"{label} loss exceeds the bound by {over.max().item():.3g}"
    fin = torch.isfinite(rstats)
    assert torch.equal(stats[~fin].double(), rstats[~fin]), f"{label} stats"
    assert ((stats.double() - rstats).abs() <= 2.0 ** -13 + 2.0 ** -21 * rstats.abs())[fin].all(), f"{label} stats"
    dx = NB.distill_loss_backward(grad, x, t, index, stats, temperature=temperature)
    assert torch.equal(dx, NB.distill_loss_backward(grad, x, t, index, stats, temperature=temperature))
    rdx, mag = _backward_ref(grad, x, t, index, stats, temperature)
    over = (dx.double() - rdx).abs() - (UNIT[dtype] * rdx.abs() + 2.0 ** -14 * mag + TINY[dtype])
    assert over.max().item() <= 0, f"{label} gradient exceeds the bound by {over.max().item():.3g}"
    assert dx.dtype == x.dtype and dx.shape == x.shape and dx.is_contiguous()
    return loss, dx


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("shape", [(1, 1, 1), (3, 5, 2), (1, 33, 33), (17, 1000, 16), (4, 8191, 64), (2, 32001, 256),
                                   (1, 131072, 100), (700, 2050, 7), (5, 262144, 64)])
def test_shapes(shape, dtype):
    x, t, index, grad = _make(*shape, dtype, sum(shape))
    _run_and_check(x, t, index, grad, dtype, label=f"{shape}")
    import torch

    z = torch.logsumexp(t.float() / 2.5, -1) + 0.3
    _run_and_check(x, t, index.int(), grad, dtype, 2.5, z, label=f"{shape} normalised")


def test_rows_without_entries_and_repeated_entries():
    import torch

    x, t, index, grad = _make(8, 500, 12, "bfloat16", 4)
    index[0] = -1                    # nothing kept
    x[0, 3] = math.nan
    index[1, 5:] = -100              # a usual "ignore" index
    index[2, 3] = 500                # past the vocabulary
    index[3, 4:8] = index[3, 0]      # one column named five times
    index[4, 1:] = -1
    t[1, 5:] = math.nan              # whatever sits in an entry that is not kept
    t[5, 0] = -math.inf              # kept, with probability 0
    loss, dx = _run_and_check(x[1:], t[1:], index[1:], grad[1:], "bfloat16")
    import neptune_opt_b200 as NB

    loss, stats = NB.run_distill_loss(x, t, index)
    dx = NB.distill_loss_backward(grad, x, t, index, stats)
    assert loss[0] == 0 and not dx[0].any() and torch.isfinite(loss).all() and torch.isfinite(dx.float()).all()
    assert stats[0, 1] == -math.inf and stats[0, 2] == 0


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("shape", [(1003, 500, 12), (401, 2003, 256), (1643, 8189, 64), (3281, 16381, 33)])
def test_many_narrow_rows(shape, dtype):
    """Row counts that are no multiple of a CTA's, with rows of every kind side by side."""
    import torch

    x, t, index, grad = _make(*shape, dtype, 9)
    rows, vocab, top = shape
    index[5::7, top // 2:] = -1      # entries that were not kept, and what sits in them
    t[5::7, top // 2:] = math.nan
    index[3::11, 4:8] = index[3::11, :1]  # one column named five times
    x[2::13, vocab // 2:] = -math.inf     # half the vocabulary masked
    index[2::13] = torch.arange(top, device="cuda")
    x[-1, vocab // 3:] = torch.finfo(x.dtype).min
    index[-1] = torch.arange(top, device="cuda")
    index[0] = vocab                 # nothing kept
    # Where an entry of NaN was kept after all (the steps above meet in some rows), loss and gradient are NaN.
    import neptune_opt_b200 as NB

    bad = ((index >= 0) & (index < vocab) & t.isnan()).any(-1)
    loss, stats = NB.run_distill_loss(x, t, index)
    dx = NB.distill_loss_backward(grad, x, t, index, stats)
    assert bad.any() and torch.equal(loss.isnan(), bad)
    assert dx[bad].isnan().all() and not dx[~bad].isnan().any()
    for first, temperature in ((0, 1.0), (1, 0.7)):
        keep = ~bad[first:]
        ref, bound, _ = _forward_ref(x[first:], t[first:], index[first:], temperature)
        got, stats = NB.run_distill_loss(x[first:], t[first:], index[first:].int(), temperature=temperature)
        assert ((got.double() - ref).abs() <= bound)[keep].all(), f"{shape} loss"
        dx = NB.distill_loss_backward(grad[first:], x[first:], t[first:], index[first:], stats, temperature=temperature)
        rdx, mag = _backward_ref(grad[first:], x[first:], t[first:], index[first:], stats, temperature)
        assert ((dx.double() - rdx).abs() <= UNIT[dtype] * rdx.abs() + 2.0 ** -14 * mag + TINY[dtype])[keep].all(), shape


def test_no_entries_at_all():
    import torch

    import neptune_opt_b200 as NB

    x, t, index, grad = _make(3, 40, 0, "float32", 4)
    loss, stats = NB.run_distill_loss(x, t, index)
    assert not loss.any() and not NB.distill_loss_backward(grad, x, t, index, stats).any()
    assert torch.allclose(stats[:, 0], torch.logsumexp(x, -1), rtol=1e-5)


def test_masked_and_extreme_logits():
    """Vocabulary masked with -inf or the dtype's lowest value, and logits near its largest."""
    import torch

    for dtype in ("float32", "bfloat16", "float16"):
        x, t, index, grad = _make(4, 3000, 8, dtype, 6)
        x[0, 100:] = -math.inf
        x[1, 1000:] = torch.finfo(x.dtype).min
        x[2, :] = -math.inf
        x[2, 17] = 2.0
        index[0] = torch.arange(8)
        index[1] = torch.arange(8)
        index[2] = -1
        index[2, 0] = 17
        x[3, 5] = 30000.0
        index[3, 0] = 5
        index[3, 1:] = -1
        _run_and_check(x, t, index, grad, dtype, label=dtype)


def test_strided_rows_and_teacher_types():
    import torch

    x, t, index, grad = _make(24, 1013, 9, "bfloat16", 2)
    pad = torch.full((24, 1024), math.nan, dtype=x.dtype, device="cuda")
    pad[:, 3:1016] = x
    wide = torch.stack([index, index + 1], -1).flatten(1)[:, ::2]
    view = pad[:, 3:1016].view(2, 12, 1013)
    for tt in (t, t.float(), t.half()):
        _run_and_check(view, tt.view(2, 12, 9), wide.reshape(2, 12, 9), grad.view(2, 12), "bfloat16", label=str(tt.dtype))
    turned = x.t().contiguous().t()  # column-major logits
    _run_and_check(turned, t, index, grad[:1].expand(24), "bfloat16", label="column-major")


def test_autograd_and_differences():
    import torch

    import neptune_opt_b200 as NB

    x, t, index, grad = _make(6, 300, 10, "float32", 3)
    index[2, 4:] = -1
    leaf = x.clone().requires_grad_()
    loss = NB.distill_loss(leaf, t, index, temperature=1.7)
    (loss * grad).sum().backward()
    _, dx = _run_and_check(x, t, index, grad, "float32", 1.7)
    assert torch.equal(leaf.grad, dx)
    d = torch.randn(x.shape, dtype=torch.float64, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    up, down = (_forward_ref(x.double() + s * d, t, index, 1.7)[0] @ grad.double() for s in (1e-6, -1e-6))
    slope, got = (up - down).item() / 2e-6, (dx.double() * d).sum().item()
    assert abs(got - slope) <= 1e-5 * (dx.double() * d).abs().sum().item() + 1e-6


def test_other_stream_and_empty():
    import torch

    import neptune_opt_b200 as NB

    x, t, index, grad = _make(0, 64, 4, "float32", 3)
    loss, stats = NB.run_distill_loss(x, t, index.long())
    assert loss.shape == (0,) and NB.distill_loss_backward(grad, x, t, index.long(), stats).shape == (0, 64)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        _run_and_check(*_make(20, 4000, 8, "bfloat16", 3), "bfloat16", label="stream")
    side.synchronize()
