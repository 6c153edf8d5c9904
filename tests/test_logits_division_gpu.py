"""The logits' divisions, by temperature and repetition penalty, against the formulas in float64.

x / temperature alone is rounded once in fp32: the error before the rounding is below 2^-40 of the value, so the result is at
most half a step (1 + 2^-16) of fp32 from the quotient. 16-bit results are rounded once from an fp32 quotient that is off by at
most 2^-22 of it. Below fp32's normal range an fp32 quotient is off by up to 2^-149.
"""
from __future__ import annotations

import math

import pytest

from conftest import cuda_available

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_available(), reason="needs a CUDA device")]


def half_step(values, dtype):
    """Half the distance between neighbours of `dtype` at each value (float64)."""
    import torch

    info = torch.finfo(dtype)
    exponent = torch.frexp(values.abs().clamp(min=info.smallest_normal))[1].double() - 1
    return torch.ldexp(torch.full_like(exponent, info.eps / 2), exponent)


def logits(rows, vocab, dtype, seed=0):
    import torch

    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(rows, vocab, device="cuda", generator=gen) * 4).to(dtype), gen


def check(got, want, off):
    """Each value within half a step of the quotient, which may itself be off by `off` of it. What is half a step or more above
    the type's largest value rounds to an infinity; just there it may be either."""
    import torch

    largest = torch.tensor(torch.finfo(got.dtype).max, dtype=torch.float64, device=got.device)
    border = largest + half_step(largest, got.dtype)
    over = want.abs() > border * (1 + 2 * off + 2.0 ** -40)
    assert bool((got.double()[over] == torch.sign(want[over]) * math.inf).all())
    rest = want.abs() < border * (1 - 2 * off - 2.0 ** -40)
    tol = half_step(want[rest], got.dtype) * (1 + 2.0 ** -16) + off * want[rest].abs() + 2.0 ** -148
    assert bool(((got.double()[rest] - want[rest]).abs() <= tol).all()), "off by more than one rounding"


@pytest.mark.parametrize("dtype,off", [("float32", 0.0), ("bfloat16", 2.0 ** -22), ("float16", 2.0 ** -22)])
@pytest.mark.parametrize("rows,vocab", [(3, 7), (5, 1003), (40, 16384), (7, 50001)])
def test_a_temperature_is_divided_by(dtype, off, rows, vocab):
    import torch

    import neptune_opt_b200 as NB

    x, gen = logits(rows, vocab, getattr(torch, dtype))
    t = torch.rand(rows, device="cuda", generator=gen) * 3 + 0.1
    check(NB.penalize_logits(x, temperature=t), x.double() / t.double()[:, None], off)


@pytest.mark.parametrize("history", [50, 9000])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_a_repetition_penalty_is_divided_by(dtype, history):
    """x / repetition is rounded to fp32 once, x * repetition too; half a step 2^-24 more before the temperature."""
    import torch

    import neptune_opt_b200 as NB

    x, gen = logits(6, 30011, getattr(torch, dtype), 1)
    tokens = torch.randint(0, 30011, (6, history), device="cuda", generator=gen)
    r = torch.rand(6, device="cuda", generator=gen) + 0.6
    seen = torch.zeros(6, 30011, dtype=torch.bool, device="cuda").scatter_(1, tokens, True)
    penalised = torch.where(x > 0, x.float() / r[:, None], x.float() * r[:, None])  # one rounding
    want = torch.where(seen, penalised, x.float()).double()
    check(NB.penalize_logits(x, tokens, repetition=r), want, 2.0 ** -40)
    t = torch.rand(6, device="cuda", generator=gen) + 0.5
    check(NB.penalize_logits(x, tokens, repetition=r, temperature=t), want / t.double()[:, None],
          0.0 if dtype == "float32" else 2.0 ** -22)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("t", [1e-45, 1e-40, 2.9e-39, 3e-39, 1.1e-38, 1.2e-38, 1e-30, 1e30, 8e37, 9e37, 3.4e38])
def test_temperatures_at_the_ends_of_fp32(dtype, t):
    """No logit of 0 and none of -inf becomes NaN, whatever the reciprocal; where fp32 holds that (from 2^-128 = 2.94e-39 on;
    below its normal range to 2^-149, 2^-21 of it) the others are the quotients."""
    import torch

    import neptune_opt_b200 as NB

    dt = getattr(torch, dtype)
    x, _ = logits(2, 4099, dt, 2)
    x[:, ::3] = 0.0
    x[:, 1::7] = torch.finfo(dt).tiny
    x[0, 5], x[1, 6] = -math.inf, torch.finfo(dt).max
    temperature = torch.full((2,), t, device="cuda")
    want = x.double() / temperature.double()[:, None]
    got = NB.penalize_logits(x, temperature=temperature)
    assert not bool(torch.isnan(got).any()) and float(got[0, 5]) == -math.inf
    assert torch.equal(torch.sign(got[:, :1]), torch.zeros_like(got[:, :1])) and bool((got * x >= 0)[x.abs() < math.inf].all())
    if t > 2.0 ** -128:
        check(got, want, 2.0 ** -20)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_an_infinite_divisor_leaves_nothing(dtype):
    """x / inf is 0 for every number x, by temperature and by repetition penalty."""
    import torch

    import neptune_opt_b200 as NB

    x, gen = logits(3, 5003, getattr(torch, dtype), 3)
    endless = torch.full((3,), math.inf, device="cuda")
    assert not bool(NB.penalize_logits(x, temperature=endless).any())
    for history in (40, 9000):
        tokens = torch.randint(0, 5003, (3, history), device="cuda", generator=gen)
        seen = torch.zeros(3, 5003, dtype=torch.bool, device="cuda").scatter_(1, tokens, True)
        got = NB.penalize_logits(x, tokens, repetition=endless)
        want = torch.where(seen, torch.where(x > 0, 0.0, x.float() * math.inf), x.float()).to(x.dtype)
        assert torch.equal(got.nan_to_num(nan=-7.0), want.nan_to_num(nan=-7.0))
