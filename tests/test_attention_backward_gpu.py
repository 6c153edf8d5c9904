"""GPU parity of attention's backward pass, and of the forward pass with shared heads, lengths and
strides, against the formulas in float64.

Tolerances. The kernel may round P and dS to bf16 (relative 2^-9) before the products that sum them, the
sums are fp32, and each result is rounded once to bf16 (2^-9; 2^-8 leaves room for the fp32 steps).
P itself is off by its exponent's error, at most 2^-22 (sum |q k| scale + |lse|) < 2^-13 here, dP and delta
by 2^-18 of their sums of magnitudes. So, elementwise and with every sum over magnitudes:
  |dv - ref| <= (2^-9 + 2^-13) P^T |dO| + 2^-8 |ref|
  |dS - ref| <= (2^-9 + 2^-13) |dS| + 2^-18 P (|dO| |V|^T + |dO| |O|)     =: E
  |dq - ref| <= scale E |K| + 2^-8 |ref|,   |dk - ref| <= scale E^T |Q| + 2^-8 |ref|
"""
from __future__ import annotations

import math

import pytest

from conftest import cuda_available

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_available(), reason="needs a CUDA device")]

D = 128


def _make(shape, seed, layout="bhsd"):
    """q, k, v, grad_out [B, H, S, D] in bf16; "bshd" and "packed" are the views a projection leaves."""
    import torch

    b, h, hk, n = shape
    gen = torch.Generator().manual_seed(seed)

    def one(heads):
        if layout == "bshd":
            return torch.randn(b, n, heads, D, generator=gen).to(torch.bfloat16).cuda().transpose(1, 2)
        if layout == "odd":  # neither the base nor the row stride is a multiple of 16 bytes
            flat = torch.randn(b * heads * n * 131 + 1, generator=gen).to(torch.bfloat16).cuda()
            return flat[1:].view(b, heads, n, 131)[..., :D]
        return torch.randn(b, heads, n, D, generator=gen).to(torch.bfloat16).cuda()

    if layout == "packed":
        both = torch.randn(b, n, h + 2 * hk, D, generator=gen).to(torch.bfloat16).cuda().transpose(1, 2)
        return both[:, :h], both[:, h:h + hk], both[:, h + hk:], one(h)
    return one(h), one(hk), one(hk), one(h)


def _visible(n, length, causal):
    import torch

    pos = torch.arange(n, device="cuda")
    ok = (pos[None, :] < length) & (pos[:, None] < length)
    return ok & (pos[None, :] <= pos[:, None]) if causal else ok


def _forward_ref(q, k, v, ok, scale):
    """Float64 O and LSE of one head; rows that see nothing read 0 and -inf."""
    import torch

    # masked rows may hold anything: take them out before they reach a product
    rows, cols = ok.any(1), ok.any(0)
    q, k, v = (torch.where(m[:, None], t.double(), 0.0) for m, t in ((rows, q), (cols, k), (cols, v)))
    s = (q @ k.T * scale).masked_fill(~ok, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.where(ok, torch.exp(s - torch.where(rows, lse, 0.0)[:, None]), 0.0)
    return p @ v, lse


def _backward_ref(q, k, v, o, lse, g, ok, scale):
    """((value, bound) of dq, dk, dv) of one query head in float64."""
    import torch

    rows, cols = ok.any(1), ok.any(0)
    q, o, g = (torch.where(rows[:, None], t.double(), 0.0) for t in (q, o, g))
    k, v = (torch.where(cols[:, None], t.double(), 0.0) for t in (k, v))
    p = torch.where(ok, torch.exp(q @ k.T * scale - torch.where(rows, lse.double(), 0.0)[:, None]), 0.0)
    delta = (g * o).sum(-1, keepdim=True)
    ds = p * (g @ v.T - delta)
    e = (2.0 ** -9 + 2.0 ** -13) * ds.abs() + 2.0 ** -18 * p * (g.abs() @ v.abs().T + (g * o).abs().sum(-1, keepdim=True))
    dq, dk, dv = ds @ k * scale, ds.T @ q * scale, p.T @ g
    return ((dq, e @ k.abs() * scale), (dk, e.T @ q.abs() * scale),
            (dv, (2.0 ** -9 + 2.0 ** -13) * (p.T @ g.abs())))


def _check(got, ref, bound, label):
    import torch

    assert torch.isfinite(got.float()).all(), f"{label}: non-finite values"
    over = (got.double() - ref).abs() - (bound + 2.0 ** -8 * ref.abs() + 1e-30)
    assert over.max().item() <= 0, f"{label}: exceeds the bound by {over.max().item():.3g} at {over.argmax().item()}"


def _check_all(q, k, v, o, lse, g, grads, lens, causal, scale, label):
    import torch

    b, h, n, _ = q.shape
    per = h // k.shape[1]
    for i in range(b):
        ok = _visible(n, int(lens[i]), causal)
        for j in range(k.shape[1]):
            sums = [torch.zeros(n, D, dtype=torch.float64, device="cuda") for _ in range(4)]
            for hh in range(j * per, (j + 1) * per):
                (dq, bq), (dk, bk), (dv, bv) = _backward_ref(q[i, hh], k[i, j], v[i, j], o[i, hh], lse[i, hh],
                                                             g[i, hh], ok, scale)
                _check(grads[0][i, hh], dq, bq, f"{label} dq ({i},{hh})")
                for t, add in zip(sums, (dk, bk, dv, bv)):
                    t += add
            _check(grads[1][i, j], sums[0], sums[1], f"{label} dk ({i},{j})")
            _check(grads[2][i, j], sums[2], sums[3], f"{label} dv ({i},{j})")


def _check_forward(q, k, v, o, lse, lens, causal, scale, label):
    import torch

    per = q.shape[1] // k.shape[1]
    for i in range(q.shape[0]):
        n = int(lens[i])
        ok = _visible(q.shape[2], n, causal)
        for hh in range(q.shape[1]):
            ro, rl = _forward_ref(q[i, hh], k[i, hh // per], v[i, hh // per], ok, scale)
            top = v[i, hh // per, :n].double().abs().max().item() if n else 0.0
            _check(o[i, hh], ro, 2.0 ** -9 * top, f"{label} o ({i},{hh})")
            assert torch.equal(lse[i, hh] == -math.inf, rl == -math.inf), f"{label} lse ({i},{hh})"
            fin = rl != -math.inf
            assert ((lse[i, hh].double() - rl).abs() <= 2e-5 * (1 + rl.abs()))[fin].all(), f"{label} lse ({i},{hh})"


def _lens_of(lens, b, n):
    import torch

    return None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")


SHAPES = [(1, 1, 1, 1), (1, 2, 1, 2), (2, 2, 2, 63), (1, 4, 2, 64), (1, 3, 1, 65), (1, 2, 2, 127), (2, 2, 1, 128),
          (1, 2, 2, 129), (1, 1, 1, 255), (1, 6, 2, 257), (1, 2, 1, 500), (1, 1, 1, 1025)]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_gradients_match_the_formulas(shape, causal):
    import torch

    import neptune_opt_b200 as NB

    q, k, v, g = _make(shape, 11 + shape[3])
    keep = [t.clone() for t in (q, k, v, g)]
    o, lse = NB.attention(q, k, v, causal=causal, return_lse=True)
    lens = [shape[3]] * shape[0]
    scale = 1.0 / math.sqrt(D)
    _check_forward(q, k, v, o, lse, lens, causal, scale, f"{shape} {causal}")
    grads = NB.attention_backward(q, k, v, o, lse, g, causal=causal)
    _check_all(q, k, v, o, lse, g, grads, lens, causal, scale, f"{shape} {causal}")
    again = NB.attention_backward(q, k, v, o, lse, g, causal=causal)
    assert all(torch.equal(a, c) for a, c in zip(grads, again)), "the result depends on scheduling"
    assert all(torch.equal(a, c) for a, c in zip((q, k, v, g), keep)), "inputs were modified"
    assert NB._lib.stream_fault() == 0


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("n,lens", [(200, [200, 0, 1, 199]), (300, [128, 129, 127, 300]), (64, [63, 64, 1, 0]),
                                    (520, [256, 257, 65, 511])])
def test_lengths_mask_whatever_the_padding_holds(n, lens, causal):
    """Tokens past a length hold NaN and infinities in q, k, v, o, grad_out and lse."""
    import torch

    import neptune_opt_b200 as NB

    q, k, v, g = _make((4, 4, 2, n), 5 + n)
    for i, m in enumerate(lens):
        for t, bad in ((q, math.nan), (k, math.inf), (v, math.nan), (g, -math.inf)):
            t[i, :, m:] = bad
    dev = _lens_of(lens, 4, n)
    scale = 0.1
    o, lse = NB.attention(q, k, v, causal=causal, scale=scale, return_lse=True, seq_lens=dev)
    _check_forward(q, k, v, o, lse, lens, causal, scale, f"{n} {lens}")
    for i, m in enumerate(lens):
        assert not o[i, :, m:].any()
        o[i, :, m:] = math.nan
        lse[i, :, m:] = math.nan
    grads = NB.attention_backward(q, k, v, o, lse, g, causal=causal, scale=scale, seq_lens=dev)
    _check_all(q, k, v, o, lse, g, grads, lens, causal, scale, f"{n} {lens}")
    for t in grads:
        for i, m in enumerate(lens):
            assert not t[i, :, m:].any(), "gradients of masked tokens are not zero"
    assert NB._lib.stream_fault() == 0


@pytest.mark.parametrize("layout", ["bshd", "packed", "odd"])
def test_strided_inputs(layout):
    import torch

    import neptune_opt_b200 as NB

    shape = (2, 4, 2, 150)
    q, k, v, g = _make(shape, 3, layout)
    scale = 1.0 / math.sqrt(D)
    o, lse = NB.attention(q, k, v, causal=True, return_lse=True)
    _check_forward(q, k, v, o, lse, [150, 150], True, scale, layout)
    grads = NB.attention_backward(q, k, v, o, lse, g, causal=True)
    _check_all(q, k, v, o, lse, g, grads, [150, 150], True, scale, layout)
    dense = NB.attention_backward(*(t.contiguous() for t in (q, k, v, o)), lse, g.contiguous(), causal=True)
    assert all(torch.equal(a, c) for a, c in zip(grads, dense)), "the result depends on the layout"


def test_expanded_gradient_and_key_value():
    """grad_out of a sum (stride 0 everywhere) and one key/value sequence expanded over the batch."""
    import torch

    import neptune_opt_b200 as NB

    q, k, v, _ = _make((3, 2, 2, 70), 9)
    k, v = k[:1].expand(3, 2, 70, D), v[:1].expand(3, 2, 70, D)
    g = torch.ones((), dtype=torch.bfloat16, device="cuda").expand(3, 2, 70, D)
    o, lse = NB.attention(q, k, v, return_lse=True)
    grads = NB.attention_backward(q, k, v, o, lse, g)
    _check_all(q, k, v, o, lse, g, grads, [70] * 3, False, 1.0 / math.sqrt(D), "expanded")


def test_probabilities_far_from_one():
    """Scores that span +-300: most probabilities vanish, a few rows are one-hot."""
    import neptune_opt_b200 as NB

    q, k, v, g = _make((1, 2, 1, 333), 21)
    o, lse = NB.attention(q, k, v, causal=True, scale=8.0, return_lse=True)
    grads = NB.attention_backward(q, k, v, o, lse, g, causal=True, scale=8.0)
    for t in grads:
        assert t.float().isfinite().all()
    # 2^-13 on P holds while 2^-22 (scale sum |q k| + |lse|) does; here that sum reaches 2^11.
    import torch

    ok = _visible(333, 333, True)
    (dq, bq), _, _ = _backward_ref(q[0, 0], k[0, 0], v[0, 0], o[0, 0], lse[0, 0], g[0, 0], ok, 8.0)
    over = (grads[0][0, 0].double() - dq).abs() - (4 * bq + 2.0 ** -8 * dq.abs())
    assert over.max().item() <= 0
    assert torch.isfinite(lse).all()


def test_autograd_gives_the_same_gradients_and_agrees_with_differences():
    import torch

    import neptune_opt_b200 as NB

    q, k, v, g = _make((1, 4, 2, 90), 17)
    lens = torch.tensor([77], dtype=torch.int32, device="cuda")
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    o = NB.attention(*leaves, causal=True, seq_lens=lens)
    o.backward(g)
    o2, lse = NB.attention(q, k, v, causal=True, seq_lens=lens, return_lse=True)
    assert not o2.requires_grad and torch.equal(o, o2)
    direct = NB.attention_backward(q, k, v, o2, lse, g, causal=True, seq_lens=lens)
    assert all(torch.equal(t.grad, d) for t, d in zip(leaves, direct))
    # Central differences of the float64 definition along a random direction of each input.
    ok, scale = _visible(90, 77, True), 1.0 / math.sqrt(D)

    def value(q, k, v):
        return sum((_forward_ref(q[0, h], k[0, h // 2], v[0, h // 2], ok, scale)[0] * g[0, h].double()).sum()
                   for h in range(4))

    gen = torch.Generator(device="cuda").manual_seed(4)
    base = [t.double() for t in (q, k, v)]
    for i, grad in enumerate(direct):
        d = torch.randn(base[i].shape, dtype=torch.float64, device="cuda", generator=gen)
        up, down = list(base), list(base)
        up[i], down[i] = base[i] + 1e-5 * d, base[i] - 1e-5 * d
        slope = (value(*up) - value(*down)).item() / 2e-5
        got = (grad.double() * d).sum().item()
        # Independent roundings of relative size 2^-8 per element, six standard deviations; delta comes
        # from the bf16 o, which moves dS by 2^-9 |delta| p coherently over a row.
        tol = 6 * 2.0 ** -8 * (grad.double() * d).norm().item() + 2.0 ** -9 * (grad.double() * d).abs().sum().item()
        assert abs(got - slope) <= tol, (i, got, slope, tol)


def test_other_stream_and_empty():
    import torch

    import neptune_opt_b200 as NB

    q, k, v, g = _make((1, 2, 2, 140), 2)
    o, lse = NB.attention(q, k, v, return_lse=True)
    want = NB.attention_backward(q, k, v, o, lse, g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = NB.attention_backward(q, k, v, o, lse, g)
    side.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    none = torch.empty(0, 2, 5, D, dtype=torch.bfloat16, device="cuda")
    out = NB.attention_backward(none, none, none, none, torch.empty(0, 2, 5, device="cuda"), none)
    assert [t.shape for t in out] == [none.shape] * 3


@pytest.mark.parametrize("lens", [[100, 2000], [1, 0], [129, 1]])
def test_parts_without_steps(lens):
    """A long tensor with short sequences: key blocks are cut into more parts than they have steps."""
    import torch

    import neptune_opt_b200 as NB

    for shape, causal in (((2, 1, 1, 2000), False), ((2, 4, 1, 2000), True)):
        q, k, v, g = _make(shape, 77)
        dev = _lens_of(lens, 2, 2000)
        o, lse = NB.attention(q, k, v, causal=causal, return_lse=True, seq_lens=dev)
        grads = NB.attention_backward(q, k, v, o, lse, g, causal=causal, seq_lens=dev)
        _check_all(q, k, v, o, lse, g, grads, lens, causal, 1.0 / math.sqrt(D), f"{shape} {lens}")
        again = NB.attention_backward(q, k, v, o, lse, g, causal=causal, seq_lens=dev)
        assert all(torch.equal(a, c) for a, c in zip(grads, again))
