"""The serving operators together: examples/decode_batch.py's step against the same step in plain torch operations, and
captured and replayed against eager steps; and in exported and compiled graphs and packages."""
from __future__ import annotations

import importlib.util
import math
import os

import pytest

from conftest import ROOT, cuda_available

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_available(), reason="needs a CUDA device")]


def _example():
    spec = importlib.util.spec_from_file_location("decode_batch", os.path.join(ROOT, "examples", "decode_batch.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _plain_norm8(x, w, residual=None):
    import torch

    y = x.float() if residual is None else x.float() + residual.float()
    h = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * w.float()
    scale = h.abs().amax(-1, keepdim=True) / 448
    return ((h / scale).to(torch.float8_e4m3fn).float() * scale).to(x.dtype)


def _plain_step(m):
    """The penalised logits of one step, in float64 between the step's own roundings."""
    import torch

    b = m.tokens.shape[0]
    rows, last = torch.arange(b, device="cuda"), (m.lens - 1).long()
    x = m.stream(m.tokens[rows, last])
    q, k, v = m.project(_plain_norm8(x, m.first))
    ck, cv = m.k.clone(), m.v.clone()
    ck[rows, :, last], cv[rows, :, last] = k, v
    o = torch.empty(b, m.heads, m.dim, dtype=torch.float64, device="cuda")
    for i in range(b):
        n = int(m.lens[i])
        for h in range(m.heads):
            g = h // (m.heads // m.kv_heads)
            kk, vv = torch.cat([m.prefix_k[g], ck[i, g, :n]]).double(), torch.cat([m.prefix_v[g], cv[i, g, :n]]).double()
            o[i, h] = torch.softmax(kk @ q[i, h].double() / math.sqrt(m.dim), -1) @ vv
    y = o.to(x.dtype).reshape(b, -1) @ m.out.t()
    z = (_plain_norm8(y, m.second, x) @ m.head.t()).double()
    for i in range(b):
        history = m.tokens[i, :m.lens[i]]
        output = history[m.prompt_lens[i]:]
        for t in history.unique():
            z[i, t] = z[i, t] / 1.2 if z[i, t] > 0 else z[i, t] * 1.2
        for t in output:
            z[i, t] -= 0.3
    z /= 0.8
    token = torch.arange(m.vocab, device="cuda")
    return z.masked_fill(((m.allowed[:, token // 32] >> (token % 32)) & 1) == 0, -math.inf)


@pytest.mark.parametrize("sizes", [{}, {"batch": 12, "heads": 6, "kv_heads": 1, "prompt": 900, "dim": 64, "width": 200}])
def test_steps_agree_with_plain_operations(sizes):
    """Logits step by step from the same state. Between the operators values are rounded to bf16 (2^-8 each, five times on
    the way) and to e4m3 by both sides alike; where fp32 sums in another order land on the other side of a border, a value
    moves by a step. Probabilities rounded to bf16 for the product move o by 2^-8 of its terms. Together about
    sqrt(7) 2^-8 = 1% of the logits' norm; 3% bounds it."""
    import torch

    with torch.no_grad():
        m = _example().Decoder(room=20, **sizes)
        for _ in range(6):
            want = _plain_step(m)
            got, p = m.step()
            shut = torch.isinf(want)
            assert torch.equal(torch.isinf(got), shut)
            assert (got.double() - want)[~shut].norm() <= 0.03 * want[~shut].norm()
            assert torch.allclose(p.sum(-1), torch.ones_like(p[:, 0]), atol=1e-5) and not p[shut].any()


def test_replayed_steps_are_the_eager_ones():
    import torch

    module = _example()
    with torch.no_grad():
        m = module.Decoder(room=16)
        for _ in range(16):
            m.step()
    assert torch.equal(module.decode(16), m.tokens)
    assert bool((m.tokens >= 0).all()) and bool((m.tokens[1::2, 1:] < m.vocab // 2).all())


def _module():
    import torch

    import neptune_opt_b200 as NB

    class Step(torch.nn.Module):
        def forward(self, q, pk, pv, k, v, lens, x, w, z, tokens, rep, allowed):
            o, lse = NB.prefix_attention(q, pk, pv, k, v, lens, return_lse=True)
            q8, scale, y = NB.quantized_rms_norm(x, w, x, group=64)
            i8, s8, _ = NB.quantized_rms_norm(x, w, dtype=torch.int8)
            return o, lse, q8.float(), scale, y, i8, s8, NB.penalize_logits(z, tokens, lens, repetition=rep, allowed=allowed)

    gen = torch.Generator(device="cuda").manual_seed(4)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=gen).to(torch.bfloat16)

    args = (normal(3, 4, 1, 128), normal(2, 200, 128), normal(2, 200, 128), normal(3, 2, 40, 128), normal(3, 2, 40, 128),
            torch.tensor([40, 0, 7], dtype=torch.int32, device="cuda"), normal(3, 256), normal(256), normal(3, 1001),
            torch.randint(0, 1001, (3, 40), device="cuda", generator=gen), torch.rand(3, device="cuda", generator=gen) + 1,
            torch.randint(-2 ** 31, 2 ** 31, (3, 32), device="cuda", generator=gen).to(torch.int32))
    return Step(), args


def _same(got, want):
    import torch

    assert len(got) == len(want)
    for a, b in zip(got, want):
        assert a.dtype == b.dtype and torch.equal(a, b)


def test_exported_and_compiled():
    import torch

    step, args = _module()
    want = step(*args)
    _same(torch.export.export(step, args).module()(*args), want)
    _same(torch.compile(step, fullgraph=True)(*args), want)


def test_packaged(tmp_path):
    import torch

    import neptune_opt_b200.aot as aot

    step, args = _module()
    aot.load()
    pkg = aot.compile_package(torch.export.export(step, args), str(tmp_path / "step.pt2"))
    _same(torch._inductor.aoti_load_package(pkg)(*args), step(*args))


def test_a_stream_behind_another():
    """Steps whose inputs another stream has just written."""
    import torch

    import neptune_opt_b200 as NB

    step, args = _module()
    want = step(*args)
    side = torch.cuda.Stream()
    for _ in range(10):
        fresh = [torch.empty_like(a) for a in args]
        for f, a in zip(fresh, args):
            f.copy_(a)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = step(*fresh)
        torch.cuda.current_stream().wait_stream(side)
        _same(got, want)
    assert NB.launch_count() > 0


def test_refusals_on_the_gpu():
    import torch

    import neptune_opt_b200 as NB

    step, args = _module()
    q, pk, pv, k, v, lens, x, w, z, tokens, rep, allowed = args
    for call, error in ((lambda: NB.prefix_attention(q.float(), pk, pv, k, v), TypeError),
                        (lambda: NB.prefix_attention(q, pk[:, :5], pv, k, v), ValueError),
                        (lambda: NB.prefix_attention(q, pk, pv, k, v, lens.cpu()), ValueError),
                        (lambda: NB.prefix_attention(q, pk, pv, k, v, lens.long()), TypeError),
                        (lambda: NB.prefix_attention(q, pk, pv, k, v, scale=0.0), ValueError),
                        (lambda: NB.prefix_attention(q[..., :96], pk[..., :96], pv[..., :96], k[..., :96], v[..., :96]),
                         NotImplementedError),
                        (lambda: NB.quantized_rms_norm(x, w.float()), TypeError),
                        (lambda: NB.quantized_rms_norm(x, w, x[:2]), ValueError),
                        (lambda: NB.quantized_rms_norm(x, w, group=0), ValueError),
                        (lambda: NB.quantized_rms_norm(x, w, group=96), ValueError),
                        (lambda: NB.quantized_rms_norm(x, w, dtype=torch.uint8), TypeError),
                        (lambda: NB.quantized_rms_norm(x, w, eps=0.0), ValueError),
                        (lambda: NB.quantized_rms_norm(x.requires_grad_(), w), NotImplementedError),
                        (lambda: NB.penalize_logits(z, repetition=rep), ValueError),
                        (lambda: NB.penalize_logits(z, tokens.float()), TypeError),
                        (lambda: NB.penalize_logits(z, tokens, repetition=rep.cpu()), ValueError),
                        (lambda: NB.penalize_logits(z, allowed=allowed[:, :31]), ValueError),
                        (lambda: NB.penalize_logits(z[0]), ValueError)):
        with pytest.raises(error):
            call()
