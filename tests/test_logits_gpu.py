"""GPU parity of the logits' penalties, biases, temperature and mask against the formulas in float64.

Tolerance, elementwise: seven fp32 steps, each off by at most 2^-24 of the magnitudes it joins, so 8 * 2^-24 of
(|x| + frequency count + presence + sum |bias|) / temperature (|x| after its repetition penalty), and half a step
of the type of the result. Forbidden tokens are -inf, and nothing else is.
"""
from __future__ import annotations

import math

import pytest

from conftest import cuda_available

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_available(), reason="needs a CUDA device")]

HALF_STEP = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}


def make(rows, vocab, dtype="float32", history=0, biases=0, masked=False, index="int64", seed=0):
    import torch

    gen = torch.Generator().manual_seed(seed)
    s = {"logits": (torch.randn(rows, vocab, generator=gen) * 4).to(getattr(torch, dtype)),
         "temperature": torch.rand(rows, generator=gen) + 0.3}
    if history:
        it = getattr(torch, index)
        # Few different tokens, so that they repeat; some outside the vocabulary.
        s["tokens"] = (torch.rand(rows, history, generator=gen) ** 3 * (vocab + 3) - 1).floor().to(it)
        s["token_lens"] = torch.randint(0, history + 1, (rows,), generator=gen, dtype=torch.int32)
        s["prompt_lens"] = torch.randint(0, history + 1, (rows,), generator=gen, dtype=torch.int32)
        s["token_lens"][0] = history
        s["repetition"] = torch.rand(rows, generator=gen) + 0.7
        s["presence"] = torch.rand(rows, generator=gen) * 2 - 1
        s["frequency"] = torch.rand(rows, generator=gen) - 0.3
    if biases:
        s["bias_index"] = torch.randint(-2, vocab + 2, (rows, biases), generator=gen).to(getattr(torch, index))
        s["bias_value"] = torch.randn(rows, biases, generator=gen) * 5
    if masked:
        s["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (rows, -(-vocab // 32)), generator=gen).to(torch.int32)
        s["allowed"][rows // 2] = 0
        s["allowed"][0] = -1
    return {k: v.cuda() for k, v in s.items()}


def reference(s):
    """(values, tolerance), row by row in float64 from Python lists."""
    import torch

    x = s["logits"].double()
    rows, vocab = x.shape
    mag = x.abs()
    for r in range(rows):
        if s.get("tokens") is not None:
            tokens = s["tokens"][r]
            n = len(tokens) if s.get("token_lens") is None else max(0, min(len(tokens), int(s["token_lens"][r])))
            p = 0 if s.get("prompt_lens") is None else max(0, min(n, int(s["prompt_lens"][r])))
            ok = lambda t: t[(t >= 0) & (t < vocab)].long()  # noqa: E731
            seen = torch.unique(ok(tokens[:n]))
            if s.get("repetition") is not None:
                f = s["repetition"][r].double()
                x[r, seen] = torch.where(x[r, seen] > 0, x[r, seen] / f, x[r, seen] * f)
            mag[r] = x[r].abs()
            token, count = torch.unique(ok(tokens[p:n]), return_counts=True)
            f = 0.0 if s.get("frequency") is None else s["frequency"][r].double()
            q = 0.0 if s.get("presence") is None else s["presence"][r].double()
            x[r, token] -= f * count + q
            mag[r, token] += abs(f) * count + abs(q)
        if s.get("bias_index") is not None:
            i, b = s["bias_index"][r].long(), s["bias_value"][r].double()
            keep = (i >= 0) & (i < vocab)
            x[r].index_add_(0, i[keep], b[keep])
            mag[r].index_add_(0, i[keep], b[keep].abs() * max(1, int(keep.sum()) // 64))
        if s.get("temperature") is not None:
            x[r] /= s["temperature"][r].double()
            mag[r] /= s["temperature"][r].double().abs()
        if s.get("allowed") is not None:
            v = torch.arange(vocab, device="cuda")
            bit = (s["allowed"][r].long()[v // 32] >> (v % 32)) & 1
            x[r].masked_fill_(bit == 0, -math.inf)
    return x, mag


def check(s, got=None):
    import torch

    import neptune_opt_b200 as NB

    before = {k: v.clone() for k, v in s.items() if v is not None}
    out = NB.penalize_logits(**s) if got is None else got
    for k, v in before.items():
        assert torch.equal(torch.nan_to_num(v), torch.nan_to_num(s[k])), f"{k} was written"
    assert out.dtype == s["logits"].dtype and out.shape == s["logits"].shape and out.is_contiguous()
    want, mag = reference(s)
    shut = torch.isinf(want)
    assert torch.equal(torch.isinf(out), shut) and bool((out[shut].float() == want[shut].float()).all())
    off = (out.double() - want).abs()
    tol = 8 * 2.0 ** -24 * mag + HALF_STEP[str(out.dtype)[6:]] * want.abs() + 2.0 ** -25
    assert bool((off <= tol)[~shut].all()), f"off by up to {(off / tol)[~shut].amax():.3f} of the bound"
    return out


@pytest.mark.parametrize("dtype", list(HALF_STEP))
@pytest.mark.parametrize("vocab", [1, 7, 31, 32, 33, 1000, 4096, 5003, 16384, 16391, 50001])
@pytest.mark.parametrize("history,biases,masked", [(0, 0, False), (0, 0, True), (60, 0, False), (0, 9, True), (200, 40, True),
                                                    (700, 200, True)])
def test_against_the_formulas(dtype, vocab, history, biases, masked):
    check(make(5, vocab, dtype, history, biases, masked, seed=vocab))


@pytest.mark.parametrize("dtype", list(HALF_STEP))
@pytest.mark.parametrize("vocab", [1, 33, 1000, 5003, 16391, 50001])
@pytest.mark.parametrize("history,biases", [(40, 257), (700, 300), (4096, 1024), (4097, 3), (9000, 600)])
def test_histories_and_biases_that_the_sweep_does_not_count(dtype, vocab, history, biases):
    check(make(3, vocab, dtype, history, biases, True, seed=vocab + history))


@pytest.mark.parametrize("dtype", list(HALF_STEP))
@pytest.mark.parametrize("history,biases", [(0, 7), (300, 0), (2049, 100), (4096, 256)])
def test_few_and_many_rows_agree(dtype, history, biases):
    """Few tiles count the history themselves, many take it from the names' kernel; rows of other boundaries, too."""
    import torch

    import neptune_opt_b200 as NB

    s = make(220, 40009, dtype, history, biases, True, seed=history)
    want = NB.penalize_logits(**s)
    check({k: v[:5] for k, v in s.items()}, want[:5])
    for lo, hi in ((0, 1), (1, 30), (30, 90)):
        assert torch.equal(NB.penalize_logits(**{k: v[lo:hi] for k, v in s.items()}), want[lo:hi])
    for at, width in ((0, 40064), (3, 40013), (8, 40017)):
        room = torch.full((220, width), math.nan, device="cuda", dtype=s["logits"].dtype)
        room[:, at:at + 40009] = s["logits"]
        assert torch.equal(NB.penalize_logits(**{**s, "logits": room[:, at:at + 40009]}), want)


@pytest.mark.parametrize("index", ["int32", "int64"])
@pytest.mark.parametrize("rows", [1, 2, 97, 700])
def test_row_counts_and_index_types(index, rows):
    check(make(rows, 2053, "bfloat16", 33, 5, True, index, seed=rows))


def test_wide_rows_in_many_chunks():
    check(make(2, 262144, "bfloat16", 5000, 300, True))
    check(make(3, 131075, "float16", 1, 1, True))


def test_each_part_alone():
    full = make(4, 999, "float32", 50, 6, True)
    for keep in (("temperature",), ("tokens", "repetition"), ("tokens", "token_lens", "presence"),
                 ("tokens", "prompt_lens", "frequency"), ("tokens", "token_lens", "prompt_lens"), ("tokens",),
                 ("bias_index", "bias_value"), ("allowed",), ()):
        check({"logits": full["logits"], **{k: full[k] for k in keep}})


def test_lengths_at_their_ends():
    import torch

    s = make(6, 100, "float32", 40)
    s["token_lens"] = torch.tensor([0, 1, 40, 99, -3, 20], dtype=torch.int32, device="cuda")
    s["prompt_lens"] = torch.tensor([0, 1, 0, 40, 5, -7], dtype=torch.int32, device="cuda")
    check(s)


def test_a_token_that_comes_again_and_again():
    import torch

    s = make(2, 70000, "float32", 100000)
    s["tokens"].fill_(69999)
    s["prompt_lens"].zero_()
    s["token_lens"].fill_(100000)
    s["frequency"].fill_(0.001)
    check(s)
    s["prompt_lens"].fill_(99999)  # once in the output, the others in the prompt
    check(s)
    s["prompt_lens"].fill_(100000)
    check(s)
    assert s["tokens"].dtype == torch.int64


def test_biases_that_name_a_token_again():
    import torch

    s = make(3, 500, "float32", 0, 1024)
    s["bias_index"] = torch.randint(0, 4, (3, 1024), device="cuda") * 166
    s["bias_value"] = torch.randn(3, 1024, device="cuda")
    first = check(s)
    import neptune_opt_b200 as NB

    for _ in range(3):
        assert torch.equal(NB.penalize_logits(**s), first)
    s["bias_value"][:, 5] = -math.inf  # a token that is ruled out by its bias
    out = NB.penalize_logits(**s)
    assert bool((out.gather(1, s["bias_index"][:, 5:6]) == -math.inf).all()) and int(torch.isinf(out).sum()) == 3


def test_infinities_and_nan():
    """-inf stays where it is whatever the penalties, NaN stays unless it is forbidden, and a row may allow nothing."""
    import torch

    import neptune_opt_b200 as NB

    for dtype in HALF_STEP:
        s = make(4, 800, dtype, 30, 4, True)
        lowest = torch.finfo(s["logits"].dtype).min
        s["logits"][:, ::5] = -math.inf
        s["logits"][:, 1::5] = lowest
        s["logits"][1, 3] = math.nan
        s["temperature"].fill_(2.0)
        s["allowed"][1, 0] |= 8
        out = NB.penalize_logits(**s)
        assert bool((out[:, ::5] == -math.inf).all()) and bool(torch.isnan(out[1, 3]))
        assert int(torch.isnan(out).sum()) == 1
        assert bool((out[2] == -math.inf).all())
        s["allowed"][1, 0] &= ~8
        assert not bool(torch.isnan(NB.penalize_logits(**s)).any())


def test_layouts():
    """Rows of a wider buffer, transposed logits, bases off the 16-byte boundary, parameters with strides, one mask
    and one history for all rows."""
    import torch

    import neptune_opt_b200 as NB

    for dtype in HALF_STEP:
        s = make(6, 1003, dtype, 20, 5, True)
        want = check(s)

        def same(**changes):
            assert torch.equal(NB.penalize_logits(**{**s, **changes}), want)

        for width, at in ((1003 + 13, 5), (1024, 0), (1024, 8), (2000, 997)):
            room = torch.full((6, width), math.nan, device="cuda", dtype=s["logits"].dtype)
            room[:, at:at + 1003] = s["logits"]
            same(logits=room[:, at:at + 1003])
        same(logits=s["logits"].t().contiguous().t())
        same(tokens=torch.cat([s["tokens"], s["tokens"]], 1)[:, :20], allowed=s["allowed"].t().contiguous().t(),
             temperature=torch.stack([s["temperature"]] * 2, 1)[:, 0], token_lens=torch.stack([s["token_lens"]] * 2, 1)[:, 0],
             bias_value=torch.cat([s["bias_value"]] * 2, 1)[:, :5])
        one = {**s, "allowed": s["allowed"][1:2].expand(6, -1), "tokens": s["tokens"][:1].expand(6, -1),
               "bias_index": s["bias_index"][:1].expand(6, -1)}
        check(one)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("vocab,rows,history", [(1, 9, 0), (5, 9, 4), (15, 9, 4), (17, 9, 0), (23, 9, 4), (1003, 9, 40),
                                                (1003, 9, 600), (8199, 9, 600), (16401, 3, 0), (16401, 3, 40),
                                                (16401, 3, 600)])
def test_rows_cut_differently_than_the_output(dtype, vocab, rows, history):
    """Every pair of places behind a 16-byte boundary, the first and the last row at the ends of their memory, NaN
    between the rows: bit for bit what contiguous logits give."""
    import torch

    import neptune_opt_b200 as NB

    gen = torch.Generator(device="cuda").manual_seed(vocab + history)
    x = torch.randn(rows, vocab, device="cuda", generator=gen).to(getattr(torch, dtype))
    given = {"temperature": torch.rand(rows, device="cuda", generator=gen) + 0.5,
             "allowed": torch.randint(-2 ** 31, 2 ** 31, (rows, -(-vocab // 32)), device="cuda", generator=gen).int()}
    if history:
        given |= {"tokens": torch.randint(0, vocab, (rows, history), device="cuda", generator=gen),
                  "presence": torch.rand(rows, device="cuda", generator=gen),
                  "frequency": torch.rand(rows, device="cuda", generator=gen)}
    want = NB.penalize_logits(x, **given)
    for at in range(8):
        for pad in range(8):
            room = torch.full((at + (rows - 1) * (vocab + pad) + vocab,), float("nan"), device="cuda", dtype=x.dtype)
            strided = room.as_strided((rows, vocab), (vocab + pad, 1), at)
            strided.copy_(x)
            assert torch.equal(NB.penalize_logits(strided, **given), want), (at, pad)


def test_offsets_past_32_bits():
    """Logits of which the later rows lie more than 2^32 elements from the first."""
    import torch

    s = make(3, 5000, "bfloat16", 10, 3, True)
    room = torch.empty(3, 2_400_000_000, device="cuda", dtype=torch.bfloat16)  # 14 GB
    room[:, 17:5017] = s["logits"]
    check({**s, "logits": room[:, 17:5017]})


def test_replays_and_streams():
    import torch

    import neptune_opt_b200 as NB

    s, other = make(9, 3001, "float32", 25, 3, True), make(300, 7001, "float32", 100, 3, True, seed=1)
    NB.penalize_logits(**s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = NB.penalize_logits(**s)
    for step in range(3):
        s["tokens"].add_(1)
        s["allowed"].bitwise_not_()
        g.replay()
        check(s, out)
    want = [NB.penalize_logits(**s), NB.penalize_logits(**other)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        got = []
        for stream, x in zip(streams, (s, other)):
            with torch.cuda.stream(stream):
                got.append(NB.penalize_logits(**x))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
