"""Several new tokens of a sequence, of which the earlier ones do not see the later ones: what those hold does not reach them,
be it an infinity or NaN. Bounds as in test_prefix_attention_gpu.py, whose reference takes each query's own keys alone."""
from __future__ import annotations

import math

import pytest

from conftest import cuda_available
from test_prefix_attention_gpu import lens_of, make, reference

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_available(), reason="needs a CUDA device")]

# (batch, heads, kv_heads, tokens, prefix, cache): the single kernel with one and two row tiles; the stream kernel with one, two
# and four, and with several tiles of a sequence's rows; behind the tensor cores.
CALLS = [(3, 4, 2, 3, 100, 70), (3, 8, 2, 4, 100, 70), (2, 2, 1, 4, 64, 3000), (2, 6, 2, 5, 3000, 333), (3, 24, 1, 1, 50, 60),
         (3, 16, 1, 7, 40, 90), (3, 16, 1, 33, 40, 90), (20, 8, 2, 5, 1000, 50)]


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("junk", [math.inf, -math.inf, math.nan])
def test_later_tokens_do_not_reach_earlier_ones(call, dim, dtype, junk):
    import torch

    import neptune_opt_b200 as NB

    batch, _, kv_heads, tokens, _, cache = call
    q, pk, pv, k, v = make(*call[:4], dim, *call[4:], dtype=dtype, seed=tokens)
    lens = lens_of(*[(cache, tokens, 49, max(1, tokens - 1), 17 + tokens, 0)[i % 6] for i in range(batch)])
    want = NB.prefix_attention(q, pk, pv, k, v, lens, return_lse=True)
    k2, v2 = k.clone(), v.clone()
    for i, n in enumerate(lens.tolist()):
        n = min(n, cache)
        for back in range(1, min(tokens, n) + 1):  # the last `back` tokens: some columns of one head or all of them
            if back in (1, 3):
                v2[i, i % kv_heads, n - back, back::3] = junk
                k2[i, i % kv_heads, n - back, 0] = math.nan if back == 1 and i % 2 else k[i, i % kv_heads, n - back, 0]
    o, lse = NB.prefix_attention(q, pk, pv, k2, v2, lens, return_lse=True)
    ro, rl, _, _ = reference(q, pk, pv, k2, v2, lens, dim ** -0.5)
    # A finite result has no junk in its column, nor NaN in its scores: its bound is that of the values without any.
    _, _, tol, tol_lse = reference(q, pk, pv, k, torch.where(torch.isfinite(v2), v2, 0.0), lens, dim ** -0.5)
    seen = torch.isfinite(ro)
    assert torch.equal(torch.isfinite(o), seen) and bool((~seen).any())
    assert bool(((o.double() - ro).abs() <= tol)[seen].all())
    known = torch.isfinite(rl)
    assert torch.equal(torch.isfinite(lse), known) and bool(((lse.double() - rl).abs() <= tol_lse)[known].all())
    # Rows that see nothing of it come out as they did.
    clean = seen.all(-1) & (torch.isfinite(rl) | (rl == -math.inf))
    assert torch.equal(o[clean], want[0][clean]) and torch.equal(lse[clean], want[1][clean])
