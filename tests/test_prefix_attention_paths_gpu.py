"""Attention behind a shared prefix on each of its kernels' forms, named by what the call asks of its workspace."""
from __future__ import annotations

import ctypes

import pytest

from conftest import cuda_available
from test_prefix_attention_gpu import check, lens_of, make

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_available(), reason="needs a CUDA device")]


def single(call, dim, dtype):
    """Whether the single kernel takes the call: it needs no workspace to speak of."""
    import neptune_opt_b200._lib as L

    batch, heads, kv_heads, tokens, prefix, cache = call
    a = L.NB200PrefixAttnArgs(batch, heads, kv_heads, tokens, dim, prefix, cache, None, 1 if dtype == "bfloat16" else 2, 0.1)
    need = L.load().nb200_prefix_attention_work_bytes(ctypes.byref(a))
    assert need > 0
    return need == 16


def lens(batch, cache, tokens):
    return lens_of(*[(cache, tokens, 0, cache // 2, max(0, tokens - 1), cache - 1, 17, 99999, -2)[i % 9] for i in range(batch)])


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("call", [
    (40, 16, 4, 1, 300, 100), (40, 16, 4, 3, 300, 100), (38, 64, 4, 1, 17, 300), (75, 18, 2, 1, 333, 33),  # more than the SMs
    (4, 16, 4, 1, 300, 100), (4, 16, 4, 3, 300, 100), (5, 13, 1, 1, 100, 200)])  # fewer
def test_the_single_kernel_with_one_and_two_row_tiles(call, dim, dtype):
    """At head dimension 128 with four warps a CTA where there are more sequences and heads than SMs, else with eight."""
    assert single(call, dim, dtype)
    args = make(*call[:4], dim, *call[4:], dtype=dtype, seed=call[0])
    check(args, lens(call[0], call[5], call[3]))


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("call", [
    (33, 36, 2, 1, 1025, 60),   # 594 rows a head: two blocks in paired streams, one of 82 in alternating ones
    (17, 17, 1, 1, 3001, 40),   # 289: one and one, of 33
    (16, 24, 1, 1, 1300, 20),   # 384: the last block is just full
    (3, 128, 1, 1, 700, 50),    # 384 of few sequences
    (257, 1, 1, 1, 5000, 9),    # 257: a block of one row
    (16, 4, 4, 6, 129 * 128, 30)])  # 96 rows of several tokens, alternating alone
def test_paired_and_alternating_streams_in_one_call(call, dim, dtype):
    assert not single(call, dim, dtype)
    args = make(*call[:4], dim, *call[4:], dtype=dtype, seed=call[0])
    check(args, lens(call[0], call[5], call[3]))
