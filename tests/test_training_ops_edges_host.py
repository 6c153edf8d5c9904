"""Training operators at the edges of their contracts, without a GPU."""
from __future__ import annotations

import ctypes

import pytest

import neptune_opt_b200._lib as L


@pytest.mark.parametrize("batch,heads,kv,seq", [(0, 8, 2, 16), (2, 0, 0, 16), (2, 8, 2, 0), (0, 0, 0, 0), (2, 0, 3, 16)])
def test_attention_backward_needs_no_work_memory_for_an_empty_call(batch, heads, kv, seq):
    a = L.NB200AttnArgs(batch, heads, kv, seq, 128, None, 0, 0.1)
    lib = L.load()
    assert lib.nb200_attention_bwd_work_bytes(ctypes.byref(a)) == 0
    s = (L.NB200AttnStrides * 8)()
    null = ctypes.c_void_p(0)
    assert lib.nb200_attention_bwd(ctypes.byref(a), s, *[null] * 10, 0, null) == L.NB200_OK
