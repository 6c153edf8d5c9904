"""Serving operators at the edges of their contracts, without a GPU."""
from __future__ import annotations

import threading

import pytest
import torch

import neptune_opt_b200 as NB
import neptune_opt_b200._lib as L
from host_code import with_fake_runtime


def _meta(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="meta")


def test_two_threads_make_their_first_8_bit_call(monkeypatch):
    """The second one comes while the first is still putting the table of types together."""
    import neptune_opt_b200.quantized_norm as module

    results = []

    def call():
        try:
            results.append(NB.quantized_rms_norm(_meta(2, 64), _meta(64))[0].dtype)
        except Exception as e:  # noqa: BLE001
            results.append(e)

    class Kinds(dict):
        met = False

        def __getitem__(self, name):
            if not Kinds.met:
                Kinds.met = True
                other = threading.Thread(target=call)
                other.start()
                other.join()
            return dict.__getitem__(self, name)

    monkeypatch.setattr(module, "_KINDS", None)
    monkeypatch.setattr(module, "KINDS", Kinds(module.KINDS))
    call()
    assert Kinds.met and results == [torch.float8_e4m3fn] * 2, results


LOGITS = """
import ctypes
import neptune_opt_b200._lib as L
lib = L.load()
p = 1 << 20
# 9000 tokens of history: the kernel that names them, then the sweep.
a = L.NB200LogitsArgs(p, p, None, None, None, None, None, None, None, None, None, 4, 50000, 9000, 0, 50000, 9000, 0, 0, 0, 0, 1, 0)
n = lib.nb200_penalize_logits_work_bytes(ctypes.byref(a))
rc = lib.nb200_penalize_logits(ctypes.byref(a), ctypes.c_void_p(1 << 30), ctypes.c_void_p(1 << 40), n, None)
print(rc, ctypes.CDLL(None).fake_launches(), lib.nb200_launch_count())
"""


@pytest.mark.parametrize("fails,launches", [(0, 2), (1, 1), (2, 2)])
def test_no_sweep_behind_names_that_were_not_launched(tmp_path, fails, launches):
    rc, made, counted = map(int, with_fake_runtime(tmp_path, LOGITS, fails).split())
    assert rc == (L.NB200_ERR_LAUNCH if fails else L.NB200_OK) and made == launches
    assert counted == launches or fails
