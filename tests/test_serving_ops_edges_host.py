"""Serving operators at the edges of their contracts, without a GPU."""
from __future__ import annotations

import threading

import torch

import neptune_opt_b200 as NB


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
