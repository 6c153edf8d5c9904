"""Serving operators at the edges of their contracts, without a GPU."""
from __future__ import annotations

import threading

import pytest
import torch

import neptune_opt_b200 as NB
import neptune_opt_b200._lib as L
from host_code import with_fake_runtime


def _meta(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="meta")


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


# ------------------------------------------------------------------ the ops themselves, traced without the Python functions
I32, I64, F32 = torch.int32, torch.int64, torch.float32


def _op_attention(**changes):
    a = {"q": _meta(3, 8, 2, 128), "pk": _meta(2, 100, 128), "pv": _meta(2, 100, 128), "k": _meta(3, 2, 50, 128),
         "v": _meta(3, 2, 50, 128), "lens": _meta(3, dtype=I32), "scale": 0.1, **changes}
    return torch.ops.nb200.prefix_attention(*a.values(), True)


def _op_norm8(**changes):
    a = {"x": _meta(4, 96), "weight": _meta(96), "residual": _meta(4, 96), "group": 32, "kind": 0, "eps": 1e-6, **changes}
    return torch.ops.nb200.norm8(*a.values())


def _op_logits(**changes):
    a = {"logits": _meta(4, 100), "tokens": _meta(4, 7, dtype=I64), "token_lens": _meta(4, dtype=I32),
         "prompt_lens": _meta(4, dtype=I32), "repetition": _meta(4, dtype=F32), "presence": _meta(4, dtype=F32),
         "frequency": _meta(4, dtype=F32), "bias_index": _meta(4, 3, dtype=I32), "bias_value": _meta(4, 3, dtype=F32),
         "allowed": _meta(4, 4, dtype=I32), "temperature": _meta(4, dtype=F32), **changes}
    return torch.ops.nb200.penalize_logits(*a.values())


@pytest.mark.parametrize("op,error,bad", [
    (_op_attention, ValueError, {"scale": 0.0}), (_op_attention, ValueError, {"scale": float("nan")}),
    (_op_attention, ValueError, {"scale": 1e-60}), (_op_attention, ValueError, {"k": _meta(3, 2, 49, 128)}),
    (_op_attention, NotImplementedError, {"q": _meta(3, 8, 2, 96), "pk": _meta(2, 100, 96), "pv": _meta(2, 100, 96),
                                          "k": _meta(3, 2, 50, 96), "v": _meta(3, 2, 50, 96)}),
    (_op_attention, TypeError, {"lens": _meta(3, dtype=I64)}),
    (_op_norm8, TypeError, {"x": _meta(4, 96, dtype=torch.float64)}), (_op_norm8, TypeError, {"weight": _meta(96, dtype=F32)}),
    (_op_norm8, TypeError, {"residual": _meta(4, 96, dtype=F32)}), (_op_norm8, TypeError, {"kind": 3}),
    (_op_norm8, ValueError, {"weight": _meta(95)}), (_op_norm8, ValueError, {"weight": _meta(1, 96)}),
    (_op_norm8, ValueError, {"residual": _meta(3, 96)}), (_op_norm8, ValueError, {"group": 64}),
    (_op_norm8, ValueError, {"group": 24}), (_op_norm8, ValueError, {"group": -32}), (_op_norm8, ValueError, {"eps": 0.0}),
    (_op_norm8, ValueError, {"eps": float("inf")}), (_op_norm8, ValueError, {"eps": 1e-60}),
    (_op_norm8, ValueError, {"x": _meta(), "residual": None}),
    (_op_norm8, ValueError, {"x": _meta(4, 0), "weight": _meta(0), "residual": None}),
    (_op_norm8, NotImplementedError, {"x": _meta(1, 16416), "weight": _meta(16416), "residual": None}),
    (_op_logits, TypeError, {"logits": _meta(4, 100, dtype=torch.float64)}), (_op_logits, TypeError, {"tokens": _meta(4, 7)}),
    (_op_logits, TypeError, {"token_lens": _meta(4, dtype=I64)}), (_op_logits, TypeError, {"temperature": _meta(4)}),
    (_op_logits, TypeError, {"allowed": _meta(4, 4, dtype=I64)}), (_op_logits, TypeError, {"bias_value": _meta(4, 3)}),
    (_op_logits, TypeError, {"bias_index": _meta(4, 3, dtype=torch.int16)}), (_op_logits, ValueError, {"logits": _meta(100)}),
    (_op_logits, ValueError, {"tokens": _meta(3, 7, dtype=I64)}), (_op_logits, ValueError, {"tokens": None}),
    (_op_logits, ValueError, {"repetition": _meta(3, dtype=F32)}), (_op_logits, ValueError, {"presence": _meta(4, 1, dtype=F32)}),
    (_op_logits, ValueError, {"bias_value": None}), (_op_logits, ValueError, {"bias_value": _meta(4, 2, dtype=F32)}),
    (_op_logits, ValueError, {"allowed": _meta(4, 3, dtype=I32)}),
    (_op_logits, NotImplementedError, {"bias_index": _meta(4, 1025, dtype=I32), "bias_value": _meta(4, 1025, dtype=F32)})])
def test_traced_ops_refuse_what_no_kernel_takes(op, error, bad):
    _meta_ops()
    op()
    with pytest.raises(error):
        op(**bad)


def _meta_ops():
    """The ops are registered by the first call of a function."""
    NB.penalize_logits(_meta(1, 1))


def test_no_workspace_is_quoted_for_logits_that_no_grid_holds():
    """Rows times tiles, or times the naming kernel's parts, past 2^31: refused before a size is worked out of them."""
    import ctypes

    lib = L.load()

    def work(rows, vocab, history):
        a = L.NB200LogitsArgs(*[1 << 20] * 2, *[None] * 9, rows, vocab, history, 0, vocab, history, 0, 0, 0, 0, 1, 0)
        return lib.nb200_penalize_logits_work_bytes(ctypes.byref(a)), lib.nb200_penalize_logits(
            ctypes.byref(a), ctypes.c_void_p(1 << 63), ctypes.c_void_p(1 << 40), 1 << 62, None)

    for sizes in ((1 << 30, 1 << 30, 1 << 28), (1 << 30, 1 << 30, 5000), (1 << 30, 1 << 24, 0), (1 << 26, 1 << 18, 1 << 20)):
        assert work(*sizes) == (L.NB200_ERR_CAPACITY,) * 2, sizes
    assert work(1 << 20, 1 << 20, 9000)[0] > 0
