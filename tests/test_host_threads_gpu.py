"""Calls of several host threads at once, each on a stream of its own."""
from __future__ import annotations

import ctypes
import threading

import pytest

from conftest import cuda_available

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not cuda_available(), reason="needs a CUDA device")]


def test_gated_norm_backward_of_several_widths():
    """The widths share one kernel and ask for different amounts of shared memory."""
    import torch

    import neptune_opt_b200._lib as L

    lib, rows, wrong = L.load(), 16, []

    def work(width):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            t = torch.randn(6, rows, width, device="cuda").to(torch.bfloat16)
            w = torch.ones(4, width, device="cuda", dtype=torch.bfloat16)
            rstd = torch.ones(rows, 2, device="cuda")
            a = L.NB200NormArgs(t[0].data_ptr(), t[1].data_ptr(), None, w[0].data_ptr(), w[1].data_ptr(), rows, width,
                                width, width, width, width, width, 1, 0, 1.0, 1e-6)
            size = lib.nb200_gated_norm_bwd_work_bytes(ctypes.byref(a))
            room = torch.empty(size, dtype=torch.uint8, device="cuda")
            p = [ctypes.c_void_p(x.data_ptr()) for x in (rstd, *t[2:6], w[2], w[3], room)]
            st = ctypes.c_void_p(stream.cuda_stream)
            for _ in range(3000):
                rc = lib.nb200_gated_norm_bwd(ctypes.byref(a), 1, p[0], p[1], p[2], p[3], p[4], None, p[5], p[6], p[7], size, st)
                if rc:
                    wrong.append((width, rc, L.last_error()))
                    return
            stream.synchronize()

    threads = [threading.Thread(target=work, args=(w,)) for w in (512, 1024, 2048, 4096, 768, 3968)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong[:3]


def test_streamed_softmax_of_several_widths():
    """The same of the streaming row kernel."""
    import torch

    import neptune_opt_b200._lib as L

    lib, wrong = L.load(), []
    launch = L.launch_struct(L.VARIANT_STREAM)

    def work(width):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            x = torch.randn(8, width, device="cuda")
            y, lse = torch.empty_like(x), torch.empty(8, device="cuda")
            p = [ctypes.c_void_p(t.data_ptr()) for t in (x, y, lse)]
            st = ctypes.c_void_p(stream.cuda_stream)
            for _ in range(3000):
                rc = lib.nb200_softmax(0, p[0], 0, 8, width, width, 1, p[1], p[2], ctypes.byref(launch), st)
                if rc:
                    wrong.append((width, rc, L.last_error()))
                    return
            stream.synchronize()

    threads = [threading.Thread(target=work, args=(w,)) for w in (1024, 2048, 4096, 5120, 6144, 3584)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong[:3]
