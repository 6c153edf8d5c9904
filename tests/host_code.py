"""Headers of the kernels that hold plain arithmetic, compiled for the host so that tests can call them."""
from __future__ import annotations

import ctypes
import os
import subprocess

from conftest import ROOT


def compiled(directory, source: str) -> ctypes.CDLL:
    """`source` (C++ with extern "C" functions; the kernels' headers are on the include path) as a loaded library."""
    path, out = os.path.join(str(directory), "host.cpp"), os.path.join(str(directory), "host.so")
    with open(path, "w") as f:
        f.write(source)
    csrc = os.path.join(ROOT, "neptune_opt_b200", "csrc")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I", csrc, "-o", out, path], check=True)
    return ctypes.CDLL(out)
