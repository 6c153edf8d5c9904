"""Headers of the kernels that hold plain arithmetic, compiled for the host so that tests can call them."""
from __future__ import annotations

import ctypes
import os
import subprocess
import sys

from conftest import ROOT


def compiled(directory, source: str) -> ctypes.CDLL:
    """`source` (C++ with extern "C" functions; the kernels' headers are on the include path) as a loaded library."""
    path, out = os.path.join(str(directory), "host.cpp"), os.path.join(str(directory), "host.so")
    with open(path, "w") as f:
        f.write(source)
    csrc = os.path.join(ROOT, "neptune_opt_b200", "csrc")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I", csrc, "-o", out, path], check=True)
    return ctypes.CDLL(out)


FAKE_RUNTIME = r"""
#include <stddef.h>
#include <stdlib.h>
static int launches, last;
int cudaGetDevice(int* device) { *device = 0; return 0; }
int cudaDeviceGetAttribute(int* value, int attribute, int device) { (void)attribute, (void)device; *value = 148; return 0; }
int cudaFuncSetAttribute(const void* f, int attribute, int value) { (void)f, (void)attribute, (void)value; return 0; }
int cudaGetLastError(void) { int e = last; last = 0; return e; }
int cudaLaunchKernelExC(const void* config, const void* f, void** args) {
    (void)config, (void)f, (void)args;
    const char* fails = getenv("FAKE_FAILS");
    if (++launches == (fails ? atoi(fails) : 0)) return last = 1;  /* cudaErrorInvalidValue */
    return 0;
}
int fake_launches(void) { return launches; }
"""


def with_fake_runtime(directory, script: str, fails: int) -> str:
    """What `script` prints in a process whose kernel launches go nowhere; launch number `fails` (from 1) returns an error.
    `ctypes.CDLL(None).fake_launches()` counts them."""
    path, out = os.path.join(str(directory), "fake.c"), os.path.join(str(directory), "fake.so")
    with open(path, "w") as f:
        f.write(FAKE_RUNTIME)
    subprocess.run(["gcc", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-o", out, path], check=True)
    env = {**os.environ, "LD_PRELOAD": out, "FAKE_FAILS": str(fails), "CUDA_VISIBLE_DEVICES": "",
           "PYTHONPATH": os.pathsep.join([ROOT, os.environ.get("PYTHONPATH", "")])}
    return subprocess.run([sys.executable, "-c", script], env=env, check=True, capture_output=True, text=True).stdout
