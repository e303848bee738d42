"""The library's own rules for the kernel of an FP8 product (csrc/qkm_fp8_choice.h), built for the host."""
import ctypes
import functools
import os
import subprocess
import tempfile

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "qwen-kernel_b200", "csrc")

PROGRAM = r"""
#include "qkm_fp8_choice.h"
extern "C" int pairs_as_lanes(int down, unsigned n, unsigned n_used, unsigned n_expert) { return qkm::fp8_pairs_as_lanes(down != 0, n, n_used, n_expert); }
extern "C" int shared_few_rows(int down, unsigned n, unsigned M, unsigned K) { return qkm::fp8_shared_few_rows(down != 0, n, M, K); }
extern "C" int dense_kernel(unsigned n, unsigned M, unsigned K, unsigned n_sms) { return (int)qkm::fp8_dense_kernel(n, M, K, n_sms); }
"""
DENSE = ("rows", "group", "128x32", "128x64", "256x128", "128x256", "256x256")


@functools.lru_cache(None)
def rules():
    with tempfile.TemporaryDirectory() as d:
        src, lib = os.path.join(d, "choice.cpp"), os.path.join(d, "choice.so")
        open(src, "w").write(PROGRAM)
        subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I" + CSRC, src, "-o", lib], check=True)
        return ctypes.CDLL(lib)


def pairs_as_lanes(down, n, n_used, n_expert):
    return bool(rules().pairs_as_lanes(int(down), n, n_used, n_expert))


def shared_few_rows(down, n, M, K):
    return bool(rules().shared_few_rows(int(down), n, M, K))


def dense_kernel(n, M, K, n_sms=148):
    return DENSE[rules().dense_kernel(n, M, K, n_sms)]
