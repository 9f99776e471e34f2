"""The rule that chooses a packed product's kernel (stwo-ml_amd/csrc/witness_cost.h), compiled for the CPU, at sizes
that both kernels were timed at with rows and weights from memory."""
import ctypes as C
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SRC = os.path.join(ROOT, "tests", "native", "witness_cost.cpp")
HDR = os.path.join(ROOT, "stwo-ml_amd", "csrc", "witness_cost.h")
OUT = os.path.join(ROOT, "tests", "native", "_build", "libwitness_cost.so")
TILES, MIXED, WIDE, BLOCKS = range(4)


@pytest.fixture(scope="module")
def kernel():
    if not os.path.exists(OUT) or os.path.getmtime(OUT) < max(os.path.getmtime(d) for d in (SRC, HDR)):
        os.makedirs(os.path.dirname(OUT), exist_ok=True)
        subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-o", OUT, SRC], check=True)
    L = C.CDLL(OUT)
    L.wc_kernel.argtypes = [C.c_uint64] * 3 + [C.c_int] * 2
    return L.wc_kernel


# fused products of int8-range words: us by k_wit_wide and by what is taken without it
@pytest.mark.parametrize("m,k,n,wide,without", [(330, 4643, 2277, 29.7, 24.2), (359, 4096, 2560, 28.6, 24.5),
                                                (257, 5120, 2560, 28.2, 24.3), (383, 13824, 4096, 65.2, 58.4),
                                                (557, 5120, 1536, 31.9, 28.7), (749, 4597, 1209, 32.7, 29.7),
                                                (476, 7958, 1944, 42.7, 38.8), (1000, 4096, 1024, 31.9, 29.3),
                                                (885, 7978, 951, 47.1, 43.3), (1517, 13824, 1024, 81.4, 75.3)])
def test_few_workgroups_are_not_slowed_down(kernel, m, k, n, wide, without):
    assert wide > 1.05 * without and kernel(m, k, n, 0, 0) != WIDE


@pytest.mark.parametrize("m,k,n,wide,without", [(512, 5120, 5120, 33.8, 44.6), (700, 576, 1536, 13.5, 19.9),
                                                (512, 2560, 2560, 23.8, 30.8), (400, 4096, 4096, 27.6, 34.1),
                                                (1024, 5120, 5120, 63.8, 70.7), (300, 5120, 5120, 31.5, 35.5),
                                                (200, 5436, 9401, 32.2, 54.8), (317, 2560, 5120, 20.6, 35.1),
                                                (2048, 576, 1536, 16.9, 22.6)])
def test_sizes_that_the_wide_kernel_leads_at(kernel, m, k, n, wide, without):
    assert wide < 0.95 * without and kernel(m, k, n, 0, 0) == WIDE


def test_what_the_rule_leaves_as_it_is(kernel):
    assert kernel(512, 13824, 5120, 0, 1) == WIDE  # quantized: no launch to join follows
    assert kernel(5000, 13824, 5120, 0, 0) == BLOCKS  # nine rounds of workgroups
    assert kernel(64 + 1, 100, 100, 0, 0) == TILES
    for m in (65, 128, 129, 256, 257, 512, 2048):
        for k, n in ((576, 1536), (5120, 5120), (13824, 5120), (5120, 13824)):
            assert kernel(m, k, n, 1, 0) != WIDE  # gated blocks have no such kernel
