"""The size limits of the witness operators' kernels (stwo-ml_amd/csrc/witness_sizes.h), compiled for the CPU:
whatever they admit has offsets and grids that the kernels and the runtime take."""
import ctypes as C
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SRC = os.path.join(ROOT, "tests", "native", "witness_sizes.cpp")
HDR = os.path.join(ROOT, "stwo-ml_amd", "csrc", "witness_sizes.h")
OUT = os.path.join(ROOT, "tests", "native", "_build", "libwitness_sizes.so")


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(OUT) or os.path.getmtime(OUT) < max(os.path.getmtime(d) for d in (SRC, HDR)):
        os.makedirs(os.path.dirname(OUT), exist_ok=True)
        subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-o", OUT, SRC], check=True)
    L = C.CDLL(OUT)
    L.ws_outside.restype = L.ws_row_lds.restype = C.c_uint32
    L.ws_max_inner.restype = C.c_uint64
    L.ws_few_rows_fit.argtypes = [C.c_uint64, C.c_uint64, C.c_uint64, C.c_int]
    return L


def around(*values):
    return sorted({v + d for v in values for d in (-17, -4, -1, 0, 1, 4, 17) if v + d > 0})


def test_few_rows(lib):
    """The output's last word is inside the one buffer that it is written through (16 rows of 2^26 columns are
    not), the rows' digits fit in LDS, and the grid has fewer than 2^32 threads."""
    outside, lds = lib.ws_outside(), lib.ws_row_lds()
    limits = [1 << 26] + [outside // (4 * m) for m in range(1, 18)]
    for m in range(1, 18):
        for k in around(1, 64, 1024, 2048, lib.ws_max_inner()):
            for n in around(1, 4096, *limits):
                for one in (0, 1):
                    if not lib.ws_few_rows_fit(m, k, n, one):
                        continue
                    assert m <= 16 and k <= lib.ws_max_inner()
                    assert 4 * ((m - 1) * n + n - 1) + 4 <= outside, (m, n)
                    assert -(-n // 32) * 1024 < 1 << 32
                    if m > 4:
                        assert one and 4 * (8 if m <= 8 else 16) * -(-k // 64) * 64 <= lds
    assert not lib.ws_few_rows_fit(16, 1, 1 << 26, 1)
    assert lib.ws_few_rows_fit(16, 1, (1 << 26) - 1, 1) and lib.ws_few_rows_fit(15, 1, 1 << 26, 1)
    assert lib.ws_few_rows_fit(4, 131071, 1 << 26, 0) and lib.ws_few_rows_fit(16, 1024, 5120, 1)
    assert lib.ws_few_rows_fit(8, 2048, 5120, 1) and not lib.ws_few_rows_fit(8, 2049, 5120, 1)
