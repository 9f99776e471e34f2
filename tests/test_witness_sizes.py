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
    L.ws_pack_groups.restype = C.c_uint64
    L.ws_pack_groups.argtypes, L.ws_packable.argtypes = [C.c_uint64] * 2, [C.c_uint64] * 3
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


def test_packed_product(lib):
    """Every grid of a packed product that is admitted has fewer than 2^32 threads in a dimension: the packing's (131072
    x 131071 words would have 2^32), and the products', a workgroup of up to 1024 threads for each group of row and
    column tiles; a workgroup's rows and the packed blocks are counted in 32 bits."""
    for m in around(5, 64, 512, 1 << 17, 1 << 20, 1 << 22):
        for k in around(1, 1024, 4096, 16384, lib.ws_max_inner()):
            groups = -(-(-(-m // 8) * -(-k // 32)) // 4)
            assert lib.ws_pack_groups(m, k) == groups
            for n in around(1, 128, 5120, 1 << 16, 1 << 21):
                if not lib.ws_packable(m, k, n):
                    continue
                assert k <= lib.ws_max_inner() and 4 * 256 * n < 1 << 32
                assert groups * 256 < 1 << 32 and 4 * groups < 1 << 32, (m, k)
                assert -(-m // 64) * -(-n // 64) * 512 < 1 << 32  # blocks, four planes of both
                runs = -(-m // 16) * -(-n // 32) // (1 << 21) + 1  # the streamed products' runs of row groups
                assert runs < 65536 and (-(-m // 16) // runs + 1) * -(-n // 32) * 1024 < 1 << 32
    for m, k in ((1 << 17, 131071), (1 << 22, 4096), (1 << 22, 4095), ((1 << 20) - 7, 16384)):
        assert m * k <= 1 << 34 and not lib.ws_packable(m, k, 32)
    for m, k, n in ((1 << 17, 131040, 32), (1 << 22, 4064, 32), (512, 13824, 5120), (5, 131071, 1 << 21)):
        assert lib.ws_packable(m, k, n)
