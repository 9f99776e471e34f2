"""The paged key-value cache's page book and its byte layout (stwo-ml_amd/csrc/kv_book.h), compiled for
the CPU: random sequences of operations against a model, refused appends that leave everything as it was,
and a layout in which every (token, dim) has a byte of its own."""
import ctypes as C
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SRC = os.path.join(ROOT, "tests", "native", "kv_book.cpp")
HDR = os.path.join(ROOT, "stwo-ml_amd", "csrc", "kv_book.h")
OUT = os.path.join(ROOT, "tests", "native", "_build", "libkv_book.so")


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(OUT) or os.path.getmtime(OUT) < max(os.path.getmtime(d) for d in (SRC, HDR)):
        os.makedirs(os.path.dirname(OUT), exist_ok=True)
        subprocess.run(["g++", "-O1", "-g", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-o", OUT, SRC],
                       check=True)
    L = C.CDLL(OUT)
    L.kvb_new.restype = C.c_void_p
    for f in ("kvb_free", "kvb_open", "kvb_close", "kvb_cut", "kvb_live", "kvb_free_pages", "kvb_len", "kvb_pages"):
        getattr(L, f).argtypes = [C.c_void_p] + ([] if f in ("kvb_free", "kvb_free_pages") else
                                                 [C.POINTER(C.c_uint32)] if f == "kvb_open" else [C.c_uint32])
    L.kvb_cut.argtypes = [C.c_void_p, C.c_uint32, C.c_uint32]
    L.kvb_pages.argtypes = [C.c_void_p, C.c_uint32, C.POINTER(C.c_uint32)]
    L.kvb_extend.argtypes = [C.c_void_p, C.POINTER(C.c_uint32), C.POINTER(C.c_uint32), C.c_size_t, C.c_int]
    return L


def pages(lib, b, seq):
    out = (C.c_uint32 * 4096)()
    return list(out[:lib.kvb_pages(b, seq, out)])


def extend(lib, b, seqs, counts, undo=0):
    n = len(seqs)
    return lib.kvb_extend(b, (C.c_uint32 * n)(*seqs), (C.c_uint32 * n)(*counts), n, undo)


@pytest.mark.parametrize("page_tokens,n_pages,max_tokens", [(64, 20, 700), (128, 9, 1 << 21), (64, 1, 64)])
def test_random_operations(lib, page_tokens, n_pages, max_tokens):
    rng = random.Random(n_pages)
    b = lib.kvb_new(n_pages, page_tokens, 5, max_tokens)
    model = {}
    for _ in range(2000):
        op = rng.randrange(6)
        if op == 0:
            s = C.c_uint32(99)
            assert lib.kvb_open(b, C.byref(s)) == (len(model) < 5)
            if len(model) < 5:
                assert s.value < 5 and s.value not in model
                model[s.value] = 0
        elif op == 1 and model:
            s = rng.choice(list(model))
            lib.kvb_close(b, s)
            del model[s]
            assert not lib.kvb_live(b, s)
        elif op == 2 and model:
            s = rng.choice(list(model))
            model[s] = rng.randrange(model[s] + 1)
            lib.kvb_cut(b, s, model[s])
        elif model:
            seqs = [rng.choice(list(model)) for _ in range(rng.randrange(1, 4))]
            counts = [rng.choice([0, 1, 3, 63, 64, 65, 200]) for _ in seqs]
            after, undo = dict(model), op == 5
            for s, n in zip(seqs, counts):
                after[s] += n
            fits = all(v <= max_tokens for v in after.values()) and \
                sum(-(-v // page_tokens) for v in after.values()) <= n_pages
            assert extend(lib, b, seqs, counts, undo) == fits
            if fits and not undo:
                model = after
        held = []
        for s, n in model.items():
            assert lib.kvb_live(b, s) and lib.kvb_len(b, s) == n
            mine = pages(lib, b, s)
            assert len(mine) == -(-n // page_tokens)
            held += mine
        assert len(set(held)) == len(held) and all(p < n_pages for p in held)  # no page twice
        assert lib.kvb_free_pages(b) == n_pages - len(held)
    lib.kvb_free(b)


def test_lengths_near_the_type_range(lib):
    """Counts whose sum with the length passes 32 bits are refused, not wrapped."""
    b = lib.kvb_new(4, 64, 1, 1 << 21)
    s = C.c_uint32()
    lib.kvb_open(b, C.byref(s))
    assert extend(lib, b, [s.value], [100]) == 1
    for n in (0xFFFFFFFF, 0xFFFFFFFF - 99, (1 << 21) - 99):
        assert extend(lib, b, [s.value], [n]) == 0
        assert lib.kvb_len(b, s.value) == 100 and len(pages(lib, b, s.value)) == 2
    lib.kvb_free(b)


@pytest.mark.parametrize("planes", [1, 4])
@pytest.mark.parametrize("dim", [1, 16, 80, 256])
def test_every_value_has_its_byte(lib, dim, planes):
    chunks = (dim + 15) // 16
    for at in (lib.kvb_key_byte, lib.kvb_value_byte):
        seen = {at(t, d, p, planes) for t in range(64) for d in range(dim) for p in range(planes)}
        assert len(seen) == 64 * dim * planes and max(seen) < 1024 * chunks * planes
    # four tokens 4 i .. 4 i + 3 of a dim are neighbours among the values
    assert all(lib.kvb_value_byte(4 * i + v, 3 % dim, 0, planes) == lib.kvb_value_byte(4 * i, 3 % dim, 0, planes) + v
               for i in range(16) for v in range(4))


@pytest.mark.parametrize("n_pages,page_tokens,kv_heads,dim,planes", [
    (1, 64, 1, 1, 1), (16, 64, 8, 128, 1), (1000, 192, 3, 80, 4), (1 << 10, 65536, 4096, 256, 4),
    ((1 << 10) + 1, 65536, 4096, 256, 4), (1 << 26, 65536, 4096, 256, 4), ((1 << 26) + 1, 65536, 4096, 256, 4),
    ((1 << 32) - 1, 65536, 4096, 256, 4), ((1 << 32) - 1, 64, 1, 1, 1), (1 << 31, 64, 128, 16, 1),
    ((1 << 31) + 1, 64, 128, 16, 1), ((1 << 32) - 1, 64, 4096, 250, 4)])
def test_pool_bytes(lib, n_pages, page_tokens, kv_heads, dim, planes):
    """A pool's size against whole numbers of any length; sizes that would wrap around 64 bits (2^26 pages of 65536
    tokens, 4096 heads of 256 general values: exactly 2^64) are refused."""
    want = n_pages * (page_tokens // 64) * kv_heads * planes * -(-dim // 16) * 1024
    got = C.c_uint64(12345)
    fits = lib.kvb_pool_bytes(n_pages, page_tokens, kv_heads, dim, planes, C.byref(got))
    assert fits == (want <= 1 << 48)
    assert got.value == (want if fits else 12345)
