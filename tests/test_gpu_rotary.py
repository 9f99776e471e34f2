"""Rotary positions (gkr_rotary_new, gkr_rotary_forward) against whole-number arithmetic with angles in 64-bit
mantissas: layouts, part of a head, odd sizes, far positions, packed and decoded rows, cut-off and field results,
in place, and what is refused."""
import numpy as np
import pytest

import gkr_mi355x as G
from test_gpu_scaled import centered
from test_gpu_witness import words

pytestmark = pytest.mark.gpu
P = G.P


def table(freqs, positions, amplitude):
    """C and S, (len(positions), pairs): the phase in whole numbers, cosines in extended precision."""
    phase = np.asarray(positions, dtype=np.uint64)[:, None] * np.asarray(freqs, dtype=np.uint64)
    angle = phase.astype(np.longdouble) / np.longdouble(2) ** 64 * (8 * np.arctan(np.longdouble(1)))
    return [(np.sign(t) * np.floor(np.abs(amplitude * t) + np.longdouble(0.5))).astype(np.int64)
            for t in (np.cos(angle), np.sin(angle))]


def turn(x, c, s, dim, shift, interleaved, limit):
    """x (rows, heads * dim) words."""
    x = centered(x).reshape(len(c), -1, dim).astype(object)
    y, half = x.copy(), c.shape[1]
    for j in range(half):
        a, b = (2 * j, 2 * j + 1) if interleaved else (j, j + half)
        cj, sj = c[:, j, None].astype(object), s[:, j, None].astype(object)
        for to, v in ((a, x[..., a] * cj - x[..., b] * sj), (b, x[..., b] * cj + x[..., a] * sj)):
            r = (2 * np.abs(v) + (1 << shift)) >> (shift + 1)
            r = np.where(v < 0, -r, r)
            y[..., to] = np.clip(r, -limit, limit) if limit else r
    return (y % P).astype(np.int64).reshape(len(c), -1)


def check(ctx, counts, starts, heads, kv, dim, turned, interleaved, kind=1, limit=127, amplitude=1 << 15, shift=15,
          positions=4096, in_place=False, seed=1, freqs=None):
    rng = np.random.default_rng(seed + sum(counts) * 7 + dim + turned)
    freqs = G.rotary_frequencies(turned) if freqs is None else freqs
    rows = sum(counts)
    at = np.concatenate([np.arange(s, s + c) for s, c in zip(starts or [0] * len(counts), counts)])
    c, s = table(freqs, at, amplitude)
    q, k = words(rng, (rows, heads * dim), kind), words(rng, (rows, max(1, kv) * dim), kind)
    r = ctx.rotary(freqs, positions, amplitude, shift)
    qm, km = ctx.upload(q), ctx.upload(k)
    qo = qm if in_place else ctx.synthetic(rows, heads * dim, 0, 9)
    ko = km if in_place else ctx.synthetic(rows, max(1, kv) * dim, 0, 10)
    ctx.rotary_forward(r, qm, qo, counts, dim, starts=starts, k=km if kv else None, k_out=ko if kv else None,
                       interleaved=interleaved, limit=limit)
    assert np.array_equal(qo.download(), turn(q, c, s, dim, shift, interleaved, limit))
    if kv:
        assert np.array_equal(ko.download(), turn(k, c, s, dim, shift, interleaved, limit))
    r.free()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("heads,kv,dim,turned", [(1, 0, 2, 2), (1, 1, 7, 2), (9, 3, 64, 64), (5, 1, 80, 80), (4, 4, 96, 40),
                                                 (3, 1, 65, 38), (40, 8, 128, 128), (2, 2, 13, 10), (2, 1, 256, 64)])
def test_layouts(gpu_ctx, heads, kv, dim, turned, interleaved):
    for kind, limit in ((1, 127), (1, 0), (0, 0), (0, 1 << 20)):
        check(gpu_ctx, [5, 0, 1, 9], [0, 17, 4095, 100], heads, kv, dim, turned, interleaved, kind, limit)
    check(gpu_ctx, [6], None, heads, kv, dim, turned, interleaved, in_place=True)


@pytest.mark.parametrize("positions", [1 << 17, 3000001])
def test_far_positions(gpu_ctx, positions):
    freqs = G.rotary_frequencies(64, 500000.0, G.ROTARY_WAVES, 8.0, 8192, 1, 4)
    check(gpu_ctx, [3, 2], [positions - 3, positions // 2], 2, 1, 64, 64, False, positions=positions, freqs=freqs)


def test_any_frequencies(gpu_ctx):
    """Quarter and eighth turns, none, the largest: exact zeros and amplitudes, signs of all quarters."""
    freqs = np.array([0, 1 << 62, 1 << 63, 3 << 62, 1 << 61, (1 << 64) - 1, 1, 0x123456789abcdef1], dtype=np.uint64)
    for amplitude, shift in ((1 << 15, 15), (1, 0), (1 << 20, 20), (12345, 3)):
        check(gpu_ctx, [40], [5], 2, 1, 16, 16, True, 0, 0, amplitude, shift, freqs=freqs)
        check(gpu_ctx, [40], [0], 2, 1, 16, 16, False, 1, 0, amplitude, shift, freqs=freqs)


def test_whole_products(gpu_ctx):
    """Full-range words by the largest amplitude, at turns whose C and S are whole: 61 bits, mod P with no shift."""
    freqs = np.array([1 << 62, 1 << 63, 0, 3 << 62], dtype=np.uint64)
    for shift in (0, 1, 29, 30):
        check(gpu_ctx, [9], None, 3, 1, 8, 8, False, 0, 0, 1 << 30, shift, freqs=freqs)


@pytest.mark.parametrize("n", [255, 256, 257, 600])
def test_many_sequences(gpu_ctx, n):
    rng = np.random.default_rng(n)
    check(gpu_ctx, [1] * n, [int(x) for x in rng.integers(0, 4096, size=n)], 3, 1, 32, 32, False)
    counts = [int(x) for x in rng.integers(0, 4, size=n)]
    counts[0] = 3
    check(gpu_ctx, counts, [int(x) for x in rng.integers(0, 4093, size=n)], 3, 1, 32, 16, True)


def test_long_prompt(gpu_ctx):
    check(gpu_ctx, [2000, 1], [1000, 7], 4, 1, 64, 64, False)


def test_refusals(gpu_ctx):
    ctx = gpu_ctx
    f = G.rotary_frequencies(8)
    r = ctx.rotary(f, 100)
    q, k, qo, ko = ctx.zeros(4, 24), ctx.zeros(4, 8), ctx.zeros(4, 24), ctx.zeros(4, 8)
    other = G.Context(0)
    theirs = other.rotary(f, 10)
    F = ctx.rotary_forward
    half = ctx.wrap_device(q.device_ptr + 4 * 24, 3, 24)
    bad = [((r, q, qo, [3], 8), {}, "q is"), ((r, q, qo, [4], 6), {}, "turned dims"), ((r, q, qo, [4], 9), {}, "whole heads"),
           ((r, q, ctx.zeros(4, 32), [4], 8), {}, "q's output"), ((r, q, qo, [4], 8), dict(k=k), "null"),
           ((r, q, qo, [4], 8), dict(k_out=ko), "null"), ((r, q, qo, [4], 8), dict(k=ctx.zeros(3, 8), k_out=ko), "k is"),
           ((r, q, qo, [4], 8), dict(k=k, k_out=ctx.zeros(4, 16)), "k's output"), ((r, q, qo, [4], 8), dict(starts=[97]), "97"),
           ((r, q, qo, [4], 8), dict(starts=[0xffffffff]), "4294967295"), ((r, q, qo, [4], 8), dict(limit=1 << 30), "limit"),
           ((r, q, k, [4], 8), dict(k=k, k_out=ko), "shares"), ((r, q, qo, [4], 8), dict(k=k, k_out=q), "shares"),
           ((r, half, ctx.wrap_device(q.device_ptr, 3, 24), [3], 8), {}, "shares"),
           ((r, q, qo, [4], 8), dict(k=k, k_out=ctx.wrap_device(qo.device_ptr, 4, 8)), "share"),
           ((theirs, q, qo, [4], 8), {}, "another"), ((r, q, other.zeros(4, 24), [4], 8), {}, "another")]
    for args, kw, why in bad:
        with pytest.raises(G.GkrError, match=why) as e:
            F(*args, **kw)
        assert e.value.code == 1
    for args in (([], 10), (f, 0), (f, (1 << 31) + 1), (f, 10, 0), (f, 10, (1 << 30) + 1), (f, 10, 1, 31)):
        with pytest.raises(G.GkrError) as e:
            ctx.rotary(*args)
        assert e.value.code == 1, args
    with pytest.raises(G.GkrError) as e:  # a table of 512 TB
        ctx.rotary(np.arange(32768, dtype=np.uint64), 1 << 31)
    assert e.value.code == 5 or e.value.code == 1 or "table" in str(e.value)
    F(r, q, qo, [4], 8, starts=[96], k=k, k_out=ko)  # and the context goes on
    assert not qo.download().any()
    other.close()
    with pytest.raises(G.GkrError, match="another"):
        F(theirs, q, qo, [4], 8)
    theirs.free()
