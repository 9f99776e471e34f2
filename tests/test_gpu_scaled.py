"""Products with scales for each row and column (gkr_matmul_forward_scaled, gkr_matmul_forward_quantized) against
whole-number arithmetic of any length: every kernel that the sizes choose, scales and shifts at their ends, rows
of zeros, the results' cut-off, parts left out, and what is refused."""
import numpy as np
import pytest

import gkr_mi355x as G
from test_gpu_witness import product, words

pytestmark = pytest.mark.gpu
P = G.P
HALF = (1 << 30) - 1


def centered(w):
    w = w.astype(np.int64)
    return np.where(w > HALF, w - P, w)


def rescale(z, r, s, shift, limit, bias=None, residual=None):
    """z (m, n) words, r (m) and s (n) whole numbers: in Python's integers."""
    c, limit = centered(z), limit or HALF
    size = np.abs(c).astype(object) * np.asarray(r).astype(object)[:, None] * np.asarray(s).astype(object)[None, :]
    t = (2 * size + (1 << shift)) >> (shift + 1)
    t = np.where(c < 0, -t, t)
    if bias is not None:
        t = t + centered(bias).astype(object)[None, :]
    y = np.clip(t, -limit, limit).astype(np.int64)
    return (y + (0 if residual is None else residual.astype(np.int64))) % P


def quantize(x, levels):
    c = centered(x)
    a = np.abs(c).max(axis=1)
    q = np.sign(c) * ((2 * levels * np.abs(c) + a[:, None]) // np.maximum(1, 2 * a[:, None]))
    return q % P, a


def check(ctx, m, k, n, xk, wk, shift, limit, bias=True, residual=True, pre=True, r=None, s=None, levels=None, seed=1, x=None):
    """levels: the quantized form, of words as wide as xk says."""
    rng = np.random.default_rng(seed + m * 31 + k * 7 + n)
    A, B = words(rng, (m, k), xk) if x is None else x, words(rng, (k, n), wk)
    r = rng.integers(1 << 14, 1 << 15, size=m) if r is None else r
    s = rng.integers(1 << 14, 1 << 15, size=n) if s is None else s
    bv, rv = words(rng, (1, n), 0) >> 8, words(rng, (m, n), 0)
    a, b, bm, rm = (ctx.upload(t) for t in (A, B, bv, rv))
    rs, cs = ctx.upload(r.reshape(m, 1).astype(np.uint32)), ctx.upload(s.reshape(1, n).astype(np.uint32))
    q, r = quantize(A, levels) if levels else (A, r)
    Z = product(q.astype(np.uint32), B)
    want = rescale(Z, r, s, shift, limit, bv[0] if bias else None, rv if residual else None)
    kw = dict(col_scales=cs, shift=shift, limit=limit, bias=bm if bias else None, residual=rm if residual else None)
    for again in range(2):  # the second finds the weight's planes built; every output is written by every call
        out, z = ctx.synthetic(m, n, 0, 5 + again), ctx.synthetic(m, n, 0, 6 + again)
        if levels:
            qm, sm = ctx.synthetic(m, k, 0, 7 + again), ctx.synthetic(m, 1, 0, 8 + again)
            ctx.matmul_forward_quantized(a, b, out, levels=levels, pre=z if pre else None, quantized=qm if pre else None,
                                         row_scales=sm if pre else None, **kw)
            if pre:
                assert np.array_equal(qm.download(), q)
                assert np.array_equal(sm.download()[:, 0], r)
        else:
            ctx.matmul_forward_scaled(a, b, out, row_scales=rs, pre=z if pre else None, **kw)
        if pre:
            assert np.array_equal(z.download(), Z)
        assert np.array_equal(out.download(), want)


# int8 results of int8 operands: about 18 + log2(k) / 2 bits of sums and 29 of scales
@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 8, 9, 16, 17, 33, 64, 65, 130, 300])
@pytest.mark.parametrize("k,n", [(1, 1), (33, 31), (576, 192), (1000, 333)])
def test_row_counts(gpu_ctx, m, k, n):
    check(gpu_ctx, m, k, n, 1, 1, 40, 127)
    check(gpu_ctx, m, k, n, 1, 0, 50, 127, residual=False)
    check(gpu_ctx, m, k, n, 0, 1, 50, 0, levels=127)
    check(gpu_ctx, m, k, n, 0, 0, 50, 1 << 20, bias=False, pre=False, levels=127)


@pytest.mark.parametrize("m,k,n", [(1, 13824, 700), (3, 20000, 65), (6, 9000, 100), (40, 17000, 96), (2, 140001, 3),
                                   (33, 131073, 5), (100, 5121, 5101), (130, 1130, 5131), (513, 2001, 2003),
                                   (200, 13825, 1030), (300, 300, 9001), (4, 16400, 8193), (16, 300, 8300)])
def test_kernels(gpu_ctx, m, k, n):
    for levels in (None, 127):
        check(gpu_ctx, m, k, n, 0 if levels else 1, 1, 45, 127, levels=levels, pre=False)
        check(gpu_ctx, m, k, n, 0, 1, 50, 0, levels=levels, residual=False)
    if m * k * n < 1 << 28:
        check(gpu_ctx, m, k, n, 0, 0, 55, 1 << 28, levels=127)


# the scales' and shift's ends: results of 92 bits down to none
@pytest.mark.parametrize("shift", [0, 1, 5, 30, 31, 32, 33, 45, 61, 62, 63])
@pytest.mark.parametrize("m", [3, 40])
def test_shifts(gpu_ctx, m, shift):
    rng = np.random.default_rng(shift)
    n = 70
    for top in (1, 2, 1 << 16, P):
        r, s = rng.integers(0, top, size=m), rng.integers(0, top, size=n)
        r[0], s[0] = 0, top - 1
        if m > 1:
            r[1] = top - 1
        for limit in (0, 1, 127, HALF):
            check(gpu_ctx, m, 64, n, 0, 0, shift, limit, r=r, s=s)


# sums that lie on halves: q q^T of small numbers by powers of two
@pytest.mark.parametrize("shift", [1, 2, 7])
def test_halves(gpu_ctx, shift):
    m, n = 5, 2048
    x = np.array([[1], [P - 1], [3], [P - 3], [0]], dtype=np.uint32)
    w = np.arange(n, dtype=np.int64) - n // 2
    W = np.where(w < 0, w + P, w).astype(np.uint32)[None, :]
    out = gpu_ctx.zeros(m, n)
    gpu_ctx.matmul_forward_scaled(gpu_ctx.upload(x), gpu_ctx.upload(W), out, shift=shift)
    z = (centered(x) * w[None, :]) % P
    assert np.array_equal(out.download(), rescale(z, np.ones(m, np.int64), np.ones(n, np.int64), shift, 0))


@pytest.mark.parametrize("levels", [1, 2, 7, 100, 127])
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (1, 700, 40), (2, 16400, 33), (3, 9000, 40), (16, 513, 50), (40, 700, 90),
                                   (7, 17000, 20), (300, 65, 40)])
def test_levels(gpu_ctx, m, k, n, levels):
    """Rows of zeros, of one value that is not zero, of the field's ends, of halves between two levels."""
    rng = np.random.default_rng(m + k + levels)
    x = words(rng, (m, k), 0)
    for i in range(m):
        kind = i % 6
        if kind == 1:
            x[i] = 0
        elif kind == 2:
            x[i] = 0
            x[i, k // 2] = P - 1
        elif kind == 3:
            x[i] = np.where(rng.random(k) < 0.5, HALF, P - HALF)
        elif kind == 4:  # c levels / a at halves: a = 2 levels, odd c
            v = 2 * rng.integers(-levels, levels, size=k) + 1
            v[0] = 2 * levels
            x[i] = np.where(v < 0, v + P, v)
        elif kind == 5:
            x[i] = rng.integers(0, 3, size=k)
    check(gpu_ctx, m, k, n, 0, 1, 40, 0, levels=levels, x=x)


def test_one_scale_word_each(gpu_ctx):
    """No scales, bias, residual or parts: a product that is cut off."""
    rng = np.random.default_rng(4)
    A, B = words(rng, (20, 50), 1), words(rng, (50, 30), 1)
    a, b, out = gpu_ctx.upload(A), gpu_ctx.upload(B), gpu_ctx.zeros(20, 30)
    z = product(A, B)
    one = np.ones(30, np.int64)
    gpu_ctx.matmul_forward_scaled(a, b, out, limit=1000)
    assert np.array_equal(out.download(), rescale(z, one[:20], one, 0, 1000))
    gpu_ctx.matmul_forward_scaled(a, b, out, shift=9)
    assert np.array_equal(out.download(), rescale(z, one[:20], one, 9, 0))


@pytest.mark.parametrize("m", [1, 20, 300])
def test_residual_in_place(gpu_ctx, m):
    rng = np.random.default_rng(m)
    A, B, R = words(rng, (m, 100), 1), words(rng, (100, 70), 1), words(rng, (m, 70), 0)
    one = np.ones(300, np.int64)
    out = gpu_ctx.upload(R)
    gpu_ctx.matmul_forward_scaled(gpu_ctx.upload(A), gpu_ctx.upload(B), out, shift=6, limit=500, residual=out)
    assert np.array_equal(out.download(), rescale(product(A, B), one[:m], one[:70], 6, 500, residual=R))
    out = gpu_ctx.upload(R)
    gpu_ctx.matmul_forward_quantized(gpu_ctx.upload(A), gpu_ctx.upload(B), out, shift=12, residual=out)
    q, a = quantize(A, 127)
    assert np.array_equal(out.download(), rescale(product(q.astype(np.uint32), B), a, one[:70], 12, 0, residual=R))


def test_refusals(gpu_ctx):
    ctx = gpu_ctx
    m, k, n = 6, 40, 20
    a, b, out, pre = ctx.zeros(m, k), ctx.zeros(k, n), ctx.zeros(m, n), ctx.zeros(m, n)
    rs, cs, q = ctx.zeros(m, 1), ctx.zeros(1, n), ctx.zeros(m, k)
    S, Q = ctx.matmul_forward_scaled, ctx.matmul_forward_quantized
    other = G.Context(0)
    bad = [
        (S, (a, ctx.zeros(k + 1, n), out), {}, "B is"),
        (S, (a, b, ctx.zeros(m, n + 1)), {}, "the output"),
        (S, (a, b, out), dict(row_scales=ctx.zeros(1, m)), "the rows' scales"),
        (S, (a, b, out), dict(col_scales=ctx.zeros(n, 1)), "the columns' scales"),
        (S, (a, b, out), dict(bias=ctx.zeros(1, n + 1)), "the bias"),
        (S, (a, b, out), dict(residual=ctx.zeros(m + 1, n)), "the residual"),
        (S, (a, b, out), dict(pre=ctx.zeros(m, n + 1)), "pre"),
        (S, (a, b, out), dict(pre=out), "two outputs share"),
        (S, (a, b, out), dict(pre=pre, residual=pre), "the residual shares"),
        (S, (out, ctx.zeros(n, n), out), {}, "shares memory with an input"),
        (S, (a, b, out), dict(shift=64), "a shift of 64"),
        (S, (a, b, out), dict(limit=HALF + 1), "a limit of"),
        (S, (a, b, other.zeros(m, n)), {}, "another"),
        (S, (a, b, out), dict(row_scales=other.zeros(m, 1)), "another"),
        (S, (a, b, out), dict(residual=other.zeros(m, n)), "another"),
        (Q, (a, b, out), dict(levels=0), "0 levels"),
        (Q, (a, b, out), dict(levels=128), "128 levels"),
        (Q, (a, b, out), dict(quantized=ctx.zeros(m, k + 1)), "the quantized rows"),
        (Q, (a, b, out), dict(row_scales=cs), "the rows' scales"),
        (Q, (a, b, out), dict(quantized=a), "shares memory with an input"),
        (Q, (a, ctx.zeros(k, k), q), dict(quantized=q), "two outputs share"),
        (Q, (a, ctx.zeros(k, k), out), {}, "the output"),
        (Q, (a, ctx.zeros(k, k), ctx.zeros(m, k)), dict(quantized=q, residual=q), "the residual shares"),
    ]
    before = out.download()
    for f, args, kw, why in bad:
        with pytest.raises(G.GkrError, match=why):
            f(*args, **kw)
    assert np.array_equal(out.download(), before)
    S(a, b, out, row_scales=rs, col_scales=cs)  # and the context is as it was
    assert not out.download().any()
    other.close()
    assert G.lib().gkr_matmul_forward_scaled(ctx.handle, None, b.handle, None, None, 0, 0, None, None, None, out.handle) == 1
