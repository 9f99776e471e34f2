"""Causal attention of whole prompts (gkr_attention_prompt) against whole-number arithmetic: head layouts, packed
lengths from none to several blocks, int8-range and full-range words on each side, every output, agreement with
the attention over a cache, and what is refused."""
import numpy as np
import pytest

import gkr_mi355x as G
from test_gpu_attention import centered, words

pytestmark = pytest.mark.gpu
P = G.P


def attend(q, k, v, heads, kv, offset, log, cols):
    """One sequence's n rows, in whole numbers."""
    n, d = len(q), q.shape[1] // heads
    q, k, v = centered(q).reshape(n, heads, d), centered(k).reshape(n, kv, d), centered(v).reshape(n, kv, d)
    out, weighted = np.zeros((n, heads, d), np.int64), np.zeros((n, heads, d), np.int64)
    sums, scores = np.zeros((n, heads), np.int64), np.zeros((n, heads, cols), np.int64)
    for h in range(heads):
        c = h // (heads // kv)
        x = np.full((n, n), offset, np.int64)
        for j in range(4):  # eight bits of the keys at a time: sums of 2^30 2^8 2^8 stay below 2^53
            part = (k[:, c] >> (8 * j)) if j == 3 else (k[:, c] >> (8 * j)) & 255
            x = (x + ((q[:, h].astype(np.float64) @ part.T.astype(np.float64)).astype(np.int64) % P << (8 * j)) % P) % P
        x = np.tril(x)
        w = np.tril(np.int64(1) << np.minimum((x % (1 << log)) >> 16, 10))
        z, total = w.sum(axis=1)[:, None], w @ v[:, c]
        out[:, h] = np.sign(total) * ((2 * abs(total) + z) // (2 * z)) % P
        weighted[:, h], sums[:, h], scores[:, h, :n] = (total % P << 16) % P, ((z % P << 16) % P)[:, 0], x
    return out.reshape(n, -1), weighted.reshape(n, -1), sums, scores.reshape(n * heads, cols)


def check(ctx, counts, heads, kv, d, kinds=(True, True, True), offset=1 << 19, log=20, extra=3, seed=1, qkv=None):
    """kinds: whether q, k and v are int8-range."""
    rng = np.random.default_rng(seed + sum(counts) + 7 * d + heads)
    rows, cols = sum(counts), max(counts) + extra
    q, k, v = qkv or (words(rng, (rows, h * d), kind) for h, kind in zip((heads, kv, kv), kinds))
    m = [ctx.upload(t) for t in (q, k, v)]
    got = [ctx.synthetic(r, c, 0, 77) for r, c in ((rows, heads * d), (rows, heads * d), (rows, heads), (rows * heads, cols))]
    ctx.attention_prompt(*m, counts, heads, kv, got[0], score_offset=offset, table_log_size=log, weighted=got[1], sums=got[2],
                         scores=got[3])
    got = [t.download() for t in got]
    bare = ctx.synthetic(rows, heads * d, 0, 78)
    ctx.attention_prompt(*m, counts, heads, kv, bare, score_offset=offset, table_log_size=log)
    assert np.array_equal(bare.download(), got[0])
    row = 0
    for n in filter(None, counts):
        want = attend(q[row:row + n], k[row:row + n], v[row:row + n], heads, kv, offset, log or 20, cols)
        for name, g, w, per in zip(("out", "weighted", "sums", "scores"), got, want, (1, 1, 1, heads)):
            assert np.array_equal(g[row * per:(row + n) * per], w), (name, n)
        row += n


KINDS = [(True, True, True), (False, True, True), (False, False, False), (True, False, True), (True, True, False)]


@pytest.mark.parametrize("kinds", KINDS)
@pytest.mark.parametrize("heads,kv,d", [(1, 1, 1), (1, 1, 16), (9, 3, 64), (4, 4, 32), (5, 1, 80), (12, 1, 128), (14, 2, 96),
                                        (40, 8, 128), (17, 1, 17), (3, 3, 100), (2, 1, 200), (6, 2, 256)])
def test_head_layouts(gpu_ctx, heads, kv, d, kinds):
    check(gpu_ctx, [70], heads, kv, d, kinds)
    check(gpu_ctx, [3, 0, 65, 1], heads, kv, d, kinds)


@pytest.mark.parametrize("kinds", KINDS[:3])
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300, 700])
def test_lengths(gpu_ctx, n, kinds):
    check(gpu_ctx, [n], 5, 1, 64, kinds)
    check(gpu_ctx, [n, 1, n], 2, 2, 80, kinds)
    check(gpu_ctx, [1, n], 4, 1, 128, kinds)


@pytest.mark.parametrize("kinds", KINDS[:3])
def test_longer_than_one_round(gpu_ctx, kinds):
    check(gpu_ctx, [2100, 33], 6, 1, 64, kinds)
    check(gpu_ctx, [1300], 3, 1, 128, kinds)
    check(gpu_ctx, [600], 2, 1, 256, kinds)


@pytest.mark.parametrize("n", [127, 128, 129, 300])
def test_many_sequences(gpu_ctx, n):
    rng = np.random.default_rng(n)
    counts = [int(x) for x in rng.integers(0, 5, size=n)]
    counts[n // 2] = 90
    for kinds in KINDS[:3]:
        check(gpu_ctx, counts, 4, 2, 32, kinds)


@pytest.mark.parametrize("offset,log", [(0, 0), (P - 1, 20), (1 << 19, 16), (12345, 1), (1 << 23, 24), (P - (1 << 20), 20),
                                        (5 << 20, 22), (1 << 19, 17)])
@pytest.mark.parametrize("kinds", KINDS[:3])
def test_offsets_and_tables(gpu_ctx, offset, log, kinds):
    check(gpu_ctx, [100, 30], 4, 2, 64, kinds, offset, log)


@pytest.mark.parametrize("fill", [P - 1, P // 2, P // 2 + 1, P - 128, 127, 128, P - 129, 0])
def test_extreme_words(gpu_ctx, fill):
    """Every word the same: the largest sums of every digit, words that a centered byte just holds or does not."""
    for d in (16, 128, 256):
        for q in (fill, P - 128, 127):
            n = 130
            t = [np.full((n, h * d), w, dtype=np.uint32) for h, w in ((2, q), (1, fill), (1, fill))]
            check(gpu_ctx, [n], 2, 1, d, qkv=t, offset=0)
            check(gpu_ctx, [n - 10, 10], 2, 1, d, qkv=t, offset=P - 5)


def test_one_high_word(gpu_ctx):
    """A single word outside the int8 range, anywhere, is enough."""
    rng = np.random.default_rng(3)
    for which in range(3):
        for at in (0, 77, -1):
            t = [words(rng, (140, h * 64), True) for h in (4, 2, 2)]
            t[which].reshape(-1)[at] = 128
            check(gpu_ctx, [130, 10], 4, 2, 64, qkv=t)


@pytest.mark.parametrize("int8", [True, False])
def test_as_over_a_cache(gpu_ctx, int8):
    """The same tokens appended to a cache and attended a row each."""
    rng = np.random.default_rng(8)
    heads, kv, d, counts = 10, 2, 80, [100, 1, 64, 37]
    rows = sum(counts)
    q, k, v = (gpu_ctx.upload(words(rng, (rows, h * d), int8)) for h in (heads, kv, kv))
    shapes = ((rows, heads * d), (rows, heads * d), (rows, heads), (rows * heads, 100))
    a, b = ([gpu_ctx.synthetic(r, c, 0, s) for r, c in shapes] for s in (1, 2))
    gpu_ctx.attention_prompt(q, k, v, counts, heads, kv, a[0], 1 << 19, 0, a[1], a[2], a[3])
    cache = gpu_ctx.kv_cache(kv, d, n_pages=8, max_seqs=4, max_tokens=128, int8=int8)
    seqs = [cache.new_sequence() for _ in counts]
    cache.append(seqs, counts, k, v)
    gpu_ctx.attention_forward(cache, q, [s for s, n in zip(seqs, counts) for _ in range(n)], heads, b[0],
                              lens=[i + 1 for n in counts for i in range(n)], score_offset=1 << 19, weighted=b[1], sums=b[2],
                              scores=b[3])
    for x, y in zip(a, b):
        assert np.array_equal(x.download(), y.download())
    cache.free()


def test_refusals(gpu_ctx):
    ctx = gpu_ctx
    q, k, v, out = ctx.zeros(6, 32), ctx.zeros(6, 16), ctx.zeros(6, 16), ctx.zeros(6, 32)
    other = G.Context(0)
    F = ctx.attention_prompt
    bad = [((q, k, v, [5], 4, 2, out), {}, "q is"), ((q, k, v, [6, 1], 4, 2, out), {}, "q is"), ((q, k, v, [6], 4, 3, out), {}, "4 query heads"),
           ((q, k, v, [6], 0, 2, out), {}, "0 query heads"), ((q, k, v, [6], 4, 0, out), {}, "0 kv heads"),
           ((q, k, v, [6], 5, 5, out), {}, "not 5 heads"), ((q, k, v, [6], 4, 4, out), {}, "k is"),
           ((q, k, ctx.zeros(5, 16), [6], 4, 2, out), {}, "v is"), ((q, k, v, [6], 4, 2, ctx.zeros(6, 33)), {}, "the output"),
           ((q, k, v, [6], 4, 2, out), dict(weighted=out), "two outputs"), ((q, k, v, [6], 4, 2, q), {}, "shares memory"),
           ((q, k, v, [6], 4, 2, out), dict(sums=ctx.zeros(6, 2)), "sums"), ((q, k, v, [6], 4, 2, out), dict(weighted=ctx.zeros(6, 4)), "weighted"),
           ((q, k, v, [6], 4, 2, out), dict(scores=ctx.zeros(24, 5)), "5 columns"), ((q, k, v, [6], 4, 2, out), dict(scores=ctx.zeros(23, 6)), "scores"),
           ((q, k, v, [6], 4, 2, out), dict(score_offset=P), "canonical"), ((q, k, v, [6], 4, 2, out), dict(table_log_size=25), "2\\^25"),
           ((q, k, v, [131072], 4, 2, out), {}, "131072 tokens"), ((q, k, other.zeros(6, 16), [6], 4, 2, out), {}, "another"),
           ((ctx.zeros(1, 257), ctx.zeros(1, 257), ctx.zeros(1, 257), [1], 1, 1, ctx.zeros(1, 257)), {}, "at most 256")]
    for args, kw, why in bad:
        with pytest.raises(G.GkrError, match=why) as e:
            F(*args, **kw)
        assert e.value.code == 1
    F(q, k, v, [2, 0, 4], 4, 2, out)  # and the context goes on
    assert not out.download().any()
    other.close()


@pytest.mark.parametrize("table", [17, 18, 19, 20, 21, 24])
@pytest.mark.parametrize("spread", [1, 20, 60, 127])
def test_weights_of_every_place(gpu_ctx, spread, table):
    """Scores all in a few places or over all of the table and past it, small weights in no block, few or all."""
    rng = np.random.default_rng(spread + table)
    counts, heads, kv, d = [310, 70], 4, 2, 64
    rows = sum(counts)
    for lonely in (False, True):
        t = []
        for h in (heads, kv, kv):
            v = rng.integers(-spread, spread + 1, size=(rows, h * d))
            t.append(v)
        if lonely:  # one key far below the others, and one far above
            t[1][5], t[1][133] = -127, 127
            t[0][300, :d] = 127
        t = [np.where(v < 0, v + P, v).astype(np.uint32) for v in t]
        for offset in (1 << 19, 5 << 16, 0):
            check(gpu_ctx, counts, heads, kv, d, qkv=t, offset=offset, log=table)
