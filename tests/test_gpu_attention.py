"""Attention over the paged key-value cache (gkr_kv_cache_*, gkr_attention_forward) against whole-number
arithmetic: head layouts, lengths from none to many pages, appends token by token and in runs, sequences that
share rows, full-range and int8 caches, every output, and what is refused."""
import resource

import numpy as np
import pytest

import gkr_mi355x as G

pytestmark = pytest.mark.gpu
P = G.P


def words(rng, shape, int8):
    if not int8:
        return rng.integers(0, P, size=shape, dtype=np.uint32)
    v = rng.integers(-127, 128, size=shape)
    return np.where(v < 0, v + P, v).astype(np.uint32)


def centered(w):
    w = w.astype(np.int64)
    return np.where(w > (P >> 1), w - P, w)


def attend(q, k, v, heads, kv, offset, log, cols=None):
    """One row: q (heads * d), k and v (n, kv * d), in whole numbers."""
    n, d = len(k), len(q) // heads
    q, k, v = q.astype(np.int64).reshape(heads, d), k.astype(np.int64).reshape(n, kv, d), centered(v).reshape(n, kv, d)
    out, weighted, sums = np.zeros((heads, d), np.int64), np.zeros((heads, d), np.int64), np.zeros(heads, np.int64)
    scores = np.zeros((heads, cols or n), np.int64)
    for h in range(heads):
        c = h // (heads // kv)
        x = np.full(n, offset, np.int64)
        for e in range(d):
            x = (x + k[:, c, e] * q[h, e]) % P
        w = np.int64(1) << np.minimum((x % (1 << log)) >> 16, 10)
        z, total = int(w.sum()), (w[:, None] * v[:, c]).sum(0)
        if n:
            out[h] = np.sign(total) * ((2 * abs(total) + z) // (2 * z)) % P
        weighted[h], sums[h] = (total % P << 16) % P, (z % P << 16) % P
        scores[h, :n] = x
    return out.reshape(-1), weighted.reshape(-1), sums, scores


def fill(ctx, cache, rng, lens, width, int8, chunk=None):
    """Sequences of the given lengths, in appends of `chunk` tokens of every sequence at once."""
    seqs = [cache.new_sequence() for _ in lens]
    ks, vs = [words(rng, (n, width), int8) for n in lens], [words(rng, (n, width), int8) for n in lens]
    at = 0
    while at < max(lens):
        take = [max(0, min(n - at, chunk or n)) for n in lens]
        rows = [np.concatenate([t[at:at + c] for t, c in zip(ts, take)]) for ts in (ks, vs)]
        cache.append(seqs, take, ctx.upload(rows[0]), ctx.upload(rows[1]))
        at += chunk or max(lens)
    assert [cache.length(s) for s in seqs] == list(lens)
    return seqs, ks, vs


def run_and_check(ctx, cache, seqs, ks, vs, heads, kv, d, int8, offset=1 << 19, log=20, lens=None, extra=3, seed=1,
                  q=None):
    rng = np.random.default_rng(seed)
    n = len(seqs)
    q = words(rng, (n, heads * d), int8) if q is None else q
    seen = [len(k) for k in ks] if lens is None else lens
    cols = max(1, max(seen) + extra)
    ones = [ctx.synthetic(r, c, 0, 77) for r, c in ((n, heads * d), (n, heads * d), (n, heads), (n * heads, cols))]
    ctx.attention_forward(cache, ctx.upload(q), seqs, heads, ones[0], lens=lens, score_offset=offset, table_log_size=log,
                          weighted=ones[1], sums=ones[2], scores=ones[3])
    got = [m.download() for m in ones]
    bare = ctx.synthetic(n, heads * d, 0, 78)
    ctx.attention_forward(cache, ctx.upload(q), seqs, heads, bare, lens=lens, score_offset=offset, table_log_size=log)
    assert np.array_equal(bare.download(), got[0])
    for i in range(n):
        want = attend(q[i], ks[i][:seen[i]], vs[i][:seen[i]], heads, kv, offset, log or 20, cols)
        for name, g, w in zip(("out", "weighted", "sums"), got, want):
            assert np.array_equal(g[i], w), (name, i, seen[i])
        assert np.array_equal(got[3][i * heads:(i + 1) * heads], want[3]), ("scores", i, seen[i])


@pytest.mark.parametrize("int8", [True, False])
@pytest.mark.parametrize("heads,kv,d", [(1, 1, 1), (1, 1, 16), (9, 3, 64), (4, 4, 32), (5, 1, 80), (12, 1, 128),
                                        (14, 2, 33), (16, 1, 64), (17, 1, 40), (40, 1, 64), (8, 2, 256), (2, 1, 200)])
def test_head_layouts(gpu_ctx, heads, kv, d, int8):
    rng = np.random.default_rng(heads * 100 + d)
    lens = [1, 0, 63, 64, 65, 130, 300]
    cache = gpu_ctx.kv_cache(kv, d, n_pages=16, max_seqs=8, max_tokens=512, int8=int8)
    seqs, ks, vs = fill(gpu_ctx, cache, rng, lens, kv * d, int8)
    run_and_check(gpu_ctx, cache, seqs, ks, vs, heads, kv, d, int8)


@pytest.mark.parametrize("int8", [True, False])
@pytest.mark.parametrize("page_tokens", [64, 192, 1024])
@pytest.mark.parametrize("chunk", [1, 3, 64, 100])
def test_appends_and_pages(gpu_ctx, page_tokens, chunk, int8):
    rng = np.random.default_rng(chunk)
    lens = [200, 1, 77, 129] if chunk > 1 else [70, 1, 65, 64]
    cache = gpu_ctx.kv_cache(2, 64, n_pages=12, page_tokens=page_tokens, max_seqs=4, max_tokens=1024, int8=int8)
    seqs, ks, vs = fill(gpu_ctx, cache, rng, lens, 128, int8, chunk)
    run_and_check(gpu_ctx, cache, seqs, ks, vs, 6, 2, 64, int8)


@pytest.mark.parametrize("int8", [True, False])
@pytest.mark.parametrize("n", [1000, 5001, 20480])
def test_long_rows(gpu_ctx, n, int8):
    """Rows that many workgroups share and join."""
    rng = np.random.default_rng(n)
    cache = gpu_ctx.kv_cache(2, 64, n_pages=2 * n // 64 + 3, max_seqs=3, max_tokens=n, int8=int8)
    seqs, ks, vs = fill(gpu_ctx, cache, rng, [n, 3], 128, int8)
    run_and_check(gpu_ctx, cache, seqs, ks, vs, 10, 2, 64, int8)


def test_many_rows(gpu_ctx):
    """More rows than one launch takes, of mixed lengths."""
    rng = np.random.default_rng(7)
    lens = [int(v) for v in rng.integers(0, 200, size=300)]
    cache = gpu_ctx.kv_cache(1, 32, n_pages=1200, max_seqs=300, max_tokens=256, int8=True)
    seqs, ks, vs = fill(gpu_ctx, cache, rng, lens, 32, True)
    run_and_check(gpu_ctx, cache, seqs, ks, vs, 2, 1, 32, True)


@pytest.mark.parametrize("int8", [True, False])
def test_rows_of_one_sequence(gpu_ctx, int8):
    """A prompt's tokens, each seeing what came before it and none of it for the first."""
    rng = np.random.default_rng(9)
    cache = gpu_ctx.kv_cache(2, 64, n_pages=8, max_seqs=2, max_tokens=256, int8=int8)
    seqs, ks, vs = fill(gpu_ctx, cache, rng, [150], 128, int8)
    n = 150
    run_and_check(gpu_ctx, cache, seqs * n, ks * n, vs * n, 4, 2, 64, int8, lens=list(range(n)))


@pytest.mark.parametrize("offset,log", [(0, 0), (P - 1, 20), (1 << 19, 16), (12345, 1), (1 << 23, 24)])
def test_offsets_and_tables(gpu_ctx, offset, log):
    rng = np.random.default_rng(log)
    for int8 in (True, False):
        cache = gpu_ctx.kv_cache(1, 128, n_pages=8, max_seqs=2, max_tokens=256, int8=int8)
        seqs, ks, vs = fill(gpu_ctx, cache, rng, [140, 64], 128, int8)
        run_and_check(gpu_ctx, cache, seqs, ks, vs, 3, 1, 128, int8, offset, log)


def test_extreme_words(gpu_ctx):
    """Words of one repeated value: the digit sums, and the weighted sums, at their largest; halves are
    rounded away from zero."""
    for fill_word, int8 in ((P >> 1, False), ((P >> 1) + 1, False), (P - 1, False), (P - 128, True), (127, True), (1, True)):
        cache = gpu_ctx.kv_cache(1, 256, n_pages=40, max_seqs=1, max_tokens=2500, int8=int8)
        s = cache.new_sequence()
        n = 2500
        k, v = np.full((n, 256), fill_word, np.uint32), np.full((n, 256), fill_word, np.uint32)
        v[::2, ::3] = fill_word - 1 if fill_word in (1, 127) else (fill_word + 1) % P
        cache.append([s], [n], gpu_ctx.upload(k), gpu_ctx.upload(v))
        q = np.full((1, 512), fill_word, np.uint32)
        run_and_check(gpu_ctx, cache, [s], [k], [v], 2, 1, 256, int8, 10 << 16, 20, q=q)


def test_general_query_over_an_int8_cache(gpu_ctx):
    rng = np.random.default_rng(12)
    cache = gpu_ctx.kv_cache(2, 64, n_pages=8, max_seqs=2, max_tokens=256, int8=True)
    seqs, ks, vs = fill(gpu_ctx, cache, rng, [100, 200], 128, True)
    run_and_check(gpu_ctx, cache, seqs, ks, vs, 6, 2, 64, True, q=words(rng, (2, 384), False))
    q = words(rng, (2, 384), True)
    q[1, 383] = 1 << 25  # one word above the range, in the last head
    run_and_check(gpu_ctx, cache, seqs, ks, vs, 6, 2, 64, True, q=q)


def test_truncate_free_and_reuse(gpu_ctx):
    rng = np.random.default_rng(13)
    cache = gpu_ctx.kv_cache(1, 64, n_pages=6, max_seqs=3, max_tokens=256)
    seqs, ks, vs = fill(gpu_ctx, cache, rng, [200, 100], 64, False)
    assert cache.free_pages() == 0
    cache.truncate(seqs[0], 70)
    assert cache.free_pages() == 2
    k, v = words(rng, (60, 64), False), words(rng, (60, 64), False)
    cache.append([seqs[0]], [60], gpu_ctx.upload(k), gpu_ctx.upload(v))
    ks[0], vs[0] = np.concatenate([ks[0][:70], k]), np.concatenate([vs[0][:70], v])
    run_and_check(gpu_ctx, cache, seqs, ks, vs, 3, 1, 64, False)
    cache.free_sequence(seqs[1])
    with pytest.raises(G.GkrError):
        cache.length(seqs[1])
    s, k2, v2 = fill(gpu_ctx, cache, rng, [190], 64, False)
    run_and_check(gpu_ctx, cache, [seqs[0]] + s, [ks[0]] + k2, [vs[0]] + v2, 3, 1, 64, False)


def test_one_sequence_twice_in_an_append(gpu_ctx):
    rng = np.random.default_rng(14)
    cache = gpu_ctx.kv_cache(1, 32, n_pages=6, max_seqs=2, max_tokens=256)
    s, t = cache.new_sequence(), cache.new_sequence()
    k, v = words(rng, (150, 32), False), words(rng, (150, 32), False)
    cache.append([s, t, s], [61, 20, 69], gpu_ctx.upload(k), gpu_ctx.upload(v))
    rows = [list(range(61)) + list(range(81, 150)), list(range(61, 81))]
    run_and_check(gpu_ctx, cache, [s, t], [k[r] for r in rows], [v[r] for r in rows], 2, 1, 32, False)


def test_refusals(gpu_ctx):
    for kw in (dict(n_kv_heads=0), dict(head_dim=0), dict(head_dim=257), dict(n_pages=0), dict(page_tokens=32),
               dict(page_tokens=100), dict(max_seqs=0), dict(max_tokens=0), dict(max_tokens=(1 << 21) + 1)):
        with pytest.raises(G.GkrError) as e:
            gpu_ctx.kv_cache(**{**dict(n_kv_heads=2, head_dim=64, n_pages=4, max_seqs=2, max_tokens=200), **kw})
        assert e.value.code == 1, kw
    cache = gpu_ctx.kv_cache(2, 64, n_pages=4, max_seqs=2, max_tokens=200, int8=True)
    s, t = cache.new_sequence(), cache.new_sequence()
    with pytest.raises(G.GkrError) as e:
        cache.new_sequence()
    assert e.value.code == 4
    rng = np.random.default_rng(1)
    rows = words(rng, (100, 128), True)
    up = gpu_ctx.upload(rows)
    cache.append([s], [100], up, up)
    wide, bad = rows.copy(), rows.copy()
    bad[99, 127] = 128
    bad = gpu_ctx.upload(bad)
    wide = gpu_ctx.zeros(201, 128)
    for code, args in ((4, ([t], [201], wide, wide)),               # too long
                       (4, ([t, s], [90, 111], wide, wide)),        # the second is too long: the first is taken back
                       (4, ([t, t], [101, 100], wide, wide)),
                       (1, ([t], [99], up, up)),                    # rows and counts differ
                       (1, ([7], [100], up, up)), (1, ([t], [100], gpu_ctx.zeros(100, 64), up)),
                       (1, ([t], [100], up, bad)), (1, ([t], [100], bad, up))):
        before = cache.free_pages()
        with pytest.raises(G.GkrError) as e:
            cache.append(*args)
        assert e.value.code == code, (code, args)
        assert cache.length(s) == 100 and cache.length(t) == 0 and cache.free_pages() == before
    q, out = gpu_ctx.zeros(1, 256), gpu_ctx.zeros(1, 256)
    other = G.Context(0)
    for kw in (dict(seqs=[9]), dict(n_heads=3), dict(n_heads=0), dict(seqs=[s, t]), dict(lens=[101]),
               dict(out=gpu_ctx.zeros(1, 255)), dict(out=q), dict(weighted=out), dict(sums=gpu_ctx.zeros(1, 5)),
               dict(scores=gpu_ctx.zeros(4, 99)), dict(scores=gpu_ctx.zeros(3, 100)), dict(score_offset=P),
               dict(table_log_size=25), dict(out=other.zeros(1, 256))):
        with pytest.raises(G.GkrError) as e:
            gpu_ctx.attention_forward(**{**dict(cache=cache, q=q, seqs=[s], n_heads=4, out=out), **kw})
        assert e.value.code == 1, kw
    with pytest.raises(G.GkrError):
        other.attention_forward(cache, q, [s], 4, out)
    mine = other.kv_cache(1, 16, n_pages=2, max_seqs=1, max_tokens=64)
    held = mine.new_sequence()
    other.close()  # a cache that outlives its context is refused, and can be freed
    with pytest.raises(G.GkrError):
        mine.length(held)
    mine.free()
    gpu_ctx.attention_forward(cache, q, [s], 4, out)
    gpu_ctx.synchronize()


@pytest.mark.parametrize("callers_stream", [False, True])
@pytest.mark.parametrize("int8", [True, False])
@pytest.mark.parametrize("launch", [1, 2])
def test_refused_append(launch, int8, callers_stream):
    """A launch of an append that the runtime refuses (the page table's, the tokens') fails that call, whichever
    thread issues it, and leaves lengths and pages as they were; the same append then goes through."""
    ctx = G.Context(0, stream=0) if callers_stream else G.Context(0)
    rng = np.random.default_rng(launch)
    cache = ctx.kv_cache(2, 64, n_pages=12, max_seqs=3, max_tokens=512, int8=int8)
    seqs, ks, vs = fill(ctx, cache, rng, [70, 0], 128, int8)
    for turn in range(3):
        counts = [100, 65] if turn < 2 else [3, 1]  # the last needs no page: its first launch is the tokens'
        k, v = words(rng, (sum(counts), 128), int8), words(rng, (sum(counts), 128), int8)
        up = ctx.upload(k), ctx.upload(v)
        before = [cache.length(s) for s in seqs], cache.free_pages()
        ctx.debug(G.DEBUG_REFUSE_LAUNCH, launch if turn < 2 else 1)
        with pytest.raises(G.GkrError) as e:
            cache.append(seqs, counts, *up)
        assert e.value.code == 2
        assert ([cache.length(s) for s in seqs], cache.free_pages()) == before
        ctx.debug(G.DEBUG_REFUSE_LAUNCH, 0)
        cache.append(seqs, counts, *up)
        for i, part in enumerate((slice(0, counts[0]), slice(counts[0], None))):
            ks[i], vs[i] = np.concatenate([ks[i], k[part]]), np.concatenate([vs[i], v[part]])
        run_and_check(ctx, cache, seqs, ks, vs, 6, 2, 64, int8, seed=turn)
    cache.free()
    ctx.close()


def test_append_behind_a_refused_launch():
    """A launch refused on the launcher thread whose call has returned is told by an append behind it, which then
    keeps nothing."""
    ctx = G.Context(0)
    rng = np.random.default_rng(5)
    cache = ctx.kv_cache(1, 64, n_pages=8, max_seqs=2, max_tokens=256)
    seqs, ks, vs = fill(ctx, cache, rng, [30], 64, False)
    a, b, out = ctx.synthetic(1, 64, 0, 1), ctx.synthetic(64, 96, 1, 2), ctx.zeros(1, 96)
    ctx.matmul_forward_fused(a, b, out)
    k, v = words(rng, (64, 64), False), words(rng, (64, 64), False)
    up = ctx.upload(k), ctx.upload(v)
    before = cache.length(seqs[0]), cache.free_pages()
    ctx.debug(G.DEBUG_REFUSE_LAUNCH, 1)
    with pytest.raises(G.GkrError) as e:  # by the product itself where its launch was issued in time
        ctx.matmul_forward_fused(a, b, out)
        cache.append(seqs, [64], *up)
    assert e.value.code == 2
    assert (cache.length(seqs[0]), cache.free_pages()) == before
    ctx.debug(G.DEBUG_REFUSE_LAUNCH, 0)
    cache.append(seqs, [64], *up)
    run_and_check(ctx, cache, seqs, [np.concatenate([ks[0], k])], [np.concatenate([vs[0], v])], 2, 1, 64, False)
    cache.free()
    ctx.close()


def test_refused_pools(gpu_ctx):
    """Pools whose size passes 64 bits (the first one's is 2^64, nothing after the wrap) or any device's memory."""
    for n_pages, page_tokens, heads, dim, int8 in ((1 << 26, 65536, 4096, 256, False), ((1 << 26) + 1, 65536, 4096, 256, False),
                                                   (1 << 28, 65536, 4096, 256, True), ((1 << 10) + 1, 65536, 4096, 256, False)):
        with pytest.raises(G.GkrError) as e:
            gpu_ctx.kv_cache(heads, dim, n_pages=n_pages, page_tokens=page_tokens, max_seqs=1, max_tokens=64, int8=int8)
        assert e.value.code == 1, (n_pages, int8)


@pytest.mark.parametrize("callers_stream", [False, True])
@pytest.mark.parametrize("int8", [True, False])
def test_every_refused_launch_is_told(int8, callers_stream):
    """A refused launch of attention (its kernel's, its join's) fails the call or the wait behind it; the next
    call writes the whole output again."""
    ctx = G.Context(0, stream=0) if callers_stream else G.Context(0)
    rng = np.random.default_rng(3)
    cache = ctx.kv_cache(2, 64, n_pages=90, max_seqs=1, max_tokens=5001, int8=int8)
    seqs, ks, vs = fill(ctx, cache, rng, [5001], 128, int8)
    q = words(rng, (1, 384), int8)
    qd = ctx.upload(q)
    want = attend(q[0], ks[0], vs[0], 6, 2, 1 << 19, 20)[0]
    for launch in (1, 2):
        for wait in (ctx.synchronize, lambda: out.download()):
            out = ctx.synthetic(1, 384, 0, launch)
            ctx.debug(G.DEBUG_REFUSE_LAUNCH, launch)
            with pytest.raises(G.GkrError) as e:
                ctx.attention_forward(cache, qd, seqs, 6, out, score_offset=1 << 19)
                wait()
            assert e.value.code == 2, launch
            ctx.debug(G.DEBUG_REFUSE_LAUNCH, 0)
            out = ctx.synthetic(1, 384, 0, launch + 10)
            ctx.attention_forward(cache, qd, seqs, 6, out, score_offset=1 << 19)
            assert np.array_equal(out.download()[0], want), launch
    cache.free()
    ctx.close()


@pytest.mark.parametrize("int8,kv", [(True, 4), (False, 1)])
@pytest.mark.parametrize("short", [0, 1, 256])
def test_longest_shares(gpu_ctx, int8, kv, short):
    """128 rows of 131072 tokens, about the steps at which a workgroup's share is longest (255 of 256 tokens) and
    then more workgroups than fit; weights and values whose lowest digits are -128, so that a share's digit sums
    are at their largest, beside random ones."""
    d, n, rows = 16, 131072, 128
    rng = np.random.default_rng(short)
    cache = gpu_ctx.kv_cache(kv, d, n_pages=n // 1024, page_tokens=1024, max_seqs=1, max_tokens=n, int8=int8)
    k, v = words(rng, (n, kv * d), int8), words(rng, (n, kv * d), int8)
    v[:, ::2] = P - (128 if int8 else 128 * 65793)
    seq = cache.new_sequence()
    cache.append([seq], [n], gpu_ctx.upload(k), gpu_ctx.upload(v))
    lens = [n] * rows
    lens[77] = 256 * (512 - short) - (short != 0)
    q = np.zeros((rows, kv * d), np.uint32)  # scores are the offset: weights of 128
    q[5], q[77] = words(rng, (kv * d,), int8), words(rng, (kv * d,), int8)
    out, weighted, sums = (gpu_ctx.synthetic(rows, c, 0, 1) for c in (kv * d, kv * d, kv))
    gpu_ctx.attention_forward(cache, gpu_ctx.upload(q), [seq] * rows, kv, out, lens=lens, score_offset=7 << 16,
                              weighted=weighted, sums=sums)
    got = out.download(), weighted.download(), sums.download()
    for i in (0, 5, 77):
        want = attend(q[i], k[:lens[i]], v[:lens[i]], kv, kv, 7 << 16, 20)
        for j in (range(rows) if i == 0 else (i,)):
            if i == 0 and j in (5, 77):
                continue
            for g, w in zip(got, want):
                assert np.array_equal(g[j], w), j
    cache.free()


def test_pools_that_do_not_fit_take_no_host_memory(gpu_ctx):
    """The most pages that can be asked for, 4 TB of pools: refused before the host's book of them is made."""
    before = resource.getrusage(resource.RUSAGE_SELF).ru_maxrss
    with pytest.raises(G.GkrError) as e:
        gpu_ctx.kv_cache(1, 1, n_pages=(1 << 32) - 1, max_seqs=1, max_tokens=64, int8=True)
    assert e.value.code == 4
    assert resource.getrusage(resource.RUSAGE_SELF).ru_maxrss - before < 1 << 20  # KiB
