"""The fused product and the gated block (gkr_matmul_forward_fused, gkr_gated_forward) against whole-number
arithmetic: every activation, with and without bias, residual and parts, rows on both sides of each rule on
sizes, int8-range and general operands, and what is refused."""
import ctypes

import numpy as np
import pytest

import gkr_mi355x as G

pytestmark = pytest.mark.gpu
P = G.P
RELU, GELU, SIGMOID, SOFTMAX, SILU = 1, 2, 3, 4, 5


def product(a, b):
    """A B mod P: bytes of A by 16-bit halves of B, every partial sum below 2^53."""
    a, b = a.astype(np.int64), b.astype(np.int64)
    out = np.zeros((a.shape[0], b.shape[1]), np.int64)
    if np.all((b < 128) | (b >= P - 128)):  # int8-range B as signed numbers, 16-bit halves of A
        c = np.where(b > P // 2, b - P, b).astype(np.float64)
        for i in range(2):
            s = ((a >> (16 * i)) & 0xFFFF).astype(np.float64) @ c
            out = (out + s.astype(np.int64) % P * pow(2, 16 * i, P)) % P
        return out
    for i in range(4):
        for j in range(2):
            s = ((a >> (8 * i)) & 255).astype(np.float64) @ ((b >> (16 * j)) & 0xFFFF).astype(np.float64)
            out = (out + s.astype(np.int64) % P * pow(2, 8 * i + 16 * j, P)) % P
    return out


def activate(z, act, log):
    if act == 0:
        return z
    if act == RELU:
        return np.where(z <= (1 << 30) - 1, z, 0)
    log = log or (20 if act == SOFTMAX else 16)
    return G.activation_table(act, log).astype(np.int64)[z % (1 << log)]


def words(rng, shape, kind):
    if kind == 0:
        return rng.integers(0, P, size=shape, dtype=np.uint32)
    v = rng.integers(-127, 128, size=shape)
    return np.where(v < 0, v + P, v).astype(np.uint32)


def check_fused(ctx, m, k, n, xk, wk, act=0, log=0, bias=True, residual=True, pre=True, seed=1, x=None):
    rng = np.random.default_rng(seed + m * 31 + k * 7 + n)
    A, B = words(rng, (m, k), xk) if x is None else x, words(rng, (k, n), wk)
    bv, rv = words(rng, (1, n), 0), words(rng, (m, n), 0)
    out, z = ctx.zeros(m, n), ctx.zeros(m, n)
    a, b, bm, rm = ctx.upload(A), ctx.upload(B), ctx.upload(bv), ctx.upload(rv)
    ref = product(A, B)
    if bias:
        ref = (ref + bv) % P
    y = activate(ref, act, log)
    if residual:
        y = (y + rv) % P
    for _ in range(2):  # the second finds the weight's planes built
        ctx.matmul_forward_fused(a, b, out, bias=bm if bias else None, activation=act, table_log_size=log,
                                 residual=rm if residual else None, pre=z if pre else None)
        assert np.array_equal(out.download(), y)
        if pre:
            assert np.array_equal(z.download(), ref)


def check_gated(ctx, m, k, n, xk, wk, act=SILU, log=0, trace=True, seed=2):
    rng = np.random.default_rng(seed + m * 31 + k * 7 + n)
    A, Wg, Wu = words(rng, (m, k), xk), words(rng, (k, n), wk), words(rng, (k, n), wk)
    a, wg, wu = ctx.upload(A), ctx.upload(Wg), ctx.upload(Wu)
    out, g, t, u = (ctx.zeros(m, n) for _ in range(4))
    gate, up = product(A, Wg), product(A, Wu)
    ac = activate(gate, act, log)
    for _ in range(2):
        ctx.gated_forward(a, wg, wu, out, activation=act, table_log_size=log, **(dict(gate=g, act=t, up=u) if trace else {}))
        assert np.array_equal(out.download(), ac * up % P)
        if trace:
            assert np.array_equal(g.download(), gate)
            assert np.array_equal(t.download(), ac)
            assert np.array_equal(u.download(), up)


@pytest.mark.parametrize("act,log", [(0, 0), (RELU, 0), (GELU, 0), (SIGMOID, 0), (SOFTMAX, 0), (SILU, 0), (SILU, 1),
                                     (GELU, 20)])
def test_activations(gpu_ctx, act, log):
    for bias, residual, pre in ((True, True, True), (False, False, False), (False, True, False)):
        check_fused(gpu_ctx, 5, 100, 70, 0, 1, act, log, bias, residual, pre)


@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 8, 9, 16, 17, 32, 33, 64, 65, 100, 129, 300])
@pytest.mark.parametrize("k,n", [(1, 1), (33, 31), (576, 192), (1000, 333)])
def test_row_counts(gpu_ctx, m, k, n):
    for xk in (1, 0):
        for wk in (1, 0):
            check_fused(gpu_ctx, m, k, n, xk, wk, GELU)
            check_gated(gpu_ctx, m, k, n, xk, wk)


# long sums (several splits or passes of K), one row to many
@pytest.mark.parametrize("m,k,n", [(1, 40001, 40), (3, 20000, 65), (8, 13825, 31), (40, 17000, 96), (70, 33001, 33),
                                   (200, 9001, 260), (2, 140001, 3), (33, 131073, 5)])
def test_long_sums(gpu_ctx, m, k, n):
    for xk, wk in ((1, 1), (0, 1), (0, 0)):
        check_fused(gpu_ctx, m, k, n, xk, wk, 0)
    check_gated(gpu_ctx, m, k, n, 0, 1)


@pytest.mark.parametrize("m,k,n", [(1, 300, 13824), (512, 700, 1100), (300, 4000, 2100), (64, 2048, 5120)])
def test_wide(gpu_ctx, m, k, n):
    for xk in (1, 0):
        check_fused(gpu_ctx, m, k, n, xk, 1, 0)
        check_gated(gpu_ctx, m, k, n, xk, 1)


# few rows by more column tiles than the chip has CUs
@pytest.mark.parametrize("m,k,n", [(1, 1025, 8225), (2, 700, 9001), (4, 16400, 8193), (7, 500, 8500), (16, 300, 8300)])
def test_few_rows_many_columns(gpu_ctx, m, k, n):
    for xk, wk in ((1, 1), (0, 1), (0, 0)):
        check_fused(gpu_ctx, m, k, n, xk, wk, RELU)
        if k < 2000:
            check_gated(gpu_ctx, m, k, n, xk, wk)


# more than 64 rows and enough work for blocks of 8 x 8 tiles, for all rows streamed through one workgroup
# where they have one plane, and for K splits; ragged edges, and K steps that end inside a stage of four
@pytest.mark.parametrize("m,k,n", [(100, 5121, 5101), (200, 2605, 5101), (130, 1130, 5131), (260, 500, 4099),
                                   (513, 2001, 2003), (300, 100, 9001)])
def test_blocks(gpu_ctx, m, k, n):
    for xk in (1, 0):
        check_fused(gpu_ctx, m, k, n, xk, 1, GELU)
        check_gated(gpu_ctx, m, k, n, xk, 1)


# five to sixteen K splits (more than are joined at a time) by few columns
@pytest.mark.parametrize("m,k,n", [(200, 13825, 1030), (520, 9001, 1030), (100, 33001, 1111), (270, 20001, 900)])
def test_many_splits(gpu_ctx, m, k, n):
    for xk in (1, 0):
        check_fused(gpu_ctx, m, k, n, xk, 1, SIGMOID)
        check_gated(gpu_ctx, m, k, n, xk, 1)


@pytest.mark.parametrize("m,k,n", [(100, 2605, 3001), (130, 500, 5131), (300, 100, 4099), (513, 801, 2003)])
def test_blocks_of_general_weights(gpu_ctx, m, k, n):
    for xk in (1, 0):
        check_fused(gpu_ctx, m, k, n, xk, 0, SILU)
    rng = np.random.default_rng(m)
    for bits in (12, 20):  # two and three planes
        A, B = words(rng, (m, k), 0), rng.integers(0, 1 << bits, size=(k, n), dtype=np.uint32)
        out = gpu_ctx.zeros(m, n)
        gpu_ctx.matmul_forward_fused(gpu_ctx.upload(A), gpu_ctx.upload(B), out)
        assert np.array_equal(out.download(), product(A, B))


@pytest.mark.parametrize("m,k", [(1, 40000), (8, 9000), (64, 9000), (260, 5000)])
@pytest.mark.parametrize("fill", [P - 1, P // 2, P // 2 + 1, P - 128, 127])
def test_extreme_words(gpu_ctx, m, k, fill):
    """Operands of one repeated word: every digit sum at its largest."""
    n = 40
    A, B = np.full((m, k), fill, np.uint32), np.full((k, n), P - 128, np.uint32)
    want = np.full((m, n), (fill - P if fill > P // 2 else fill) * -128 * k % P)
    out = gpu_ctx.zeros(m, n)
    gpu_ctx.matmul_forward_fused(gpu_ctx.upload(A), gpu_ctx.upload(B), out)
    assert np.array_equal(out.download(), want)
    B[:] = P // 2 + 1
    c = P // 2 + 1 - P
    gpu_ctx.matmul_forward_fused(gpu_ctx.upload(A), gpu_ctx.upload(B), out)
    assert np.array_equal(out.download(), np.full((m, n), (fill - P if fill > P // 2 else fill) * c * k % P))


@pytest.mark.parametrize("m,k,n", [(2, 65, 40), (30, 600, 100), (300, 300, 300), (260, 2000, 500)])
def test_one_high_word(gpu_ctx, m, k, n):
    """A single word outside the int8 range, in the last place, after a call without one and before another."""
    rng = np.random.default_rng(4)
    x = words(rng, (m, k), 1)
    check_fused(gpu_ctx, m, k, n, 1, 1, x=x)
    x[-1, -1] = 1 << 20
    check_fused(gpu_ctx, m, k, n, 1, 1, x=x)
    check_fused(gpu_ctx, m, k, n, 1, 1, seed=9)


@pytest.mark.parametrize("m,k,n", [(1, 4000, 500), (40, 4000, 500), (300, 900, 700)])
def test_weights_of_two_and_three_planes(gpu_ctx, m, k, n):
    rng = np.random.default_rng(6)
    for bits in (12, 20):
        B = rng.integers(0, 1 << bits, size=(k, n), dtype=np.uint32)
        A = words(rng, (m, k), 0)
        out = gpu_ctx.zeros(m, n)
        gpu_ctx.matmul_forward_fused(gpu_ctx.upload(A), gpu_ctx.upload(B), out)
        assert np.array_equal(out.download(), product(A, B))
        H = gpu_ctx.zeros(m, n)  # a gate and an up weight of different plane counts
        W2 = words(rng, (k, n), 1)
        gpu_ctx.gated_forward(gpu_ctx.upload(A), gpu_ctx.upload(B), gpu_ctx.upload(W2), H, activation=RELU)
        assert np.array_equal(H.download(), activate(product(A, B), RELU, 0) * product(A, W2) % P)


@pytest.mark.parametrize("m", [1, 20, 300])
def test_residual_in_place(gpu_ctx, m):
    rng = np.random.default_rng(5)
    A, B, R = words(rng, (m, 500), 0), words(rng, (500, 130), 1), words(rng, (m, 130), 0)
    a, b, h = gpu_ctx.upload(A), gpu_ctx.upload(B), gpu_ctx.upload(R)
    ref = R.astype(np.int64)
    for _ in range(3):
        gpu_ctx.matmul_forward_fused(a, b, h, residual=h)
        ref = (ref + product(A, B)) % P
        assert np.array_equal(h.download(), ref)


def test_changed_weights_and_outputs(gpu_ctx):
    """An output that was a weight is no longer taken from its old planes."""
    rng = np.random.default_rng(8)
    A, B, W = words(rng, (4, 64), 1), words(rng, (64, 64), 1), words(rng, (64, 64), 1)
    a, b, w, out = gpu_ctx.upload(A), gpu_ctx.upload(B), gpu_ctx.upload(W), gpu_ctx.zeros(4, 64)
    gpu_ctx.matmul_forward_fused(a, w, out)
    gpu_ctx.matmul_forward_fused(b, b, w)
    gpu_ctx.matmul_forward_fused(a, w, out)
    assert np.array_equal(out.download(), product(A, product(B, B)))


def test_refusals(gpu_ctx):
    a, b, out = gpu_ctx.zeros(3, 40), gpu_ctx.zeros(40, 50), gpu_ctx.zeros(3, 50)
    other = G.Context(0)
    stray = other.zeros(3, 50)
    part = gpu_ctx.wrap_device(out.device_ptr + 4, 1, 50)
    half = gpu_ctx.wrap_device(out.device_ptr, 2, 50)
    bad = [dict(bias=gpu_ctx.zeros(1, 49)), dict(bias=gpu_ctx.zeros(3, 50)), dict(residual=gpu_ctx.zeros(3, 51)),
           dict(pre=gpu_ctx.zeros(2, 50)), dict(pre=out), dict(residual=stray), dict(pre=stray), dict(bias=part),
           dict(pre=half), dict(activation=6), dict(activation=SILU, table_log_size=25)]
    for kw in bad:
        with pytest.raises(G.GkrError) as e:
            gpu_ctx.matmul_forward_fused(a, b, out, **kw)
        assert e.value.code == 1, kw
    shifted = gpu_ctx.wrap_device(gpu_ctx.zeros(4, 50).device_ptr, 3, 50)
    for args in ((a, a, out), (a, b, a), (a, b, gpu_ctx.zeros(3, 40)), (stray, b, out)):
        with pytest.raises(G.GkrError):
            gpu_ctx.matmul_forward_fused(*args)
    with pytest.raises(G.GkrError):
        gpu_ctx.matmul_forward_fused(a, b, out, residual=gpu_ctx.wrap_device(out.device_ptr + 200, 3, 50))
    for kw in (dict(gate=out), dict(act=gpu_ctx.zeros(3, 49)), dict(up=stray), dict(activation=9)):
        with pytest.raises(G.GkrError):
            gpu_ctx.gated_forward(a, b, b, out, **kw)
    with pytest.raises(G.GkrError):
        gpu_ctx.gated_forward(a, b, gpu_ctx.zeros(40, 51), out)
    with pytest.raises(G.GkrError):
        gpu_ctx.zeros(0, 3)
    del shifted
    gpu_ctx.matmul_forward_fused(a, b, out)  # and the context goes on
    assert not out.download().any()
    other.close()


def test_refused_launch_leaves_the_context_usable(gpu_ctx):
    for m in (1, 40, 300):
        a, b, out = gpu_ctx.synthetic(m, 64, 0, 1), gpu_ctx.synthetic(64, 96, 1, 2), gpu_ctx.zeros(m, 96)
        gpu_ctx.matmul_forward_fused(a, b, out)
        want = out.download()
        for nth in (1, 2):
            gpu_ctx.debug(G.DEBUG_REFUSE_LAUNCH, nth)
            try:
                gpu_ctx.matmul_forward_fused(a, b, out)
                gpu_ctx.matmul_forward_fused(a, b, out)
                gpu_ctx.synchronize()
            except G.GkrError:
                pass
            gpu_ctx.debug(G.DEBUG_REFUSE_LAUNCH, 0)
            try:
                gpu_ctx.matmul_forward_fused(a, b, out)
            except G.GkrError:  # the launcher thread's refusal, told by the next call
                gpu_ctx.matmul_forward_fused(a, b, out)
            assert np.array_equal(out.download(), want)


def test_on_the_callers_stream():
    """A context on a stream of the caller's (one of its own, then the default one): ordered with the copies
    and fills that the caller puts on it before and behind each call."""
    G.lib()
    hip = ctypes.CDLL("libamdhip64.so.7")  # the runtime the library has loaded
    vp, size = ctypes.c_void_p, ctypes.c_size_t
    copy, fill, stream = hip.hipMemcpyAsync, hip.hipMemsetAsync, vp()
    copy.argtypes, fill.argtypes = [vp, vp, size, ctypes.c_int, vp], [vp, ctypes.c_int, size, vp]
    assert hip.hipStreamCreate(ctypes.byref(stream)) == 0
    to_device, within_device = 1, 3
    rng = np.random.default_rng(3)
    B = words(rng, (700, 300), 1)
    for s in (stream, vp()):
        ctx = G.Context(0, stream=s.value or 0)
        a, b, o, kept = ctx.zeros(4, 700), ctx.upload(B), ctx.zeros(4, 300), ctx.zeros(4, 300)
        for i in range(20):
            A = words(rng, (4, 700), i % 2)
            assert copy(a.device_ptr, A.ctypes.data, A.nbytes, to_device, s) == 0
            ctx.matmul_forward_fused(a, b, o)
            assert copy(kept.device_ptr, o.device_ptr, 4800, within_device, s) == 0
            assert fill(o.device_ptr, 0, 4800, s) == 0
            assert hip.hipStreamSynchronize(s) == 0
            assert np.array_equal(kept.download(), product(A, B)) and not o.download().any()
        ctx.close()
    assert hip.hipStreamDestroy(stream) == 0


def test_captured_into_a_graph():
    """Products of one row, 40 and 200 rows, the gated block, and attention with its join, captured once and
    replayed over changed inputs, int8-range and general in turn, with calls of the context's own between."""
    from test_gpu_attention import attend

    G.lib()
    hip = ctypes.CDLL("libamdhip64.so.7")
    vp, size = ctypes.c_void_p, ctypes.c_size_t
    copy, stream, graph, run = hip.hipMemcpyAsync, vp(), vp(), vp()
    copy.argtypes = [vp, vp, size, ctypes.c_int, vp]
    hip.hipStreamBeginCapture.argtypes, hip.hipStreamEndCapture.argtypes = [vp, ctypes.c_int], [vp, ctypes.POINTER(vp)]
    hip.hipGraphInstantiate.argtypes = [ctypes.POINTER(vp), vp, vp, vp, size]
    hip.hipGraphLaunch.argtypes, hip.hipGraphExecDestroy.argtypes, hip.hipGraphDestroy.argtypes = [vp, vp], [vp], [vp]
    assert hip.hipStreamCreate(ctypes.byref(stream)) == 0
    ctx = G.Context(0, stream=stream.value)
    rng = np.random.default_rng(11)
    k, n, kv_len = 500, 300, 2000
    W, V = words(rng, (k, n), 1), words(rng, (k, n), 1)
    w, v = ctx.upload(W), ctx.upload(V)
    rows = (1, 40, 200)
    xs = {m: ctx.zeros(m, k) for m in rows}
    fused, gated = {m: ctx.zeros(m, n) for m in rows}, {m: ctx.zeros(m, n) for m in rows}
    keys, values = words(rng, (kv_len, 64), 0), words(rng, (kv_len, 64), 0)
    cache = ctx.kv_cache(1, 64, n_pages=40, max_seqs=1, max_tokens=kv_len)
    seq = cache.new_sequence()
    cache.append([seq], [kv_len], ctx.upload(keys), ctx.upload(values))
    q, att = ctx.zeros(1, 128), ctx.zeros(1, 128)

    def calls():
        for m in rows:
            ctx.matmul_forward_fused(xs[m], w, fused[m], activation=GELU)
            ctx.gated_forward(xs[m], w, v, gated[m])
        ctx.attention_forward(cache, q, [seq], 2, att, score_offset=1 << 19)

    calls()  # planes, tables and buffers are there from here on
    ctx.synchronize()
    thread_local = 1
    assert hip.hipStreamBeginCapture(stream, thread_local) == 0
    calls()
    assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(run), graph, None, None, 0) == 0
    for turn in range(4):
        host = {m: words(rng, (m, k), turn % 2) for m in rows}
        Q = words(rng, (1, 128), 0)
        for dev, h in [(xs[m], host[m]) for m in rows] + [(q, Q)]:
            assert copy(dev.device_ptr, h.ctypes.data, h.nbytes, 1, stream) == 0
        assert hip.hipGraphLaunch(run, stream) == 0
        got = [{m: o[m].download() for m in rows} for o in (fused, gated)] + [att.download()]
        for m in rows:
            z = product(host[m], W)
            assert np.array_equal(got[0][m], activate(z, GELU, 0))
            assert np.array_equal(got[1][m], activate(z, SILU, 0) * product(host[m], V) % P)
        assert np.array_equal(got[2][0], attend(Q[0], keys, values, 2, 1, 1 << 19, 20)[0])
        if turn != 2:  # an eager call between two replays
            other = words(rng, (40, k), 1 - turn % 2)
            out = ctx.zeros(40, n)
            ctx.matmul_forward_fused(ctx.upload(other), w, out)
            assert np.array_equal(out.download(), product(other, W))
    assert hip.hipGraphExecDestroy(run) == 0 and hip.hipGraphDestroy(graph) == 0
    cache.free()
    ctx.close()
    assert hip.hipStreamDestroy(stream) == 0


# short sums, so that blocks of 8 x 8 tiles are nearly all end: lanes exchange their sums through LDS, half of a
# wave's tiles at a time; K splits leave them as parts (the last two)
@pytest.mark.parametrize("m,k,n", [(512, 33, 8192), (300, 65, 6001), (257, 1, 4129), (520, 9001, 1030), (200, 13825, 1030)])
def test_block_ends(gpu_ctx, m, k, n):
    rng = np.random.default_rng(m)
    for xk in (1, 0):
        A, B, C2, R = words(rng, (m, k), xk), words(rng, (k, n), 1), words(rng, (k, n), 1), words(rng, (m, n), 0)
        a, b, c2, h, z = (gpu_ctx.upload(x) for x in (A, B, C2, R, R))
        p, q, ref = product(A, B), product(A, C2), R.astype(np.int64)
        for _ in range(3):  # added in place: a word that another lane's reads or stores went past shows
            gpu_ctx.matmul_forward_fused(a, b, h, residual=h, pre=z)
            ref = (ref + p) % P
            assert np.array_equal(h.download(), ref) and np.array_equal(z.download(), p)
        out, parts = gpu_ctx.upload(R), [gpu_ctx.upload(R) for _ in range(3)]
        gpu_ctx.gated_forward(a, b, c2, out, activation=RELU, gate=parts[0], act=parts[1], up=parts[2])
        act = activate(p, RELU, 0)
        for got, want in zip([out] + parts, (act * q % P, p, act, q)):
            assert np.array_equal(got.download(), want)


def test_sixteen_rows_of_the_most_columns(gpu_ctx):
    """16 x 2^26 words, an output of 2^32 bytes, and one column fewer: the last words are there, with their
    residual, and so are those of a gated block."""
    rng = np.random.default_rng(7)
    for n in (1 << 26, (1 << 26) - 1):
        A, tail = words(rng, (16, 1), 1), 70
        a, b = gpu_ctx.upload(A), gpu_ctx.synthetic(1, n, 1, 3)
        res, out = gpu_ctx.synthetic(16, n, 0, 4), gpu_ctx.synthetic(16, n, 0, 5)

        def last(m, row):  # the last words of a row
            return gpu_ctx.wrap_device(m.device_ptr + 4 * (row * n + n - tail), 1, tail).download().astype(np.int64)[0]

        B = last(b, 0)
        gpu_ctx.matmul_forward_fused(a, b, out, residual=res)
        for row in (0, 7, 15):
            assert np.array_equal(last(out, row), (int(A[row, 0]) * B + last(res, row)) % P)
        gpu_ctx.gated_forward(a, b, b, out, activation=0)
        for row in (0, 15):
            z = int(A[row, 0]) * B % P
            assert np.array_equal(last(out, row), z * z % P)


@pytest.mark.parametrize("callers_stream", [False, True])
@pytest.mark.parametrize("launch", [1, 2])
@pytest.mark.parametrize("m", [1, 40])
def test_refused_launch_of_the_weights_planes(m, launch, callers_stream):
    """A refused launch of those that make a weight's planes (which planes there are, their packing) fails the
    call, and nothing of it is kept: the same call then gives the product, here of weights of four planes."""
    rng = np.random.default_rng(m)
    A, B = words(rng, (m, 300), 0), words(rng, (300, 70), 0)
    for call in ("matmul_forward_fused", "matmul_forward_into", "gated_forward"):
        ctx = G.Context(0, stream=0) if callers_stream else G.Context(0)
        a, b, out = ctx.upload(A), ctx.upload(B), ctx.synthetic(m, 70, 0, 3)
        args = (a, b, b, out) if call == "gated_forward" else (a, b, out)
        kw = dict(activation=0) if call == "gated_forward" else {}
        ctx.debug(G.DEBUG_REFUSE_LAUNCH, launch)
        with pytest.raises(G.GkrError) as e:
            getattr(ctx, call)(*args, **kw)
        assert e.value.code == 2
        ctx.debug(G.DEBUG_REFUSE_LAUNCH, 0)
        getattr(ctx, call)(*args, **kw)
        want = product(A, B)
        assert np.array_equal(out.download(), want * want % P if call == "gated_forward" else want), call
        ctx.close()


@pytest.mark.parametrize("callers_stream", [False, True])
@pytest.mark.parametrize("m,k,n,launches", [(1, 64, 96, 1), (40, 64, 96, 2), (300, 64, 96, 2), (200, 13825, 1030, 3)])
def test_every_refused_launch_is_told(m, k, n, launches, callers_stream):
    """Whichever launch of a product, of one kernel to three, is refused, the call or the wait behind it says so,
    and the next call writes the whole output again."""
    ctx = G.Context(0, stream=0) if callers_stream else G.Context(0)
    rng = np.random.default_rng(m)
    A, B = words(rng, (m, k), 0), words(rng, (k, n), 1)
    a, b, want = ctx.upload(A), ctx.upload(B), product(A, B)
    ctx.matmul_forward_fused(a, b, ctx.zeros(m, n))  # the planes are there
    ctx.synchronize()
    for call in ("matmul_forward_fused", "gated_forward"):
        weights, kw, ref = ((b,), {}, want) if call == "matmul_forward_fused" else ((b, b), dict(activation=0), want * want % P)
        for nth in range(1, launches + 1):
            for wait in (ctx.synchronize, lambda: out.download()):
                out = ctx.synthetic(m, n, 0, nth)
                ctx.debug(G.DEBUG_REFUSE_LAUNCH, nth)
                with pytest.raises(G.GkrError) as e:
                    getattr(ctx, call)(a, *weights, out, **kw)
                    wait()
                assert e.value.code == 2, (call, nth)
                ctx.debug(G.DEBUG_REFUSE_LAUNCH, 0)
                ctx.synchronize()  # told once
                out = ctx.synthetic(m, n, 0, nth + 10)
                getattr(ctx, call)(a, *weights, out, **kw)
                assert np.array_equal(out.download(), ref), (call, nth)
    ctx.close()


def test_graph_replayed_after_larger_calls():
    """A graph holds the addresses of the context's buffers: calls of larger sizes, which outgrow them, leave what
    a replay writes and reads in place, so that it neither gives wrong words nor touches others' memory."""
    from test_gpu_attention import attend

    G.lib()
    hip = ctypes.CDLL("libamdhip64.so.7")
    vp, size = ctypes.c_void_p, ctypes.c_size_t
    copy, stream, graph, run = hip.hipMemcpyAsync, vp(), vp(), vp()
    copy.argtypes = [vp, vp, size, ctypes.c_int, vp]
    hip.hipStreamBeginCapture.argtypes, hip.hipStreamEndCapture.argtypes = [vp, ctypes.c_int], [vp, ctypes.POINTER(vp)]
    hip.hipGraphInstantiate.argtypes = [ctypes.POINTER(vp), vp, vp, vp, size]
    hip.hipGraphLaunch.argtypes, hip.hipGraphExecDestroy.argtypes, hip.hipGraphDestroy.argtypes = [vp, vp], [vp], [vp]
    assert hip.hipStreamCreate(ctypes.byref(stream)) == 0
    ctx = G.Context(0, stream=stream.value)
    rng = np.random.default_rng(21)
    m, k, n, kv_len = 200, 5001, 300, 2000  # packed, with K splits that are joined
    W = words(rng, (k, n), 1)
    w, x, out = ctx.upload(W), ctx.zeros(m, k), ctx.zeros(m, n)
    keys, values = words(rng, (kv_len, 64), 0), words(rng, (kv_len, 64), 0)
    cache = ctx.kv_cache(1, 64, n_pages=200, max_seqs=3, max_tokens=9000)
    seq, long = cache.new_sequence(), cache.new_sequence()
    cache.append([seq], [kv_len], ctx.upload(keys), ctx.upload(values))
    q, att = ctx.zeros(1, 128), ctx.zeros(1, 128)

    def calls():
        ctx.matmul_forward_fused(x, w, out)
        ctx.attention_forward(cache, q, [seq], 2, att, score_offset=1 << 19)

    calls()
    ctx.synchronize()
    thread_local = 1
    assert hip.hipStreamBeginCapture(stream, thread_local) == 0
    calls()
    assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(run), graph, None, None, 0) == 0
    others = []
    for turn in range(4):
        if turn:  # larger rows, K and splits than any before, and more of the heads' parts
            M, K = 200 + 300 * turn, 5001 + 4000 * turn
            A, B = words(rng, (M, K), 1), words(rng, (K, n), 1)
            big = ctx.zeros(M, n)
            ctx.matmul_forward_fused(ctx.upload(A), ctx.upload(B), big)
            assert np.array_equal(big.download(), product(A, B))
            more = words(rng, (2900, 64), 0)
            cache.append([long], [2900], ctx.upload(more), ctx.upload(more))
            wide = ctx.zeros(40 * turn, 128)
            ctx.attention_forward(cache, ctx.zeros(40 * turn, 128), [long] * (40 * turn), 2, wide)
            others += [ctx.zeros(1, e) for e in (1 << 16, 1 << 20, 1 << 22, 1 << 24)]  # where freed memory was
        X, Q = words(rng, (m, k), turn % 2), words(rng, (1, 128), 0)
        for dev, h in ((x, X), (q, Q)):
            assert copy(dev.device_ptr, h.ctypes.data, h.nbytes, 1, stream) == 0
        for _ in range(2):
            assert hip.hipGraphLaunch(run, stream) == 0
            assert np.array_equal(out.download(), product(X, W))
            assert np.array_equal(att.download()[0], attend(Q[0], keys, values, 2, 1, 1 << 19, 20)[0])
        assert not any(o.download().any() for o in others)
    assert hip.hipGraphExecDestroy(run) == 0 and hip.hipGraphDestroy(graph) == 0
    cache.free()
    ctx.close()
    assert hip.hipStreamDestroy(stream) == 0


def test_captured_products_of_two_and_three_planes():
    """The forward product by weights of two and three digit planes, which it extends to four in scratch, and a
    fused product beyond the longest inner size, which takes the same path, captured and replayed with other
    products in between that leave other planes there."""
    G.lib()
    hip = ctypes.CDLL("libamdhip64.so.7")
    vp, size = ctypes.c_void_p, ctypes.c_size_t
    copy, stream, graph, run = hip.hipMemcpyAsync, vp(), vp(), vp()
    copy.argtypes = [vp, vp, size, ctypes.c_int, vp]
    hip.hipStreamBeginCapture.argtypes, hip.hipStreamEndCapture.argtypes = [vp, ctypes.c_int], [vp, ctypes.POINTER(vp)]
    hip.hipGraphInstantiate.argtypes = [ctypes.POINTER(vp), vp, vp, vp, size]
    hip.hipGraphLaunch.argtypes, hip.hipGraphExecDestroy.argtypes, hip.hipGraphDestroy.argtypes = [vp, vp], [vp], [vp]
    assert hip.hipStreamCreate(ctypes.byref(stream)) == 0
    ctx = G.Context(0, stream=stream.value)
    rng = np.random.default_rng(31)
    shapes = ((33, 700, 90, 12), (5, 900, 200, 20), (3, 131073, 6, 12))
    weights = [rng.integers(0, 1 << bits, size=(k, n), dtype=np.uint32) for _, k, n, bits in shapes]
    ws = [ctx.upload(w) for w in weights]
    xs, outs = [ctx.zeros(m, k) for m, k, _, _ in shapes], [ctx.zeros(m, n) for m, _, n, _ in shapes]
    X = words(rng, (20, 700), 0)
    full = words(rng, (700, 2500), 0)
    full[:, ::2] = rng.integers(0, 1 << 20, size=(700, 1250))
    other = rng.integers(0, 1 << 22, size=(131073, 40), dtype=np.uint32)
    xo, wo, fo, oo = ctx.upload(words(rng, (3, 131073), 0)), ctx.upload(other), ctx.upload(full), ctx.zeros(3, 40)

    def calls():
        for i, (m, k, n, _) in enumerate(shapes):
            if k > 131071:
                ctx.matmul_forward_fused(xs[i], ws[i], outs[i], activation=RELU)
            else:
                ctx.matmul_forward_into(xs[i], ws[i], outs[i])

    def between():
        ctx.matmul_forward_into(xo, wo, oo)
        out = ctx.zeros(20, 2500)
        ctx.matmul_forward_into(ctx.upload(X), fo, out)
        return out

    between()
    calls()
    ctx.synchronize()
    thread_local = 1
    assert hip.hipStreamBeginCapture(stream, thread_local) == 0
    calls()
    assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(run), graph, None, None, 0) == 0
    for turn in range(5):
        host = [words(rng, (m, k), turn % 2) for m, k, _, _ in shapes]
        for x, h in zip(xs, host):
            assert copy(x.device_ptr, h.ctypes.data, h.nbytes, 1, stream) == 0
        assert hip.hipGraphLaunch(run, stream) == 0
        for i, (_, k, _, _) in enumerate(shapes):
            z = product(host[i], weights[i])
            assert np.array_equal(outs[i].download(), activate(z, RELU, 0) if k > 131071 else z), (turn, i)
        if turn != 3:
            assert np.array_equal(between().download(), product(X, full))
    assert hip.hipGraphExecDestroy(run) == 0 and hip.hipGraphDestroy(graph) == 0
    ctx.close()
    assert hip.hipStreamDestroy(stream) == 0


@pytest.mark.parametrize("m,k,n", [(1, 576, 192), (9, 300, 70), (40, 900, 333), (200, 2605, 5101), (300, 500, 4099),
                                   (3, 131073, 5)])
@pytest.mark.parametrize("wk", [1, 0])
def test_every_call_writes_every_output(gpu_ctx, m, k, n, wk):
    """Calls over outputs that hold other words each time, by weights whose planes are built and whose masks the
    calls before have left set or clear."""
    rng = np.random.default_rng(m)
    B, C2 = words(rng, (k, n), wk), words(rng, (k, n), wk)
    b, c2 = gpu_ctx.upload(B), gpu_ctx.upload(C2)
    for turn, xk in enumerate((1, 0, 0, 1, 1)):
        A = words(rng, (m, k), xk)
        a, outs = gpu_ctx.upload(A), [gpu_ctx.synthetic(m, n, 0, 10 * turn + i) for i in range(6)]
        gpu_ctx.matmul_forward_fused(a, b, outs[0], activation=GELU, pre=outs[1])
        gpu_ctx.gated_forward(a, b, c2, outs[2], gate=outs[3], act=outs[4], up=outs[5])
        z, u = product(A, B), product(A, C2)
        act = activate(z, SILU, 0)
        for i, (got, want) in enumerate(zip(outs, (activate(z, GELU, 0), z, act * u % P, z, act, u))):
            assert np.array_equal(got.download(), want), (turn, i)


@pytest.mark.parametrize("callers_stream", [False, True])
def test_an_allocation_that_fails_is_told_once(callers_stream):
    """More memory than there is fails its own call; the calls behind it are not taken to have failed."""
    ctx = G.Context(0, stream=0) if callers_stream else G.Context(0)
    rng = np.random.default_rng(2)
    A, B = words(rng, (3, 64), 1), words(rng, (64, 50), 1)
    a, b = ctx.upload(A), ctx.upload(B)
    cache = ctx.kv_cache(1, 16, n_pages=2, max_seqs=1, max_tokens=128)
    seq, kv = cache.new_sequence(), ctx.upload(words(rng, (1, 16), 0))
    for call in (lambda: ctx.zeros(1 << 19, 1 << 20), lambda: ctx.synthetic(1 << 19, 1 << 20, 1, 1),
                 lambda: ctx.kv_cache(8, 128, n_pages=1 << 24, max_seqs=1, max_tokens=64)):
        for behind in ("product", "append"):
            with pytest.raises(G.GkrError):
                call()
            if behind == "append":
                cache.append([seq], [1], kv, kv)
            out = ctx.synthetic(3, 50, 0, 1)
            ctx.matmul_forward_fused(a, b, out)
            ctx.synchronize()
            assert np.array_equal(out.download(), product(A, B))
    assert cache.length(seq) == 3
    cache.free()
    ctx.close()
