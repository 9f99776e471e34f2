"""Products with scales, rotary positions and attention over prompts as callers use them: on a stream of the
caller's, captured into a graph that is replayed between other calls, over outputs that hold other words, from
several contexts and threads, and with launches that are refused."""
import ctypes
import threading

import numpy as np
import pytest

import gkr_mi355x as G
from test_gpu_prompt import attend
from test_gpu_rotary import table, turn
from test_gpu_scaled import centered, check, quantize, rescale
from test_gpu_witness import GELU, check_fused, product, words

pytestmark = pytest.mark.gpu
P = G.P
HEADS, KV, DIM, OFFSET = 4, 2, 32, 1 << 19


class Calls:
    """One of each operator over inputs of `kind` (int8-range or any words), with what it has to give."""

    def __init__(self, ctx, m, counts, seed, n=90, k=500):
        self.ctx, self.m, self.counts, self.n, self.k = ctx, m, counts, n, k
        rng = self.rng = np.random.default_rng(seed)
        self.W, self.S = words(rng, (k, n), 1), rng.integers(1 << 14, 1 << 15, size=n)
        self.w, self.s = ctx.upload(self.W), ctx.upload(self.S.reshape(1, n).astype(np.uint32))
        tokens = sum(counts)
        self.freqs = G.rotary_frequencies(DIM)
        self.rotary = ctx.rotary(self.freqs, 1000)
        self.inputs = {"a": ctx.zeros(m, k), "q": ctx.zeros(tokens, HEADS * DIM), "k": ctx.zeros(tokens, KV * DIM),
                       "v": ctx.zeros(tokens, KV * DIM)}
        shapes = {"scaled": (m, n), "quantized": (m, n), "rows": (m, k), "scales": (m, 1), "pre": (m, n),
                  "q_turned": (tokens, HEADS * DIM), "k_turned": (tokens, KV * DIM), "attended": (tokens, HEADS * DIM)}
        self.outputs = {name: ctx.synthetic(*shape, 0, 40 + i) for i, (name, shape) in enumerate(shapes.items())}

    def __call__(self):
        i, o, ctx = self.inputs, self.outputs, self.ctx
        ctx.matmul_forward_scaled(i["a"], self.w, o["scaled"], col_scales=self.s, shift=20)
        ctx.matmul_forward_quantized(i["a"], self.w, o["quantized"], col_scales=self.s, shift=40, limit=1 << 20,
                                     quantized=o["rows"], row_scales=o["scales"], pre=o["pre"])
        ctx.rotary_forward(self.rotary, i["q"], o["q_turned"], self.counts, DIM, starts=[7] * len(self.counts), k=i["k"],
                           k_out=o["k_turned"], limit=127)
        ctx.attention_prompt(o["q_turned"], o["k_turned"], i["v"], self.counts, HEADS, KV, o["attended"],
                             score_offset=OFFSET)

    def fresh(self, kind):
        """New words for the inputs: name -> array."""
        return {name: words(self.rng, (t.rows, t.cols), kind) for name, t in self.inputs.items()}

    def matches(self, x):
        want = {"scaled": rescale(product(x["a"], self.W), np.ones(self.m, np.int64), self.S, 20, 0)}
        rows, scales = quantize(x["a"], 127)
        want["rows"], want["scales"] = rows, scales[:, None]
        want["pre"] = product(rows.astype(np.uint32), self.W)
        want["quantized"] = rescale(want["pre"], scales, self.S, 40, 1 << 20)
        at = np.concatenate([7 + np.arange(n) for n in self.counts])
        c, s = table(self.freqs, at, 1 << 15)
        want["q_turned"], want["k_turned"] = (turn(x[t], c, s, DIM, 15, False, 127) for t in "qk")
        out, row = [], 0
        for n in filter(None, self.counts):
            part = [t[row : row + n] for t in (want["q_turned"], want["k_turned"], x["v"])]
            out.append(attend(*part, HEADS, KV, OFFSET, 20, n)[0])
            row += n
        want["attended"] = np.concatenate(out)
        for name, t in want.items():
            assert np.array_equal(self.outputs[name].download(), t), name


def upload(ctx, calls, x, copy, stream):
    for name, host in x.items():
        assert copy(calls.inputs[name].device_ptr, host.ctypes.data, host.nbytes, 1, stream) == 0


def runtime():
    G.lib()
    hip = ctypes.CDLL("libamdhip64.so.7")  # the runtime the library has loaded
    vp, size = ctypes.c_void_p, ctypes.c_size_t
    hip.hipMemcpyAsync.argtypes = [vp, vp, size, ctypes.c_int, vp]
    hip.hipStreamBeginCapture.argtypes, hip.hipStreamEndCapture.argtypes = [vp, ctypes.c_int], [vp, ctypes.POINTER(vp)]
    hip.hipGraphInstantiate.argtypes = [ctypes.POINTER(vp), vp, vp, vp, size]
    hip.hipGraphLaunch.argtypes, hip.hipGraphExecDestroy.argtypes, hip.hipGraphDestroy.argtypes = [vp, vp], [vp], [vp]
    return hip


def test_on_the_callers_stream():
    hip, stream = runtime(), ctypes.c_void_p()
    assert hip.hipStreamCreate(ctypes.byref(stream)) == 0
    for s in (stream, ctypes.c_void_p()):
        ctx = G.Context(0, stream=s.value or 0)
        for m, counts in ((1, [1]), (40, [33, 0, 5])):
            calls = Calls(ctx, m, counts, m)
            for turn_ in range(4):
                x = calls.fresh(turn_ % 2)
                upload(ctx, calls, x, hip.hipMemcpyAsync, s)
                calls()
                calls.matches(x)
        ctx.close()
    assert hip.hipStreamDestroy(stream) == 0


@pytest.mark.parametrize("m,counts", [(1, [1]), (9, [9]), (200, [150, 1, 0, 70])])
def test_captured_into_a_graph(m, counts):
    """Captured once and replayed over changed inputs, int8-range and general in turn, with calls of the context's
    own between, of the same sizes and of larger ones, whose buffers outgrow the graph's."""
    hip, stream = runtime(), ctypes.c_void_p()
    graph, run = ctypes.c_void_p(), ctypes.c_void_p()
    assert hip.hipStreamCreate(ctypes.byref(stream)) == 0
    ctx = G.Context(0, stream=stream.value)
    calls, same = Calls(ctx, m, counts, 5), Calls(ctx, m, counts, 6)
    upload(ctx, calls, calls.fresh(0), hip.hipMemcpyAsync, stream)
    calls()  # planes, tables and buffers are there from here on
    ctx.synchronize()
    thread_local = 1
    assert hip.hipStreamBeginCapture(stream, thread_local) == 0
    calls()
    assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(run), graph, None, None, 0) == 0
    others = []
    for turn_ in range(5):
        x = calls.fresh(turn_ % 2)
        upload(ctx, calls, x, hip.hipMemcpyAsync, stream)
        for _ in range(2):
            assert hip.hipGraphLaunch(run, stream) == 0
            calls.matches(x)
        between = same if turn_ < 2 else Calls(ctx, m + 150 * turn_, [200 * turn_, 40], turn_, k=500 + 900 * turn_)
        y = between.fresh(1 - turn_ % 2)
        upload(ctx, between, y, hip.hipMemcpyAsync, stream)
        between()
        between.matches(y)
        others += [ctx.zeros(1, e) for e in (1 << 16, 1 << 20, 1 << 22)]  # where freed memory was
        assert not any(o.download().any() for o in others)
    assert hip.hipGraphExecDestroy(run) == 0 and hip.hipGraphDestroy(graph) == 0
    ctx.close()
    assert hip.hipStreamDestroy(stream) == 0


def test_two_contexts_from_two_threads():
    failed = []

    def work(seed):
        try:
            ctx = G.Context(0)
            calls = [Calls(ctx, m, counts, seed + m) for m, counts in ((1, [1]), (70, [64, 6]), (300, [257]))]
            for turn_ in range(4):
                for c in calls:
                    x = c.fresh((turn_ + seed) % 2)
                    for name, host in x.items():
                        c.inputs[name] = ctx.upload(host)
                    c()
                    c.matches(x)
            ctx.close()
        except BaseException as e:  # told by the test
            failed.append(e)

    threads = [threading.Thread(target=work, args=(s,)) for s in (1, 2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


@pytest.mark.parametrize("callers_stream", [False, True])
@pytest.mark.parametrize("m,counts,k", [(1, [1], 64), (4, [3], 5000), (40, [70], 64), (300, [40, 33], 13825)])
def test_every_refused_launch_is_told(m, counts, k, callers_stream):
    """Whichever launch of the four operators is refused, a call or the wait behind them says so, and the next
    calls write every output again."""
    ctx = G.Context(0, stream=0) if callers_stream else G.Context(0)
    calls = Calls(ctx, m, counts, m, n=1030, k=k)
    x = calls.fresh(0)
    for name, host in x.items():
        calls.inputs[name] = ctx.upload(host)
    calls()
    ctx.synchronize()  # planes and buffers are there

    refused = 0
    for nth in range(1, 40):
        for name, t in calls.outputs.items():
            calls.outputs[name] = ctx.synthetic(t.rows, t.cols, 0, nth)
        ctx.synchronize()
        ctx.debug(G.DEBUG_REFUSE_LAUNCH, nth)
        try:
            calls()
            ctx.synchronize()
        except G.GkrError as e:
            assert e.code == 2
            refused += 1
        else:
            ctx.debug(G.DEBUG_REFUSE_LAUNCH, 0)
            break
        ctx.debug(G.DEBUG_REFUSE_LAUNCH, 0)
        ctx.synchronize()  # told once
        calls()
        calls.matches(x)
    assert 5 <= refused < 39  # a launch of each, the prompt's two
    calls.matches(x)
    ctx.close()


# the longest rows that a few rows' product quantizes by itself, and one more
@pytest.mark.parametrize("m,k", [(1, 16384), (1, 16385), (2, 8192), (2, 8193), (4, 4096), (3, 4097), (8, 2048), (16, 1024),
                                 (7, 1985), (1, 65), (1, 70001), (17, 16385), (40, 20000)])
@pytest.mark.parametrize("n", [70, 8300])
def test_longest_rows_quantized_by_the_product(gpu_ctx, m, k, n):
    if n * k > 1 << 28:
        n = 333
    check(gpu_ctx, m, k, n, 0, 1, 50, 127, levels=127)
    check(gpu_ctx, m, k, n, 1, 1, 40, 0, levels=3, residual=False, bias=False)


@pytest.mark.parametrize("levels", [1, 2, 127])
@pytest.mark.parametrize("m", [1, 40])
def test_quantized_halves(gpu_ctx, m, levels):
    """Every magnitude about the halves between two levels, for largest magnitudes of every size."""
    rng = np.random.default_rng(m)
    for a in (0, 1, 2, 3, 126, 127, 128, 255, 65537, (1 << 24) - 1, 1 << 29, (1 << 30) - 1):
        half = [(2 * i + 1) * a // (2 * levels) + d for i in range(levels) for d in (-1, 0, 1)]
        c = np.array([a] + [min(a, max(0, h)) for h in half] + [0], dtype=np.int64)
        c = c * rng.choice([-1, 1], size=(m, len(c)))
        x = (c % P).astype(np.uint32)
        k, out = x.shape[1], gpu_ctx.zeros(m, 2)
        q, s = gpu_ctx.synthetic(m, k, 0, 1), gpu_ctx.synthetic(m, 1, 0, 2)
        gpu_ctx.matmul_forward_quantized(gpu_ctx.upload(x), gpu_ctx.upload(words(rng, (k, 2), 1)), out, levels=levels,
                                         quantized=q, row_scales=s)
        want, scale = quantize(x, levels)
        assert np.array_equal(q.download(), want), a
        assert np.array_equal(s.download()[:, 0], scale), a


# rows between the sizes of the streamed kernels and those that fill the chip with blocks; ragged in both
@pytest.mark.parametrize("m,k,n", [(300, 700, 5001), (257, 1001, 8111), (700, 65, 4100), (1000, 333, 1551), (385, 2100, 5000)])
def test_some_hundred_rows(gpu_ctx, m, k, n):
    check(gpu_ctx, m, k, n, 1, 1, 40, 127)
    check(gpu_ctx, m, k, n, 0, 1, 50, 0, residual=False, pre=False)
    check(gpu_ctx, m, k, n, 0, 1, 50, 1 << 20, levels=127)
    x = np.zeros((m, k), np.uint32)
    x[m // 2, k - 1] = 12345  # one word above a byte
    check(gpu_ctx, m, k, n, 1, 1, 0, 0, x=x)
    check_fused(gpu_ctx, m, k, n, 1, 1, act=GELU, log=0)
    check_fused(gpu_ctx, m, k, n, 0, 1)


def tail(ctx, m, rows):
    """The last rows of a matrix, as a matrix over the same memory."""
    return ctx.wrap_device(m.device_ptr + 4 * (m.rows - rows) * m.cols, rows, m.cols)


@pytest.mark.parametrize("kind", [1, 0])
def test_prompts_and_turns_past_4_gib(gpu_ctx, kind):
    """Packed sequences whose queries and outputs pass 2^32 bytes: the last ones equal a call with them alone."""
    each, n, heads, kv, d = 1000, 215, 40, 8, 128
    q, k, v = (gpu_ctx.synthetic(each * n, h * d, kind, 3 + i) for i, h in enumerate((heads, kv, kv)))
    out, sums = gpu_ctx.synthetic(each * n, heads * d, 0, 1), gpu_ctx.synthetic(each * n, heads, 0, 2)
    counts = [each] * (n - 3) + [each + 7, each - 7, each]
    gpu_ctx.attention_prompt(q, k, v, counts, heads, kv, out, score_offset=OFFSET, sums=sums)
    rows = counts[-1] + counts[-2]
    alone, alone_sums = gpu_ctx.zeros(rows, heads * d), gpu_ctx.zeros(rows, heads)
    gpu_ctx.attention_prompt(tail(gpu_ctx, q, rows), tail(gpu_ctx, k, rows), tail(gpu_ctx, v, rows), counts[-2:], heads, kv,
                             alone, score_offset=OFFSET, sums=alone_sums)
    assert np.array_equal(tail(gpu_ctx, out, rows).download(), alone.download())
    assert np.array_equal(tail(gpu_ctx, sums, rows).download(), alone_sums.download())
    rotary = gpu_ctx.rotary(G.rotary_frequencies(d), 2 * each)
    starts = [i % 900 for i in range(n)]
    gpu_ctx.rotary_forward(rotary, q, out, counts, d, starts=starts, k=k, k_out=k, limit=127)
    gpu_ctx.rotary_forward(rotary, tail(gpu_ctx, q, rows), alone, counts[-2:], d, starts=starts[-2:], limit=127)
    assert np.array_equal(tail(gpu_ctx, out, rows).download(), alone.download())
    rotary.free()


def test_scores_past_4_gib(gpu_ctx):
    heads, n, d = 64, 4200, 16
    rng = np.random.default_rng(5)
    Q, K = words(rng, (n, heads * d), 1), words(rng, (n, d), 1)
    q, k = gpu_ctx.upload(Q), gpu_ctx.upload(K)
    out, scores = gpu_ctx.zeros(n, heads * d), gpu_ctx.zeros(n * heads, n + 1)
    gpu_ctx.attention_prompt(q, k, k, [n], heads, 1, out, score_offset=OFFSET, scores=scores)
    want = (OFFSET + centered(Q[-1]).reshape(heads, d) @ centered(K).T) % P
    got = tail(gpu_ctx, scores, 65).download()  # the last token's, and one of the token before
    assert np.array_equal(got[1:, :n], want) and not got[:, n].any() and got[0, n - 1] == 0 and got[0, n - 2] != 0


def test_scaled_results_past_4_gib(gpu_ctx):
    m, k, n = 70001, 64, 16400
    rows = 300
    a, b, s = gpu_ctx.synthetic(m, k, 1, 1), gpu_ctx.synthetic(k, n, 1, 2), gpu_ctx.synthetic(1, n, 0, 3)
    out, alone = gpu_ctx.synthetic(m, n, 0, 4), gpu_ctx.zeros(rows, n)
    gpu_ctx.matmul_forward_scaled(a, b, out, col_scales=s, shift=38, limit=127)
    gpu_ctx.matmul_forward_scaled(tail(gpu_ctx, a, rows), b, alone, col_scales=s, shift=38, limit=127)
    assert np.array_equal(tail(gpu_ctx, out, rows).download(), alone.download())
    gpu_ctx.matmul_forward_quantized(a, b, out, col_scales=s, shift=45, limit=127)
    gpu_ctx.matmul_forward_quantized(tail(gpu_ctx, a, rows), b, alone, col_scales=s, shift=45, limit=127)
    assert np.array_equal(tail(gpu_ctx, out, rows).download(), alone.download())


@pytest.mark.parametrize("general", [False, True])
def test_longest_prompt(gpu_ctx, general):
    """The most tokens of one sequence, with weights and values that fill the sums: rows of it against whole
    numbers."""
    n, d = 131071, 16
    rng = np.random.default_rng(9)
    place = 7 if general else 10  # the largest weights of a plane
    Q, K = np.zeros((n, d), np.uint32), words(rng, (n, d), 0 if general else 1)
    V = np.full((n, d), (P - (128 + (128 << 8) + (128 << 16) + (62 << 24))) if general else P - 128, np.uint32)
    Q[n // 2 :] = words(rng, (n - n // 2, d), 0 if general else 1)  # the earlier rows have one weight
    Q[-1] = 0
    V[::7] = words(rng, V[::7].shape, 0 if general else 1)
    V[1::7] = V[2]
    out, weighted, sums = gpu_ctx.zeros(n, d), gpu_ctx.zeros(n, d), gpu_ctx.zeros(n, 1)
    gpu_ctx.attention_prompt(gpu_ctx.upload(Q), gpu_ctx.upload(K), gpu_ctx.upload(V), [n], 1, 1, out,
                             score_offset=place << 16, weighted=weighted, sums=sums)
    out, weighted, sums = out.download(), weighted.download(), sums.download()
    ck, cv = centered(K), centered(V)
    for t in (0, 1, 63, 64, 4097, n // 2 - 1, n // 2, n - 65, n - 2, n - 1):
        x = ((place << 16) + (ck[: t + 1] * centered(Q[t]) % P).sum(axis=1)) % P
        w = np.int64(1) << np.minimum((x % (1 << 20)) >> 16, 10)
        z, total = int(w.sum()), [int(c) for c in w @ cv[: t + 1]]
        assert sums[t, 0] == (z << 16) % P, t
        assert [int(c) for c in weighted[t]] == [(c << 16) % P for c in total], t
        assert [int(c) for c in out[t]] == [(1 if c > 0 else -1) * ((2 * abs(c) + z) // (2 * z)) % P for c in total], t
