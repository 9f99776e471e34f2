"""What a call of the operators leaves behind for the next: copies derived from a matrix that another handle of the
same call writes, and the packing's word about digits above the lowest."""
import ctypes

import numpy as np
import pytest

import gkr_mi355x as G
from test_gpu_operator_calls import OFFSET, runtime
from test_gpu_prompt import attend
from test_gpu_scaled import quantize, rescale
from test_gpu_witness import product, words

pytestmark = pytest.mark.gpu
P = G.P


@pytest.mark.parametrize("m", [9, 70])
@pytest.mark.parametrize("form", ["fused", "scaled", "quantized"])
def test_residual_that_is_the_output_by_another_handle(gpu_ctx, form, m):
    """The residual's handle has been a product's weights: once the call has written its memory, its digit planes are
    made again, as are the output's own."""
    rng = np.random.default_rng(m)
    A, B, R, X = words(rng, (m, 100), 1), words(rng, (100, m), 1), words(rng, (m, m), 1), words(rng, (3, m), 1)
    a, b, x, memory = (gpu_ctx.upload(t) for t in (A, B, X, R))
    residual, out = (gpu_ctx.wrap_device(memory.device_ptr, m, m) for _ in range(2))
    y = gpu_ctx.zeros(3, m)
    for handle in (residual, out):
        gpu_ctx.matmul_forward_fused(x, handle, y)
        assert np.array_equal(y.download(), product(X, R))
    if form == "fused":
        gpu_ctx.matmul_forward_fused(a, b, out, residual=residual)
        want = product(A, B)
    elif form == "scaled":
        gpu_ctx.matmul_forward_scaled(a, b, out, residual=residual)
        want = rescale(product(A, B), [1] * m, [1] * m, 0, 0)
    else:
        gpu_ctx.matmul_forward_quantized(a, b, out, shift=7, residual=residual)
        q, r = quantize(A, 127)
        want = rescale(product(q.astype(np.uint32), B), r, [1] * m, 7, 0)
    want = ((want.astype(np.int64) + R) % P).astype(np.uint32)
    for handle in (out, residual):
        assert np.array_equal(handle.download(), want)
        gpu_ctx.matmul_forward_fused(x, handle, y)
        assert np.array_equal(y.download(), product(X, want))


def test_captured_prompt_after_general_words():
    """A graph of one prompt: a replay over general words leaves nothing that sends the next replays over int8-range
    words through the kernel of general words, which takes several times as long."""
    hip, stream = runtime(), ctypes.c_void_p()
    graph, run = ctypes.c_void_p(), ctypes.c_void_p()
    hip.hipEventElapsedTime.argtypes = [ctypes.POINTER(ctypes.c_float), ctypes.c_void_p, ctypes.c_void_p]
    hip.hipEventRecord.argtypes = [ctypes.c_void_p, ctypes.c_void_p]
    hip.hipEventSynchronize.argtypes = hip.hipEventDestroy.argtypes = [ctypes.c_void_p]
    assert hip.hipStreamCreate(ctypes.byref(stream)) == 0
    events = [ctypes.c_void_p(), ctypes.c_void_p()]
    for e in events:
        assert hip.hipEventCreate(ctypes.byref(e)) == 0
    ctx = G.Context(0, stream=stream.value)
    heads, d, counts = 16, 128, [1500]
    rows = sum(counts)
    rng = np.random.default_rng(4)
    kinds = {kind: [words(rng, (rows, heads * d), kind) for _ in range(3)] for kind in (1, 0)}
    q, k, v, out = (ctx.zeros(rows, heads * d) for _ in range(4))

    def put(kind):
        for m, host in zip((q, k, v), kinds[kind]):
            assert hip.hipMemcpyAsync(m.device_ptr, host.ctypes.data, host.nbytes, 1, stream) == 0
        ctx.synchronize()

    def replay():
        times = []
        for _ in range(5):
            assert hip.hipEventRecord(events[0], stream) == 0
            assert hip.hipGraphLaunch(run, stream) == 0
            assert hip.hipEventRecord(events[1], stream) == 0 and hip.hipEventSynchronize(events[1]) == 0
            ms = ctypes.c_float()
            assert hip.hipEventElapsedTime(ctypes.byref(ms), *events) == 0
            times.append(ms.value)
        return min(times)

    def matches(kind):
        columns = [slice(h * d, (h + 1) * d) for h in (0, heads - 1)]
        got = out.download()
        for c in columns:
            assert np.array_equal(got[:, c], attend(*(t[:, c] for t in kinds[kind]), 1, 1, OFFSET, 20, rows)[0])

    put(1)
    call = lambda: ctx.attention_prompt(q, k, v, counts, heads, heads, out, score_offset=OFFSET)  # noqa: E731
    call()
    ctx.synchronize()
    assert hip.hipStreamBeginCapture(stream, 1) == 0
    call()
    assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(run), graph, None, None, 0) == 0
    fresh = replay()
    matches(1)
    put(0)
    general = replay()
    matches(0)
    put(1)
    after = replay()
    matches(1)
    assert general > 2 * fresh  # else nothing is told by the times
    assert after < 1.5 * fresh, (fresh, general, after)
    assert hip.hipGraphExecDestroy(run) == 0 and hip.hipGraphDestroy(graph) == 0
    ctx.close()
    for e in events:
        assert hip.hipEventDestroy(e) == 0
    assert hip.hipStreamDestroy(stream) == 0
