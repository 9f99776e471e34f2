"""What a call of the operators leaves behind for the next: copies derived from a matrix that another handle of the
same call writes."""
import numpy as np
import pytest

import gkr_mi355x as G
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
