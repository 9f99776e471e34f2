"""The 8-bit decoder layer example: its witness against whole-number arithmetic, call by call (prompts, single
tokens, a few tokens at a time), and its proof."""
import os
import sys

import gkr_mi355x as G
import numpy as np
import pytest

from test_gpu_attention import attend
from test_gpu_rotary import table, turn
from test_gpu_scaled import quantize, rescale
from test_gpu_witness import activate, product

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "stwo-ml_amd", "examples"))
import quantized_layer  # noqa: E402

pytestmark = pytest.mark.gpu
P = G.P


def quantized(x, w, s, shift, limit=0, bias=None, residual=None):
    q, a = quantize(x, 127)
    z = product(q.astype(np.uint32), w)
    return rescale(z, a, s[0].astype(np.int64), shift, limit, None if bias is None else bias[0], residual), q, a, z


@pytest.mark.parametrize("calls", [((5, 3), (1, 1), (1, 2)), ((40, 23), (1, 1)), ((0, 70), (1, 1), (9, 2))])
def test_prompts_and_tokens(calls):
    seen, done = [([], []), ([], [])], []  # keys and values of each sequence

    def visit(layer, x, counts, out, parts):
        w = layer.host
        q, k, v = (quantized(x, w["w" + n], w["s" + n], layer.SHIFT_IN, 127, w["b" + n])[0] for n in "qkv")
        at = np.concatenate([len(ks) + np.arange(n) for (ks, _), n in zip(seen, counts)])
        c, s = table(layer.frequencies, at, 1 << 15)
        q, k = (turn(t, c, s, layer.head_dim, 15, False, 127) for t in (q, k))
        att, row = np.zeros_like(q), 0
        for (ks, vs), n in zip(seen, counts):
            for i in range(n):
                ks.append(k[row])
                vs.append(v[row])
                att[row] = attend(q[row], np.array(ks), np.array(vs), layer.heads, layer.kv_heads, 1 << 19, 20)[0]
                row += 1
        z = product(att.astype(np.uint32), w["wo"])
        h = rescale(z, np.ones(len(x), np.int64), w["so"][0].astype(np.int64), layer.SHIFT_ATTENTION, 0, None, x)
        h = h.astype(np.uint32)
        hidden = activate(product(h, w["wg"]), quantized_layer.SILU, 0) * product(h, w["wu"]) % P
        want, rows, scales, sums = quantized(hidden, w["wd"], w["sd"], layer.SHIFT_DOWN, residual=h)
        assert np.array_equal(parts["quantized"].download(), rows)
        assert np.array_equal(parts["scales"].download()[:, 0], scales)
        assert np.array_equal(parts["sums"].download(), sums)
        assert np.array_equal(out, want)
        done.append(counts)

    quantized_layer.main(calls=calls, visit=visit)
    assert len(done) == len(calls)
