"""The decoder layer example: its witness against whole-number arithmetic, call by call, and its proof."""
import os
import sys

import gkr_mi355x as G
import numpy as np
import pytest

from test_gpu_attention import attend
from test_gpu_witness import activate, product

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "stwo-ml_amd", "examples"))
import decoder_layer  # noqa: E402

pytestmark = pytest.mark.gpu
P = G.P


def test_prompt_and_tokens():
    seen = [([], []), ([], [])]  # keys and values of each sequence
    calls = []

    def visit(layer, x, counts, out, parts):
        w = layer.host
        q, k, v = ((product(x, w["w" + n]) + w["b" + n]) % P for n in "qkv")
        att, row = np.zeros_like(q), 0
        for (ks, vs), n in zip(seen, counts):
            for i in range(n):
                ks.append(k[row])
                vs.append(v[row])
                att[row] = attend(q[row], np.array(ks), np.array(vs), layer.heads, layer.kv_heads, 1 << 19, 20)[0]
                row += 1
        h = (product(att, w["wo"]) + x) % P
        gate, up = product(h, w["wg"]), product(h, w["wu"])
        act = activate(gate, decoder_layer.SILU, 0)
        assert np.array_equal(parts["gate"].download(), gate) and np.array_equal(parts["up"].download(), up)
        assert np.array_equal(parts["act"].download(), act)
        hidden = act * up % P
        assert np.array_equal(parts["product"].download(), hidden)
        assert np.array_equal(out, (product(hidden, w["wd"]) + h) % P)
        calls.append(counts)

    decoder_layer.main(visit=visit)
    assert len(calls) == 3
