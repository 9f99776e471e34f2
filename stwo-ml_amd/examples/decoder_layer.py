"""One decoder layer: its witness on the GPU, from a prompt and then token by token, and a proof of what the
last call computed in the feed-forward block.

    python stwo-ml_amd/examples/decoder_layer.py

Each call of `Layer.forward` takes the rows of new tokens of several sequences: projections with their biases
(gkr_matmul_forward_fused), the cache (gkr_kv_cache_append), attention over it (gkr_attention_forward), the
output projection added to the residual stream, the gated block (gkr_gated_forward) and the down projection
added again.  All values are words of the field; there is no norm here, so that the layer stays small.
"""
import os
import sys

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import gkr_mi355x as G  # noqa: E402

P = G.P
SILU = 5


def int8_words(rng, shape):
    v = rng.integers(-127, 128, size=shape)
    return np.where(v < 0, v + P, v).astype(np.uint32)


class Layer:
    def __init__(self, ctx, hidden=96, heads=6, kv_heads=2, head_dim=16, inner=160, seed=1):
        self.ctx, self.heads, self.kv_heads, self.head_dim = ctx, heads, kv_heads, head_dim
        self.hidden, self.inner = hidden, inner
        rng = np.random.default_rng(seed)
        q, kv = heads * head_dim, kv_heads * head_dim
        self.host = {"wq": int8_words(rng, (hidden, q)), "wk": int8_words(rng, (hidden, kv)),
                     "wv": int8_words(rng, (hidden, kv)), "wo": int8_words(rng, (q, hidden)),
                     "wg": int8_words(rng, (hidden, inner)), "wu": int8_words(rng, (hidden, inner)),
                     "wd": int8_words(rng, (inner, hidden)), "bq": int8_words(rng, (1, q)),
                     "bk": int8_words(rng, (1, kv)), "bv": int8_words(rng, (1, kv))}
        self.dev = {name: ctx.upload(w) for name, w in self.host.items()}

    def forward(self, x, cache, seqs, counts):
        """The rows of x: counts[i] new tokens of sequence seqs[i].  Returns the layer's output and the parts of
        the gated block that its proof reads."""
        ctx, w = self.ctx, self.dev
        rows, q, kv = x.rows, self.heads * self.head_dim, self.kv_heads * self.head_dim
        query, k, v, att = ctx.zeros(rows, q), ctx.zeros(rows, kv), ctx.zeros(rows, kv), ctx.zeros(rows, q)
        for out, wn, bn in ((query, "wq", "bq"), (k, "wk", "bk"), (v, "wv", "bv")):
            ctx.matmul_forward_fused(x, w[wn], out, bias=w[bn])
        before = [cache.length(s) for s in seqs]
        cache.append(seqs, counts, k, v)
        row_seqs = [s for s, n in zip(seqs, counts) for _ in range(n)]
        lens = [b + i + 1 for b, n in zip(before, counts) for i in range(n)]  # a token sees itself and those before it
        ctx.attention_forward(cache, query, row_seqs, self.heads, att, lens=lens, score_offset=1 << 19)
        h = ctx.zeros(rows, self.hidden)
        ctx.matmul_forward_fused(att, w["wo"], h, residual=x)
        parts = {name: ctx.zeros(rows, self.inner) for name in ("gate", "act", "up", "product")}
        ctx.gated_forward(h, w["wg"], w["wu"], parts["product"], activation=SILU, gate=parts["gate"], act=parts["act"],
                          up=parts["up"])
        out = ctx.zeros(rows, self.hidden)
        ctx.matmul_forward_fused(parts["product"], w["wd"], out, residual=h)
        return out, parts

    def prove(self, parts):
        """The down projection, the gate's product and the activation behind it in one walk, and its replay by
        the verifier.  Returns the number of field elements of the proof."""
        rows = parts["gate"].rows
        ch = G.PoseidonChannel()
        ch.mix_u64(rows)
        proof = G.Proof()
        steps = [(G.STEP_MATMUL, G.CLAIM_FRESH, parts["product"], self.dev["wd"], 0, 0),
                 (G.STEP_MUL, G.CLAIM_CHAINED, parts["act"], parts["up"], 0, 0),
                 (G.STEP_ACTIVATION, G.CLAIM_CHAINED, parts["gate"], None, SILU, 0)]
        point, value = G.prove_walk(self.ctx, ch, steps, proof)
        proof.set_input_claim(point, value)
        felts = proof.serialize()
        shapes = [(G.STEP_MATMUL, rows, self.inner, self.hidden, 0, 0, G.CLAIM_FRESH),
                  (G.STEP_MUL, rows, self.inner, 0, 0, 0, G.CLAIM_CHAINED),
                  (G.STEP_ACTIVATION, rows, self.inner, 0, SILU, 0, G.CLAIM_CHAINED)]
        again = G.PoseidonChannel()
        again.mix_u64(rows)
        got = G.verify_walk(felts, shapes, None, None, again, [proof.layer_claim_value(0)])
        assert got[:2] == (point, value) and again.digest() == ch.digest()
        return len(felts)


def main(calls=((5, 3), (1, 1), (1, 1)), seed=2, visit=None):
    """Two sequences: a prompt of calls[0] tokens each, then token by token; visit(x, out, parts) sees each call."""
    ctx = G.Context(0)
    layer = Layer(ctx)
    cache = ctx.kv_cache(layer.kv_heads, layer.head_dim, n_pages=4, max_seqs=2, max_tokens=128)
    seqs = [cache.new_sequence(), cache.new_sequence()]
    rng = np.random.default_rng(seed)
    for counts in calls:
        x = int8_words(rng, (sum(counts), layer.hidden))
        out, parts = layer.forward(ctx.upload(x), cache, seqs, counts)
        if visit:
            visit(layer, x, counts, out.download(), parts)
    felts = layer.prove(parts)
    print("tokens in the cache:", [cache.length(s) for s in seqs], "proof:", felts, "felts")
    ctx.close()


if __name__ == "__main__":
    main()
