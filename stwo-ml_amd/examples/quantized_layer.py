"""One decoder layer in 8 bits: its witness on the GPU, whole prompts first and then token by token, and a proof of
the last call's down projection.

    python stwo-ml_amd/examples/quantized_layer.py

Each call of `Layer.forward` takes the rows of new tokens of several sequences.  The projections bring their rows to
8 bits and their results back to 8 bits by scales of the rows and of the weights' columns
(gkr_matmul_forward_quantized); queries and keys are turned by their positions (gkr_rotary_forward); the keys and
values go into an int8 cache.  Prompts of sequences that the cache has nothing of attend within the call's own rows
(gkr_attention_prompt), later tokens over the cache (gkr_attention_forward).  The attention's 8-bit rows are
projected back onto the residual stream (gkr_matmul_forward_scaled); behind the gated block (gkr_gated_forward) the
down projection keeps the 8-bit rows that it made, which its proof reads.  There is no norm here, so that the layer
stays small.
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
    # bits that the results of a projection of `hidden` values, of the attention and of the block are shifted by
    SHIFT_IN, SHIFT_ATTENTION, SHIFT_DOWN = 27, 18, 40

    def __init__(self, ctx, hidden=96, heads=6, kv_heads=2, head_dim=16, inner=160, max_tokens=128, seed=1):
        self.ctx, self.heads, self.kv_heads, self.head_dim = ctx, heads, kv_heads, head_dim
        self.hidden, self.inner = hidden, inner
        rng = np.random.default_rng(seed)
        q, kv = heads * head_dim, kv_heads * head_dim
        shapes = {"q": (hidden, q), "k": (hidden, kv), "v": (hidden, kv), "o": (q, hidden), "g": (hidden, inner),
                  "u": (hidden, inner), "d": (inner, hidden)}
        self.host = {"w" + name: int8_words(rng, shape) for name, shape in shapes.items()}
        for name in "qkvod":  # the columns' scales
            self.host["s" + name] = rng.integers(1 << 9, 1 << 10, size=(1, shapes[name][1]), dtype=np.uint32)
        for name in "qkv":
            self.host["b" + name] = int8_words(rng, (1, shapes[name][1])) % 16
        self.dev = {name: ctx.upload(w) for name, w in self.host.items()}
        self.frequencies = G.rotary_frequencies(head_dim)
        self.rotary = ctx.rotary(self.frequencies, max_tokens)

    def forward(self, x, cache, seqs, counts):
        """The rows of x: counts[i] new tokens of sequence seqs[i].  Returns the layer's output and what the down
        projection read and summed up, before its scales."""
        ctx, w = self.ctx, self.dev
        rows, q, kv = x.rows, self.heads * self.head_dim, self.kv_heads * self.head_dim
        query, k, v, att = ctx.zeros(rows, q), ctx.zeros(rows, kv), ctx.zeros(rows, kv), ctx.zeros(rows, q)
        for out, name in ((query, "q"), (k, "k"), (v, "v")):
            ctx.matmul_forward_quantized(x, w["w" + name], out, col_scales=w["s" + name], shift=self.SHIFT_IN, limit=127,
                                         bias=w["b" + name])
        before = [cache.length(s) for s in seqs]
        ctx.rotary_forward(self.rotary, query, query, counts, self.head_dim, starts=before, k=k, k_out=k, limit=127)
        cache.append(seqs, counts, k, v)
        if any(before):
            row_seqs = [s for s, n in zip(seqs, counts) for _ in range(n)]
            lens = [b + i + 1 for b, n in zip(before, counts) for i in range(n)]  # a token sees itself and those before it
            ctx.attention_forward(cache, query, row_seqs, self.heads, att, lens=lens, score_offset=1 << 19)
        else:
            ctx.attention_prompt(query, k, v, counts, self.heads, self.kv_heads, att, score_offset=1 << 19)
        h, product, out = ctx.zeros(rows, self.hidden), ctx.zeros(rows, self.inner), ctx.zeros(rows, self.hidden)
        ctx.matmul_forward_scaled(att, w["wo"], h, col_scales=w["so"], shift=self.SHIFT_ATTENTION, residual=x)
        ctx.gated_forward(h, w["wg"], w["wu"], product, activation=SILU)
        parts = {"quantized": ctx.zeros(rows, self.inner), "scales": ctx.zeros(rows, 1), "sums": ctx.zeros(rows, self.hidden)}
        ctx.matmul_forward_quantized(product, w["wd"], out, col_scales=w["sd"], shift=self.SHIFT_DOWN, residual=h,
                                     quantized=parts["quantized"], row_scales=parts["scales"], pre=parts["sums"])
        return out, parts

    def prove(self, parts):
        """The down projection of the 8-bit rows, and its replay by the verifier.  Returns the number of field
        elements of the proof."""
        rows = parts["quantized"].rows
        ch = G.PoseidonChannel()
        ch.mix_u64(rows)
        proof = G.Proof()
        point, value = G.prove_walk(self.ctx, ch, [(G.STEP_MATMUL, G.CLAIM_FRESH, parts["quantized"], self.dev["wd"], 0, 0)],
                                    proof)
        proof.set_input_claim(point, value)
        felts = proof.serialize()
        again = G.PoseidonChannel()
        again.mix_u64(rows)
        shapes = [(G.STEP_MATMUL, rows, self.inner, self.hidden, 0, 0, G.CLAIM_FRESH)]
        got = G.verify_walk(felts, shapes, None, None, again, [proof.layer_claim_value(0)])
        assert got[:2] == (point, value) and again.digest() == ch.digest()
        return len(felts)


def main(calls=((5, 3), (1, 1), (1, 2)), seed=2, visit=None):
    """Two sequences: a prompt of calls[0] tokens each, then a few at a time; visit(x, out, parts) sees each call."""
    ctx = G.Context(0)
    layer = Layer(ctx)
    cache = ctx.kv_cache(layer.kv_heads, layer.head_dim, n_pages=4, max_seqs=2, max_tokens=128, int8=True)
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
