"""The witness operators between a transformer layer's stored values: products whose operands and results are
8-bit integers with scales, rotary positions, and attention over whole prompts, as they are timed and compared.

Values are canonical words of the prime field with P = 2^31 - 1 elements; a word above P/2 stands for a
negative number, and c(x) is the number that a word x stands for ("centered").  round() is to whole numbers,
halves away from zero.  Four operators:

  scaled     t = round(c(X W) r_i s_j / 2^shift) + c(bias_j) for whole scales r of the rows and s of the
             columns, Y = t cut off at +-limit, + residual (mod P), and Z = X W;
  quantized  the same of rows that are brought to 8 bits first: a_i the largest |c(x)| of row i, q =
             round(c(x) levels / a_i), Z = q W and r_i = a_i; with q and a where asked for;
  rotary     pairs of a head's values turned by position times frequency, y0 = round((x0 C - x1 S) / 2^shift),
             y1 = round((x1 C + x0 S) / 2^shift) with whole C and S; frequencies are whole numbers of 2^-64
             turns a position, so that angles of far positions lose nothing;
  prompt     causal attention of packed sequences: a token sees itself and those before it in its sequence,
             with the weights of the softmax lookup table and the mean of the values, as the attention over
             the cache (perf/operators.py) has them.

With `own` false, run() computes them with elementary torch operations, exactly: matrix products in float64
over parts small enough that every sum stays below 2^53.  With `own` true it makes the framework's calls.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

P = (1 << 31) - 1
HALF = (1 << 30) - 1
SCORE_OFFSET = 1 << 19  # the middle of a 2^20 table: negative scores stay below it


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # the key projection of one decoded token into an int8 cache, SmolLM2-135M: all latency
        {"name": "scaled_token", "op": "scaled", "m": 1, "k": 576, "n": 192, "w": "int8", "limit": 127, "bias": True,
         "residual": False, "pre": False},
        # the query projection of a 512-token prompt, Qwen2.5-14B
        {"name": "scaled_prompt", "op": "scaled", "m": 512, "k": 5120, "n": 5120, "w": "int8", "limit": 127,
         "bias": True, "residual": False, "pre": False},
        # the down projection of one decoded token, Qwen2.5-14B: it reads the gated product's wide values
        {"name": "quantized_token", "op": "quantized", "m": 1, "k": 13824, "n": 5120, "w": "int8", "limit": 0,
         "bias": False, "residual": True, "pre": False, "parts": False},
        # odd sizes, weights that are not int8, and all that a proof of it reads
        {"name": "quantized_odd", "op": "quantized", "m": 37, "k": 1537, "n": 1111, "w": "m31", "limit": 1 << 20,
         "bias": True, "residual": True, "pre": True, "parts": True},
        # the down projection of a 512-token prompt with its 8-bit rows, the proof's input: the largest product
        {"name": "quantized_prompt", "op": "quantized", "m": 512, "k": 13824, "n": 5120, "w": "int8", "limit": 0,
         "bias": False, "residual": True, "pre": False, "parts": True},
        # one decoded token, SmolLM2-135M (9 query heads on 3 kv heads of 64)
        {"name": "rotary_token", "op": "rotary", "seqs": 1, "tokens": 1, "heads": 9, "kv": 3, "dim": 64, "turned": 64,
         "interleaved": False, "positions": 8192, "stretch": 1.0, "values": "int8", "limit": 127},
        # a decoded token of each of 64 sequences, far along a context that the frequencies are stretched for,
        # Qwen2.5-14B heads
        {"name": "rotary_batch", "op": "rotary", "seqs": 64, "tokens": 1, "heads": 40, "kv": 8, "dim": 128,
         "turned": 128, "interleaved": False, "positions": 131072, "stretch": 4.0, "values": "int8", "limit": 127},
        # two prompts, one of 4096 tokens, half of each head turned, full-range values
        {"name": "rotary_prompt", "op": "rotary", "seqs": 2, "tokens": 4096, "heads": 40, "kv": 8, "dim": 128,
         "turned": 64, "interleaved": True, "positions": 8192, "stretch": 1.0, "values": "m31", "limit": 0},
        # one short prompt with the traces that a proof of it reads, SmolLM2-135M heads
        {"name": "prompt_short", "op": "prompt", "seqs": 1, "tokens": 100, "heads": 9, "kv": 3, "dim": 64,
         "values": "int8", "trace": True},
        # sixteen prompts of very different lengths, Qwen2.5-14B heads, int8-range values
        {"name": "prompt_packed", "op": "prompt", "seqs": 16, "tokens": 1024, "heads": 40, "kv": 8, "dim": 128,
         "values": "int8", "trace": False},
        # one long prompt of int8-range values
        {"name": "prompt_long", "op": "prompt", "seqs": 1, "tokens": 4096, "heads": 40, "kv": 8, "dim": 128,
         "values": "int8", "trace": False},
        # one prompt of full-range values, of odd length
        {"name": "prompt_general", "op": "prompt", "seqs": 1, "tokens": 1501, "heads": 40, "kv": 8, "dim": 128,
         "values": "m31", "trace": False},
    ]


LARGEST = 512 * 13824 * 5120       # multiply-adds of a product; general weights are four digits
LARGEST_SCORES = 40 * 128 * 4096 ** 2  # of a head's values, over all pairs of tokens
LARGEST_TURN = 4096 * 48 * 128     # values


def _size(rng, lo, hi):
    """A size spread over the logarithm of [lo, hi], odd as often as not."""
    v = int(round(lo * (hi / lo) ** rng.random()))
    return max(lo, min(hi, v | 1 if rng.random() < 0.5 else v))


def draw(rng):
    op = rng.choice(["scaled", "quantized", "quantized", "rotary", "prompt", "prompt"])
    if op in ("scaled", "quantized"):
        c = {"op": op, "m": _size(rng, 1, 512), "k": _size(rng, 33, 13824), "n": _size(rng, 33, 13824),
             "w": rng.choice(["int8", "int8", "int8", "m31"])}
        while c["m"] * c["k"] * c["n"] * (4 if c["w"] == "m31" else 1) > LARGEST:
            c["m"] = (c["m"] + 1) // 2
        c.update(limit=rng.choice([127, 127, 1 << 15, 0]), bias=rng.random() < 0.5, residual=rng.random() < 0.5,
                 pre=rng.random() < 0.3)
        if op == "quantized":
            c["parts"] = rng.random() < 0.5
        return c
    c = {"op": op, "kv": rng.choice([1, 2, 3, 4, 8]), "dim": rng.choice([32, 64, 80, 96, 128])}
    c["heads"] = c["kv"] * rng.choice([1, 2, 3, 4, 5, 7, 8])
    if op == "rotary":
        c.update(seqs=_size(rng, 1, 64), tokens=rng.choice([1, _size(rng, 1, 4096)]), turned=c["dim"],
                 interleaved=rng.random() < 0.5, positions=rng.choice([8192, 32768, 131072]),
                 stretch=rng.choice([1.0, 1.0, 2.0, 8.0]))
        if rng.random() < 0.4:
            c["turned"] = 2 * rng.randint(1, c["dim"] // 2)
        c["values"], c["limit"] = rng.choice([("int8", 127), ("int8", 0), ("m31", 0)])
        while c["seqs"] * c["tokens"] * (c["heads"] + c["kv"]) * c["dim"] > LARGEST_TURN:
            c["seqs"], c["tokens"] = (c["seqs"] + 1) // 2, (c["tokens"] + 1) // 2
        return c
    c.update(seqs=rng.choice([1, _size(rng, 1, 32)]), tokens=_size(rng, 1, 4096), values=rng.choice(["int8", "m31"]),
             trace=rng.random() < 0.4)
    cost = 8 if c["values"] == "m31" else 1
    while (c["seqs"] * c["tokens"] ** 2 * c["heads"] * c["dim"] * cost > LARGEST_SCORES
           or c["trace"] and c["seqs"] * c["tokens"] ** 2 * c["heads"] > 1 << 26):
        c["seqs"], c["tokens"] = (c["seqs"] + 1) // 2, 3 * c["tokens"] // 4 + 1
    return c


# ------------------------------------------------------------------ inputs
class Inputs:
    """Seeded words in device memory."""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(seed)

    def ints(self, lo, hi, shape):
        return torch.randint(lo, hi, shape, generator=self.gen, device="cuda", dtype=torch.int32)

    def words(self, shape, values):
        """Quantized values in [-127, 127], negatives as P + v, or words over the whole field."""
        if values == "int8":
            v = self.ints(-127, 128, shape)
            return torch.where(v < 0, v + P, v)
        return self.ints(0, P, shape)

    def wide(self, m, k):
        """What a gated product leaves: rows of very different size, single values far above their row's rest."""
        v = torch.randn((m, k), generator=self.gen, device="cuda") * 2.0 ** 17
        v *= 2.0 ** (8 * torch.rand((m, 1), generator=self.gen, device="cuda"))
        v *= torch.where(torch.rand((m, k), generator=self.gen, device="cuda") < 0.001, 12.0, 1.0)
        v = torch.clamp(v.round(), -float(1 << 29), float(1 << 29)).to(torch.int32)
        return torch.where(v < 0, v + P, v)


def _shift(case):
    """The power of two that brings the sums of a product, times scales of 2^14 .. 2^15, to the size of its
    results: int8, or 20 bits where they are not cut off that low."""
    size = 73.0 * math.sqrt(case["k"]) * (73.0 if case["w"] == "int8" else 2.0 ** 29)
    if case["w"] == "m31":
        size = 2.0 ** 29  # wrapped: any word
    bits = math.log2(size) + 14.5 + (14.5 if case["op"] == "scaled" else 24)
    return int(min(63, max(0, round(bits - (4 if case["limit"] == 127 else 18)))))


def _counts(case):
    """Lengths of the packed sequences, the case's own: the first has `tokens`, one is empty and one a single
    token where there are several, the others are spread evenly."""
    n, t = case["seqs"], case["tokens"]
    counts = [int(v) for v in np.random.default_rng(n * 8192 + t).integers(1, t + 1, size=n)]
    counts[0] = t
    if n > 2 and t > 1:
        counts[1], counts[2] = 0, 1
    return counts


def _frequencies(case):
    """Turns a position, in 2^-64: a geometric series down from 1 / (2 pi); the long waves of a stretched
    context are slowed down by its factor, the short ones stay, those between are in between."""
    half = case["turned"] // 2
    f = 10000.0 ** (-np.arange(half) * 2.0 / case["turned"]) / (2 * np.pi)
    if case["stretch"] != 1.0:
        waves = case["positions"] / case["stretch"] * f
        keep = np.clip((waves - 1) / (4 - 1), 0, 1)
        f = f * (keep + (1 - keep) / case["stretch"])
    return np.floor(f * 2.0 ** 64).astype(np.uint64)


AMPLITUDE, TURN_SHIFT = 1 << 15, 15


def _inputs(case, seed):
    """The tensors of a case, from its seed alone."""
    inp, op = Inputs(seed), case["op"]
    t = {}
    if op in ("scaled", "quantized"):
        m, k, n = case["m"], case["k"], case["n"]
        t["x"] = inp.words((m, k), "int8") if op == "scaled" else inp.wide(m, k)
        t["w"] = inp.words((k, n), case["w"])
        if op == "scaled":
            t["row_scales"] = inp.ints(1 << 14, 1 << 15, (m, 1))
        t["col_scales"] = inp.ints(1 << 14, 1 << 15, (1, n))
        t["bias"] = inp.ints(-20, 21, (1, n)).remainder(P) if case["bias"] else None
        t["residual"] = inp.words((m, n), "int8" if case["limit"] == 127 else "m31") if case["residual"] else None
        return t
    t["counts"] = _counts(case)
    if op == "rotary":  # where the sequences' tokens stand in their contexts
        rng = np.random.default_rng(seed)
        t["starts"] = [int(rng.integers(0, case["positions"] - c + 1)) for c in t["counts"]]
    rows, d = sum(t["counts"]), case["dim"]
    t["q"] = inp.words((rows, case["heads"] * d), case["values"])
    t["k"] = inp.words((rows, case["kv"] * d), case["values"])
    if op == "prompt":
        t["v"] = inp.words((rows, case["kv"] * d), case["values"])
    return t


_contexts = {}


def _framework():
    """The framework's binding and a context on the stream that this program's tensors are made on."""
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "stwo-ml_amd"))
    import gkr_mi355x

    stream = torch.cuda.current_stream().cuda_stream
    if stream not in _contexts:
        _contexts[stream] = gkr_mi355x.Context(0, stream=stream)
    return gkr_mi355x, _contexts[stream]


def _turns(frequencies, positions):
    """C and S of every position, whole numbers: the angle's quarter turn first, in whole numbers, so that
    the rest, at most an eighth of a turn, keeps all of a float64's bits."""
    f = torch.from_numpy(frequencies.view(np.int64)).cuda()
    phase = torch.arange(positions, device="cuda", dtype=torch.int64)[:, None] * f  # mod 2^64
    quarter = ((phase >> 61) + 1) >> 1
    rest = (phase - (quarter << 62)).double() * (2 * math.pi * 2.0 ** -64)
    c, s = torch.cos(rest), torch.sin(rest)
    c, s = (torch.where((quarter & 1) == 0, a, b) for a, b in ((c, -s), (s, c)))
    turned = (quarter & 2) != 0
    return [_round(torch.where(turned, -x, x) * AMPLITUDE).to(torch.int64) for x in (c, s)]


def prepare(case, seed):
    st = _inputs(case, seed)
    st["case"] = case
    op = case["op"]

    def zeros(rows, cols):
        return torch.zeros((rows, cols), device="cuda", dtype=torch.int32)

    if op in ("scaled", "quantized"):
        m, k, n = case["m"], case["k"], case["n"]
        st["out"] = zeros(m, n)
        if case["pre"]:
            st["pre"] = zeros(m, n)
        if op == "quantized" and case["parts"]:
            st["quantized"], st["row_scales"] = zeros(m, k), zeros(m, 1)
    elif op == "rotary":
        st["q_out"], st["k_out"] = torch.zeros_like(st["q"]), torch.zeros_like(st["k"])
        if not own:  # the plan: every position's C and S
            st["turns"] = _turns(_frequencies(case), case["positions"])
            st["at"] = torch.cat([torch.arange(s, s + c, device="cuda") for s, c in zip(st["starts"], st["counts"])])
    else:
        st["out"] = torch.zeros_like(st["q"])
        if case["trace"]:
            rows = len(st["q"])
            st["weighted"], st["sums"] = torch.zeros_like(st["q"]), zeros(rows, case["heads"])
            st["scores"] = zeros(rows * case["heads"], max(st["counts"]))
    if own:  # the handles, and the plan
        _, ctx = _framework()
        st["ctx"] = ctx
        st["h"] = {name: ctx.wrap_device(t.data_ptr(), t.shape[0], t.shape[1]) for name, t in st.items()
                   if isinstance(t, torch.Tensor) and t.dim() == 2 and t.dtype == torch.int32}
        if op == "rotary":
            st["plan"] = ctx.rotary(_frequencies(case), max_positions=case["positions"], amplitude=AMPLITUDE,
                                    shift=TURN_SHIFT)
    torch.cuda.synchronize()
    return st


# ------------------------------------------------------------------ the plain forms
def _centered(w):
    """Words as signed numbers in float64."""
    w = w.double()
    return torch.where(w > HALF, w - P, w)


def _round(x):
    return torch.sign(x) * torch.floor(x.abs() + 0.5)


def _product(x, w, small):
    """X W mod P.  A centered word has 30 bits and K at most 14, so int8-range weights leave the sums below
    2^53; others go in two parts of 16 bits, as do the words of X."""
    if small:
        return (_centered(x) @ _centered(w)).to(torch.int64).remainder(P)
    x, w = x.to(torch.int64), w.to(torch.int64)
    x0, x1, w0, w1 = (x & 0xFFFF).double(), (x >> 16).double(), (w & 0xFFFF).double(), (w >> 16).double()
    low = (x0 @ w0).to(torch.int64)
    mid = (x0 @ w1 + x1 @ w0).to(torch.int64).remainder(P)
    high = (x1 @ w1).to(torch.int64).remainder(P)
    return (low + (mid << 16) + (high << 1)).remainder(P)  # 2^32 = 2 (mod P)


def _rescale(z, r, s, shift):
    """round(c(z) r s / 2^shift) in int64, cut off at +-2^62: magnitudes of up to 92 bits in two parts, the
    lower one of 31."""
    z = torch.where(z > HALF, z - P, z)
    a = z.abs() * r
    high, low = (a >> 31) * s, (a & P) * s
    if shift:
        half = 1 << (shift - 1)
        low = low + (half & P)
        high = high + (half >> 31)
    high, low = high + (low >> 31), low & P
    if shift >= 31:
        t = high >> (shift - 31)
    else:
        t = torch.where(high >> (31 + shift) > 0, 1 << 62, (high << (31 - shift)) | (low >> shift))
    return torch.sign(z) * t


def _plain_product(st):
    case = st["case"]
    x, out = st["x"], {}
    if case["op"] == "quantized":
        c = torch.where(x > HALF, x - P, x).to(torch.int64)
        r = c.abs().amax(1, keepdim=True)
        q = torch.sign(c) * ((2 * 127 * c.abs() + r) // (2 * r).clamp(min=1))
        x = q.remainder(P)
        if case["parts"]:
            out.update(quantized=x.to(torch.int32), row_scales=r.to(torch.int32))
    else:
        r = st["row_scales"].to(torch.int64)
    z = _product(x, st["w"], case["w"] == "int8")
    t = _rescale(z, r, st["col_scales"].to(torch.int64), _shift(case))
    if case["bias"]:
        t = t + _centered(st["bias"]).to(torch.int64)
    limit = case["limit"] or HALF
    y = t.clamp(-limit, limit)
    if case["residual"]:
        y = y + st["residual"]
    out["out"] = y.remainder(P).to(torch.int32)
    if case["pre"]:
        out["pre"] = z.to(torch.int32)
    return out


def _plain_rotary(st):
    case = st["case"]
    turned, limit = case["turned"], case["limit"]
    c, s = (t[st["at"]][:, None, :] for t in st["turns"])
    out = {}
    for name in ("q", "k"):
        x = st[name].reshape(len(st[name]), -1, case["dim"]).to(torch.int64)
        y = x.clone()
        part = torch.where(x[..., :turned] > HALF, x[..., :turned] - P, x[..., :turned])
        if case["interleaved"]:
            x0, x1 = part[..., 0::2], part[..., 1::2]
        else:
            x0, x1 = part[..., : turned // 2], part[..., turned // 2 :]
        pair = []
        for t in (x0 * c - x1 * s, x1 * c + x0 * s):
            t = torch.sign(t) * ((t.abs() + (1 << (TURN_SHIFT - 1))) >> TURN_SHIFT)
            if limit:
                t = t.clamp(-limit, limit)
            pair.append(t.remainder(P))
        y[..., :turned] = torch.stack(pair, -1).flatten(-2) if case["interleaved"] else torch.cat(pair, -1)
        out[name + "_out"] = y.reshape(st[name].shape).to(torch.int32)
    return out


def _plain_prompt(st):
    case = st["case"]
    kv, d, hd = case["kv"], case["dim"], case["heads"]
    g, small = hd // kv, case["values"] == "int8"
    rows, width = len(st["q"]), max(st["counts"])
    q = st["q"].reshape(rows, kv, g, d)
    k, v = (st[name].reshape(rows, kv, d) for name in ("k", "v"))
    out = {"out": torch.zeros((rows, kv, g, d), device="cuda", dtype=torch.int32)}
    if case["trace"]:
        out["weighted"] = torch.zeros_like(out["out"])
        out["sums"] = torch.zeros((rows, kv, g), device="cuda", dtype=torch.int32)
        out["scores"] = torch.zeros((rows, kv, g, width), device="cuda", dtype=torch.int32)
    row0 = 0
    for n in st["counts"]:
        at = slice(row0, row0 + n)
        row0 += n
        if n == 0:
            continue
        seen = torch.tril(torch.ones((n, n), device="cuda", dtype=torch.bool))[:, None, :]
        for h in range(kv):
            qh, kh = q[at, h].reshape(n * g, d), k[at, h]
            if small:
                s = (_centered(qh) @ _centered(kh).t()).to(torch.int64)
            else:
                qi, ki = qh.to(torch.int64), kh.t().to(torch.int64)
                q0, q1, k0, k1 = (qi & 0xFFFF).double(), (qi >> 16).double(), (ki & 0xFFFF).double(), (ki >> 16).double()
                mid, high = (q0 @ k1 + q1 @ k0).to(torch.int64).remainder(P), (q1 @ k1).to(torch.int64).remainder(P)
                s = (q0 @ k0).to(torch.int64) + (mid << 16) + (high << 1)
            x = torch.where(seen, (s + SCORE_OFFSET).remainder(P).reshape(n, g, n), 0)
            e = torch.where(seen, 1 << torch.clamp((x & 0xFFFFF) >> 16, max=10), 0).reshape(n * g, n)
            z = e.sum(-1, keepdim=True)
            e, c = e.double(), _centered(v[at, h])
            high = torch.floor(c / 65536)  # two parts: sums of 2^10 2^16 2^12 and below
            total = ((e @ high).to(torch.int64) << 16) + (e @ (c - 65536 * high)).to(torch.int64)
            mean = torch.sign(total) * torch.div(2 * total.abs() + z, 2 * z, rounding_mode="floor")
            out["out"][at, h] = mean.remainder(P).reshape(n, g, d).to(torch.int32)
            if case["trace"]:
                out["weighted"][at, h] = (total.remainder(P) << 16).remainder(P).reshape(n, g, d).to(torch.int32)
                out["sums"][at, h] = (z.remainder(P) << 16).remainder(P).reshape(n, g).to(torch.int32)
                out["scores"][at, h, :, :n] = x.to(torch.int32)
    shapes = {"out": (rows, hd * d), "weighted": (rows, hd * d), "sums": (rows, hd), "scores": (rows * hd, width)}
    return {name: t.reshape(shapes[name]) for name, t in out.items()}


# ------------------------------------------------------------------ one pass
def run(st):
    case, op = st["case"], st["case"]["op"]
    if not own:
        return {"scaled": _plain_product, "quantized": _plain_product, "rotary": _plain_rotary,
                "prompt": _plain_prompt}[op](st)
    ctx, h = st["ctx"], st["h"]
    if op == "scaled":
        ctx.matmul_forward_scaled(h["x"], h["w"], h["out"], row_scales=h["row_scales"], col_scales=h["col_scales"],
                                  shift=_shift(case), limit=case["limit"], bias=h.get("bias"),
                                  residual=h.get("residual"), pre=h.get("pre"))
        names = ("out", "pre")
    elif op == "quantized":
        ctx.matmul_forward_quantized(h["x"], h["w"], h["out"], levels=127, col_scales=h["col_scales"],
                                     shift=_shift(case), limit=case["limit"], bias=h.get("bias"),
                                     residual=h.get("residual"), pre=h.get("pre"), quantized=h.get("quantized"),
                                     row_scales=h.get("row_scales"))
        names = ("out", "pre", "quantized", "row_scales")
    elif op == "rotary":
        ctx.rotary_forward(st["plan"], h["q"], h["q_out"], st["counts"], case["dim"], starts=st["starts"], k=h["k"],
                           k_out=h["k_out"], interleaved=case["interleaved"], limit=case["limit"])
        names = ("q_out", "k_out")
    else:
        ctx.attention_prompt(h["q"], h["k"], h["v"], st["counts"], case["heads"], case["kv"], h["out"],
                             score_offset=SCORE_OFFSET, table_log_size=20, weighted=h.get("weighted"),
                             sums=h.get("sums"), scores=h.get("scores"))
        names = ("out", "weighted", "sums", "scores")
    return {name: st[name] for name in names if name in st}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    """bytes: each input read once (int8-range weights, which a program keeps, as one byte), each output
    written once.  flops: the products' multiply-adds, two operations each; six a turned pair."""
    op = case["op"]
    if op in ("scaled", "quantized"):
        m, k, n = case["m"], case["k"], case["n"]
        b = (1 if case["w"] == "int8" else 4) * k * n + 4 * m * k + 4 * m * n + 4 * n
        b += 4 * m * n * (case["residual"] + case["pre"]) + (4 * n if case["bias"] else 0)
        if op == "scaled":
            b += 4 * m
        elif case["parts"]:
            b += 4 * m * k + 4 * m
        return {"bytes": b, "flops": 2 * m * k * n}
    counts = _counts(case)
    rows, d, heads = sum(counts), case["dim"], case["heads"] + case["kv"]
    if op == "rotary":
        # the angles of a token are its heads' to share: eight bytes a pair
        return {"bytes": 8 * rows * heads * d + 4 * rows * case["turned"], "flops": 3 * rows * heads * case["turned"]}
    pairs = sum(n * (n + 1) // 2 for n in counts)
    b = 4 * rows * d * (2 * case["heads"] + 2 * case["kv"])
    if case["trace"]:
        b += 4 * rows * case["heads"] * (d + 1 + max(counts))
    return {"bytes": b, "flops": 4 * pairs * case["heads"] * d}


# ------------------------------------------------------------------ the definition, in whole numbers
def _numbers(t):
    a = t.cpu().numpy().astype(np.int64)
    return np.where(a > HALF, a - P, a)


def _exact_product(case, t):
    x, w = _numbers(t["x"]), _numbers(t["w"])
    m, n = case["m"], case["n"]
    got = {}
    if case["op"] == "quantized":
        r = np.abs(x).max(axis=1)
        q = np.zeros_like(x)
        for i in range(m):
            if r[i]:
                q[i] = np.sign(x[i]) * ((254 * np.abs(x[i]) + r[i]) // (2 * r[i]))
        if case["parts"]:
            got["quantized"], got["row_scales"] = q % P, r[:, None]
        x = q
    else:
        r = t["row_scales"].cpu().numpy().astype(np.int64)[:, 0]
    # digits of seven bits of |w|, so that a sum of 2^7 2^7 2^14 is exact in float64
    z = np.zeros((m, n), dtype=np.int64)
    size, sign = np.abs(w), np.sign(w)
    for j in range(5):
        part = (sign * ((size >> (7 * j)) & 127)).astype(np.float64)
        if part.any():
            z = (z + ((x.astype(np.float64) @ part).astype(np.int64) % P) * pow(2, 7 * j, P)) % P
    if case["pre"]:
        got["pre"] = z
    c = np.where(z > HALF, z - P, z)
    s, shift = t["col_scales"].cpu().numpy().astype(np.int64)[0], _shift(case)
    bias = _numbers(t["bias"])[0] if case["bias"] else np.zeros(n, np.int64)
    limit = case["limit"] or HALF
    y = np.empty((m, n), dtype=np.int64)
    whole = s.astype(object)
    for i in range(m):  # Python's integers
        size = np.abs(c[i]).astype(object) * int(r[i]) * whole
        rounded = (2 * size + (1 << shift)) >> (shift + 1)
        t_i = np.where(c[i] < 0, -rounded, rounded) + bias.astype(object)
        y[i] = np.clip(t_i, -limit, limit).astype(np.int64)
    got["out"] = (y + t["residual"].cpu().numpy()) % P if case["residual"] else y % P
    return got


def _exact_rotary(case, t):
    f = _frequencies(case)
    at = np.concatenate([np.arange(s, s + c, dtype=np.uint64) for s, c in zip(t["starts"], t["counts"])])
    phase = at[:, None] * f  # mod 2^64
    angle = phase.astype(np.longdouble) / np.longdouble(2) ** 64 * (8 * np.arctan(np.longdouble(1)))
    c, s = (np.rint(AMPLITUDE * fn(angle)).astype(np.int64) for fn in (np.cos, np.sin))
    half, got = case["turned"] // 2, {}
    for name in ("q", "k"):
        x = _numbers(t[name]).reshape(len(at), -1, case["dim"])
        y = x.copy()
        for j in range(half):
            a, b = (2 * j, 2 * j + 1) if case["interleaved"] else (j, j + half)
            for to, v in ((a, x[..., a] * c[:, j, None] - x[..., b] * s[:, j, None]),
                          (b, x[..., b] * c[:, j, None] + x[..., a] * s[:, j, None])):
                r = (2 * np.abs(v) + (1 << TURN_SHIFT)) // (2 << TURN_SHIFT) * np.sign(v)
                y[..., to] = np.clip(r, -case["limit"], case["limit"]) if case["limit"] else r
        got[name + "_out"] = (y % P).reshape(len(at), -1)
    return got


def _exact_prompt(case, t):
    kv, d, hd = case["kv"], case["dim"], case["heads"]
    g, rows, width = hd // kv, sum(t["counts"]), max(t["counts"])
    q, k, v = (_numbers(t[name]).reshape(rows, -1, d) for name in ("q", "k", "v"))
    out, weighted = np.zeros((rows, hd, d), np.int64), np.zeros((rows, hd, d), np.int64)
    sums, scores = np.zeros((rows, hd), np.int64), np.zeros((rows, hd, width), np.int64)
    row0 = 0
    for n in t["counts"]:
        for h in range(hd):
            qh, kh, vh = q[row0 : row0 + n, h], k[row0 : row0 + n, h // g], v[row0 : row0 + n, h // g]
            x = np.zeros((n, n), np.int64)
            for j in range(4):  # eight bits of the keys at a time: sums of 2^30 2^8 2^8 stay below 2^53
                part = ((kh >> (8 * j)) if j == 3 else (kh >> (8 * j)) & 255).astype(np.float64)
                x = (x + ((qh.astype(np.float64) @ part.T).astype(np.int64) % P << (8 * j)) % P) % P
            x = (x + SCORE_OFFSET) % P
            for i in range(n):
                seen = x[i, : i + 1]
                e = np.int64(1) << np.minimum((seen % (1 << 20)) >> 16, 10)
                z, total = int(e.sum()), e @ vh[: i + 1]  # below 2^10 2^30 2^12
                out[row0 + i, h] = np.sign(total) * ((2 * np.abs(total) + z) // (2 * z)) % P
                weighted[row0 + i, h] = (total % P << 16) % P
                sums[row0 + i, h] = (z << 16) % P
                scores[row0 + i, h, : i + 1] = seen
        row0 += n
    got = {"out": out.reshape(rows, -1), "weighted": weighted.reshape(rows, -1), "sums": sums,
           "scores": scores.reshape(rows * hd, width)}
    return {name: a for name, a in got.items() if name == "out" or case["trace"]}


def exact(case, seed):
    op = case["op"]
    if op in ("scaled", "quantized"):
        if case["m"] * case["k"] * case["n"] * (5 if case["w"] == "m31" else 1) > 1 << 34:
            return None
    elif op == "prompt" and (case["seqs"] + 2) * case["tokens"] ** 2 * case["heads"] * case["dim"] > 1 << 32:
        return None
    t = _inputs(case, seed)
    got = {"scaled": _exact_product, "quantized": _exact_product, "rotary": _exact_rotary,
           "prompt": _exact_prompt}[op](case, t)
    return {name: a.astype(np.int32) for name, a in got.items()}
