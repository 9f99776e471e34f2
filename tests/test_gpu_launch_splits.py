"""Calls that take several launches of a kernel, with rows on both sides of each cut against whole numbers: turns past
2^22 rows, prompts whose packing passes 2^14 blocks and whose items pass 2^22, rows past 2^21 that are quantized by a
launch of their own.  And a table of turns that memory does not hold."""
import numpy as np
import pytest

import gkr_mi355x as G
from test_gpu_operator_calls import OFFSET
from test_gpu_prompt import attend
from test_gpu_rotary import table, turn
from test_gpu_scaled import centered, quantize
from test_gpu_witness import product, words

pytestmark = pytest.mark.gpu
P = G.P


def part(ctx, m, first, rows):
    """Some rows of a matrix, as a matrix over the same memory."""
    return ctx.wrap_device(m.device_ptr + 4 * first * m.cols, rows, m.cols)


@pytest.mark.parametrize("interleaved", [False, True])
def test_turns_past_one_launch(gpu_ctx, interleaved):
    cut = 1 << 22  # rows of a launch; the second sequence goes on in the next
    counts, starts = [5, cut - 3, 40], [3, 10, 100]
    rows = sum(counts)
    q, out = gpu_ctx.synthetic(rows, 2, 0, 3), gpu_ctx.synthetic(rows, 2, 0, 4)
    freqs = np.array([0x0123456789abcdef], dtype=np.uint64)
    rotary = gpu_ctx.rotary(freqs, cut + 100)
    gpu_ctx.rotary_forward(rotary, q, out, counts, 2, starts=starts, interleaved=interleaved)
    at = np.concatenate([np.arange(s, s + c) for s, c in zip(starts, counts)])
    for first, n in ((0, 20), (cut // 2, 20), (cut - 30, rows - cut + 30)):
        c, s = table(freqs, at[first : first + n], 1 << 15)
        want = turn(part(gpu_ctx, q, first, n).download(), c, s, 2, 15, interleaved, 0)
        assert np.array_equal(part(gpu_ctx, out, first, n).download(), want), first
    halves = gpu_ctx.synthetic(rows, 2, 0, 5)
    half = 5 + cut // 2
    for first, n, count, start in ((0, half, [5, half - 5], [3, 10]), (half, rows - half, [cut - 3 - half + 5, 40], [10 + half - 5, 100])):
        gpu_ctx.rotary_forward(rotary, part(gpu_ctx, q, first, n), part(gpu_ctx, halves, first, n), count, 2, starts=start,
                               interleaved=interleaved)
    assert np.array_equal(out.download(), halves.download())
    rotary.free()


def means(q, k, v, token):
    """A token of one sequence of one head of one dim: its sum of weights and its mean."""
    x = (OFFSET + centered(k[: token + 1]) * int(centered(q[token : token + 1])[0]) % P) % P
    w = np.int64(1) << np.minimum((x % (1 << 20)) >> 16, 10)
    z, total = int(w.sum()), int((w.astype(object) * centered(v[: token + 1])).sum())
    return (z << 16) % P, (1 if total > 0 else -1) * ((2 * abs(total) + z) // (2 * z)) % P


@pytest.mark.parametrize("general", [False, True])
def test_packing_past_one_launch(gpu_ctx, general, write_words):
    """127 sequences of 130 blocks; general: one word of the last sequence's keys and one of its values."""
    counts = [8300 - i % 50 for i in range(127)]
    assert sum((c + 63) // 64 for c in counts) > 1 << 14
    rows = sum(counts)
    q, k, v = (gpu_ctx.synthetic(rows, 1, 1, 11 + i) for i in range(3))
    gpu_ctx.synchronize()
    if general:
        write_words(k, rows - 100, [123456789])
        write_words(v, rows - 70, [987654321])
    out, sums = gpu_ctx.synthetic(rows, 1, 0, 14), gpu_ctx.synthetic(rows, 1, 0, 15)
    gpu_ctx.attention_prompt(q, k, v, counts, 1, 1, out, score_offset=OFFSET, sums=sums)
    q, k, v, out, sums = (t.download()[:, 0] for t in (q, k, v, out, sums))
    first = np.concatenate([[0], np.cumsum(counts)])
    for i in (0, 1, 63, 124, 125, 126):
        here = slice(first[i], first[i + 1])
        for token in (0, 63, 64, 4099, counts[i] - 100, counts[i] - 65, counts[i] - 1):
            got = int(sums[here][token]), int(out[here][token])
            assert got == means(q[here], k[here], v[here], token), (i, token)


@pytest.mark.parametrize("general", [False, True])
def test_items_past_one_launch(general, write_words):
    """115 sequences of ten tiles by 4096 kv heads are more than 2^22 items; general: queries of the shortest
    sequence, which the last launch takes."""
    heads, counts = 4096, [577 + i * 7 % 24 for i in range(115)]
    assert sum((c + 63) // 64 for c in counts) * heads > 1 << 22
    first = np.concatenate([[0], np.cumsum(counts)])
    shortest, longest = (int(f(counts)) for f in (np.argmin, np.argmax))
    ctx = G.Context(0)  # its work buffers take 39 GB
    rows = sum(counts)
    k, out = ctx.synthetic(rows, heads, 1, 21), ctx.synthetic(rows, heads, 0, 22)
    q = ctx.synthetic(rows, heads, 1, 23) if general else k
    ctx.synchronize()
    if general:
        write_words(q, int(first[shortest] + 300) * heads + 4095, [1 << 29])
    ctx.attention_prompt(q, k, k, counts, heads, heads, out, score_offset=OFFSET)
    for i in (0, 57, 114, shortest, longest):
        Q, K, got = (part(ctx, t, int(first[i]), counts[i]).download() for t in (q, k, out))
        for h in (0, 1777, 4095):
            want = attend(*(t[:, h : h + 1] for t in (Q, K, K)), 1, 1, OFFSET, 20, counts[i])[0]
            assert np.array_equal(got[:, h : h + 1], want), (i, h)
    ctx.close()


def test_quantized_rows_past_one_launch(gpu_ctx):
    m, k, n = (1 << 22) + 3, 4, 3
    rng = np.random.default_rng(8)
    a, b = gpu_ctx.synthetic(m, k, 0, 31), words(rng, (k, n), 1)
    s = rng.integers(1 << 13, 1 << 14, size=n)
    out, q, r, z = (gpu_ctx.synthetic(m, c, 0, 32 + c) for c in (n, k, 1, n))
    gpu_ctx.matmul_forward_quantized(a, gpu_ctx.upload(b), out, col_scales=gpu_ctx.upload(s.reshape(1, n).astype(np.uint32)),
                                     shift=30, quantized=q, row_scales=r, pre=z)
    want, scale = quantize(a.download(), 127)
    assert np.array_equal(q.download(), want)
    assert np.array_equal(r.download()[:, 0], scale)
    Z = product(want.astype(np.uint32), b)
    assert np.array_equal(z.download(), Z)
    c = centered(Z)  # below 2^16; by scales of 30 and 14 bits whole in 64
    t = (2 * np.abs(c) * scale[:, None] * s + (1 << 30)) >> 31
    assert np.array_equal(out.download(), np.clip(np.where(c < 0, -t, t), -(P // 2), P // 2) % P)


def test_table_larger_than_memory(gpu_ctx):
    """Turns of 2^31 positions by 32768 pairs, 512 TiB: the code says what was short, and the context goes on."""
    with pytest.raises(G.GkrError, match="the table") as e:
        gpu_ctx.rotary(np.arange(32768, dtype=np.uint64), 1 << 31)
    assert e.value.code == 4
    gpu_ctx.rotary(np.arange(4, dtype=np.uint64), 10).free()
