"""Frequencies of rotary positions (gkr_rotary_frequencies): the series and its scalings against their formulas,
and what is refused (no GPU)."""
import math
from fractions import Fraction

import gkr_mi355x as G
import numpy as np
import pytest


def turns(freqs):
    return [float(Fraction(int(f), 1 << 64)) for f in freqs]


def plain(turned, base):
    return [base ** (-2 * i / turned) / (2 * math.pi) for i in range(turned // 2)]


# pow, the division and the scalings' steps are each off by an ulp or two: far below 1e-13
def close(a, b):
    return all(abs(x - y) <= 1e-13 * y + 2.0 ** -63 for x, y in zip(a, b)) and len(a) == len(b)


@pytest.mark.parametrize("turned", [2, 4, 64, 80, 128, 1024])
@pytest.mark.parametrize("base", [10000.0, 500000.0, 1e6])
def test_series_and_scalings(turned, base):
    f = plain(turned, base)
    assert close(turns(G.rotary_frequencies(turned, base)), f)
    assert close(turns(G.rotary_frequencies(turned, base, G.ROTARY_LINEAR, 4.0)), [x / 4 for x in f])
    wide = base * 8.0 ** (turned / (turned - 2)) if turned > 2 else base
    assert close(turns(G.rotary_frequencies(turned, base, G.ROTARY_BASE, 8.0)), plain(turned, wide))
    got = turns(G.rotary_frequencies(turned, base, G.ROTARY_WAVES, 8.0, positions=8192, low=1, high=4))
    want = []
    for x in f:
        w = 8192 * x
        g = 0.0 if w <= 1 else 1.0 if w >= 4 else (w - 1) / 3
        want.append(x * (g + (1 - g) / 8))
    assert close(got, want)


def test_whole_turns_drop_out():
    # a factor below one makes the first frequency more than a turn
    got = turns(G.rotary_frequencies(4, 10000.0, G.ROTARY_LINEAR, 1 / 16))
    assert abs(got[0] - (16 / (2 * math.pi) - 2)) < 1e-14


def test_refusals():
    for args in ((0,), (3,), (65538,), (4, 0.0), (4, -1.0), (4, math.inf), (4, math.nan), (4, 1e4, 9, 1.0), (4, 1e4, 1, 0.0),
                 (4, 1e4, 2, -2.0), (4, 1e4, 3, math.nan, 10.0, 1.0, 4.0), (4, 1e4, 3, 2.0, 0.0, 1.0, 4.0),
                 (4, 1e4, 3, 2.0, 10.0, 4.0, 4.0), (4, 1e4, 3, 2.0, 10.0, -1.0, 4.0)):
        with pytest.raises(G.GkrError) as e:
            G.rotary_frequencies(*args)
        assert e.value.code == 1, args
    assert G.lib().gkr_rotary_frequencies(4, 1e4, None, None) == 1
    assert len(np.unique(G.rotary_frequencies(128))) == 64


def test_frequencies_past_float64_are_refused():
    """Turns a position, or a changed base, that a float64 does not hold: not zeros for them."""
    for args in ((128, 1e-320), (128, 1e4, G.ROTARY_LINEAR, 1e-320), (128, 1e308, G.ROTARY_BASE, 1e10),
                 (128, 1e-308, G.ROTARY_BASE, 1e-30), (4, 1e4, G.ROTARY_BASE, 1e300)):
        with pytest.raises(G.GkrError, match="base") as e:
            G.rotary_frequencies(*args)
        assert e.value.code == 1, args
    assert close(turns(G.rotary_frequencies(2, 1e308)), [1 / (2 * math.pi)])
