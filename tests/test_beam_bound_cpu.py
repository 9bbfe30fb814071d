"""How far the logarithms of the beam selection may be off, from the roundings of its exponentials, and that the header says so."""
import os
import re

import numpy as np
import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LOG2E, LN2, L32 = np.float64(1.4426950408889634), np.log(2.0), np.float32(1.4426950408889634)
EX2 = 2.0 ** -22                # ex2.approx.ftz.f32: two units in the last place, of a value whose unit is 2^-23 of it at most
SUM = 5 * 2.0 ** -24            # 32 exponentials are added up in five steps; what comes behind them is exact to 2^-40


def half_step(x):
    """Half a unit in the last place of 32-bit numbers at |x|."""
    return 2.0 ** (np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** -60))) - 24)


def exponential_off(d):
    """Bound of the relative error of exp(-d): the difference is rounded, times the rounded log2 e, the product rounded, then ex2."""
    d = np.asarray(d, np.float64)
    return half_step(d) + half_step(d * LOG2E) * LN2 + d * abs(np.float64(L32) / LOG2E - 1) + EX2


MOST = 65536                    # logits that have one maximum in common: a warp's of a segment (64 rounds of 1024)


def logarithm_off(vocab):
    """Bound of the error of the logarithm of a row's sum.  Of a warp's values it is the maximum's 1 and n others at a distance d, of weight n exp(-d) / (1 + n exp(-d)); where they
    lie at several distances the error is a mean of theirs, so that one distance for all of them is the worst.  What joins warps and segments is exact to 2^-40, and a
    row's error a mean of its warps'."""
    d = np.concatenate([np.linspace(2.0 ** -10, 40, 400001), 2.0 ** np.arange(0, 6), 2.0 ** np.arange(0, 6) / LOG2E])
    others = (min(vocab, MOST) - 1) * np.exp(-d)
    return (exponential_off(d) * others / (1 + others)).max() + SUM


def stated():
    """The header's distance between totals."""
    with open(os.path.join(REPO, "include", "nnopt_b200.h")) as f:
        text = re.sub(r"\s*\n \*\s*", " ", f.read())
    m = re.search(r"totals of different beams which are nearer than 2\^-(\d+) may come in either order", text)
    assert m, "the header states no such distance"
    return 2.0 ** -int(m.group(1))


def rounded_off(peak, values):
    """What rounding alone does to the logarithm of a warp's sum of one peak and MOST - 1 equal values (the power of two taken as exact), for each of these values."""
    m = np.float32(np.float16(peak))
    t = ((values - m).astype(np.float32) * L32).astype(np.float32)
    exact = np.exp(values.astype(np.float64) - np.float64(m))
    return np.log1p(np.exp2(t.astype(np.float64)) * (MOST - 1)) - np.log1p(exact * (MOST - 1))


@pytest.mark.parametrize("vocab", [1000, 49152, 151936, 1 << 20, 1 << 26])
def test_the_header_states_what_two_rows_can_be_apart(vocab):
    assert 2 * logarithm_off(vocab) < stated()


def test_one_peak_and_equal_values():
    """The worst rows, by the roundings of 32-bit numbers themselves: equal values have equal errors, which do not average out."""
    x = np.arange(1, 1 << 16, dtype=np.uint16).view(np.float16).astype(np.float32)
    x = x[np.isfinite(x) & (x >= 2.0 ** -4) & (x < 24)]
    off = np.concatenate([rounded_off(peak, v) for peak in (0.0, 2.0 ** -24, 0.0001, 0.001, 0.0999, 3.0, 10.0) for v in (-x, x[x < np.float32(np.float16(peak))])])
    assert np.abs(off).max() < logarithm_off(MOST) - SUM
    assert off.max() - off.min() < stated()
