"""The logarithms of the beam selection where its roundings add up: rows of one peak and equal values, and maxima that rise round after round."""
import numpy as np
import pytest

from helpers import report
from test_beam_bound_cpu import MOST, logarithm_off, rounded_off

pytestmark = pytest.mark.gpu


def logarithms(nnb, ctx, rows, tokens, vocab, beams=32):
    """rows: of fp16 logits, `vocab` each; the largest of row i is at tokens[i] and nowhere else.  Its total is score - log(sum of exponentials of differences to it), and
    the score is that logarithm, rounded: the total is small, and shows the kernel's logarithm to 2^-24 of its distance.  -> the error of each logarithm."""
    n = len(rows)
    groups, kinds = -(-n // beams), {}
    lb = ctx.alloc(2 * groups * beams * vocab)
    exact = np.zeros(groups * beams)
    for i in range(groups * beams):
        row = rows[i % n]
        if id(row) not in kinds:
            x = row.astype(np.float64)
            e = np.exp(x - x.max())
            kinds[id(row)] = np.log1p(np.sort(np.delete(e, e.argmax())).sum())
        exact[i] = kinds[id(row)]
        nnb._check(ctx.L.nn_buf_write(ctx.h, lb, 2 * vocab * i, row.ctypes.data, row.nbytes))
    ctx.sync()
    score = exact.astype(np.float32)
    sb, outs = ctx.upload(score.reshape(groups, beams)), [ctx.alloc(4 * groups * beams) for _ in range(3)]
    ctx.beam_select(groups, beams, vocab, lb, 0, sb, None, -1, beams, *outs, None)
    ctx.sync()
    total, token, parent = [ctx.download(o, (groups, beams), t) for o, t in zip(outs, (np.float32, np.int32, np.int32))]
    for b in (lb, sb, *outs):
        ctx.free(b)
    off = np.zeros(groups * beams)
    for g in range(groups):
        assert np.array_equal(np.sort(parent[g]), np.arange(beams)), (g, parent[g])      # (every other logit is far below)
        for p in range(beams):
            i = g * beams + parent[g, p]
            assert token[g, p] == tokens[i % n], (i, token[g, p])
            off[i] = (np.float64(score[i]) - exact[i]) - np.float64(total[g, p])
    return off


@pytest.mark.parametrize("vocab,beams,count", [(49152, 4, 64), (49152, 32, 128), (151936, 32, 128), (1 << 20, 32, 64)])
def test_one_peak_and_equal_values(nnb, ctx, vocab, beams, count):
    rng = np.random.default_rng(131)
    step = 2.0 ** -7                  # of fp16 numbers between 8 and 16
    rows, tokens = [], []
    for i in range(count):
        row = np.full(vocab, -(8 + step * int(rng.integers(0, 1024))) if i >= 8 else -(11.09375 + step * (i // 4)), np.float16)
        tokens.append(int(rng.integers(0, vocab)))
        row[tokens[-1]] = (0.0, 0.0001, 0.0999, 0.5)[i % 4]
        rows.append(row)
    off, bound = logarithms(nnb, ctx, rows, tokens, vocab, beams), logarithm_off(vocab) + 2.0 ** -40
    report(f"one peak, {vocab}: errors {off.min() * 2 ** 20:.3f} to {off.max() * 2 ** 20:.3f} of 2^-20, bound {bound * 2 ** 20:.3f}")
    assert (np.abs(off) <= bound).all(), (off.min(), off.max(), bound)


@pytest.mark.parametrize("of_a_kind", [1, 37])
def test_maxima_that_rise(nnb, ctx, of_a_kind):
    """Rows that rise or fall in steps, one every 8192 values: a thread's maximum rises in each round of its segment (two, and 64, rounds to a segment)."""
    vocab, rows = 1 << 20, []
    for low, step in [(-1, 2.0 ** -11), (-2, 2.0 ** -10), (-4, 2.0 ** -9), (-4, 2.0 ** -7), (-8, 2.0 ** -6), (-8, 0.0625), (-16, 0.109375), (-16, 0.125), (-32, 0.25), (-64, 0.5), (-64, 0.4375),
                      (-128, 1), (-700, 5.5), (0, 2.0 ** -10), (0, 2.0 ** -24), (3, 0.0234375)]:
        for down in (False, True):
            row = (low + step * (np.arange(vocab) // 8192)).astype(np.float16)
            row = np.ascontiguousarray(row[::-1]) if down else row
            row[-1] = row.max() + np.float16(max(step, 2.0 ** -9))
            assert (row == row[-1]).sum() == 1
            rows.append(row)
    off, bound = logarithms(nnb, ctx, rows * of_a_kind, [vocab - 1] * len(rows) * of_a_kind, vocab), logarithm_off(vocab) + 2.0 ** -40
    report(f"rising maxima, {len(off)} rows: errors {off.min() * 2 ** 20:.3f} to {off.max() * 2 ** 20:.3f} of 2^-20, bound {bound * 2 ** 20:.3f}")
    assert (np.abs(off) <= bound).all(), (off.min(), off.max(), bound)


def test_a_peak_for_every_warp(nnb, ctx):
    """The worst rows: in each warp's part of a segment one peak, and behind it equal values whose errors go the same way."""
    vocab, rows, wanted = 1 << 20, [], []
    for peak in (0.0, 0.0001, 0.0999, 0.5):
        values = np.float32(np.float16(peak)) - np.arange(5, 14, 2.0 ** -8, dtype=np.float32)
        values = np.unique(values.astype(np.float16)).astype(np.float32)
        off = rounded_off(peak, values)
        for i in (*np.argsort(off)[:4], *np.argsort(off)[-4:]):
            row = np.full(vocab, values[i], np.float16)
            for segment in range(0, vocab, 8 * MOST):
                row[segment:segment + 8 * 256:256] = peak
            row[7 * 256] = peak + 2.0 ** -9
            rows.append(row)
            wanted.append(off[i])
    off, bound = logarithms(nnb, ctx, rows * 37, [7 * 256] * len(rows) * 37, vocab), logarithm_off(vocab) + 2.0 ** -40
    report(f"a peak for every warp: errors {off.min() * 2 ** 20:.3f} to {off.max() * 2 ** 20:.3f} of 2^-20 (by rounding alone {min(wanted) * 2 ** 20:.3f} to {max(wanted) * 2 ** 20:.3f}), "
           f"bound {bound * 2 ** 20:.3f}")
    assert (np.abs(off) <= bound).all(), (off.min(), off.max(), bound)
    assert off.max() - off.min() > 2.0 ** -21      # (otherwise these are not the rows that they are meant to be)
