"""The best continuations of groups of beams against log-softmax and a sort in 64 bits."""
import numpy as np
import pytest

import branch_reference as br
from helpers import alloc_with_canary, check_canary, report

pytestmark = pytest.mark.gpu

# Totals of different beams that are nearer than this may come in another order: both are sums of 64-bit numbers, but the exponentials under the
# logarithm may have 32 bits.  Inputs are drawn so that none are (asserted on the host, before the call).
NEAR = 2.0 ** -19


def run(nnb, ctx, logits, vocab, score, done, eos, picks, in_place=False, offset=0):
    groups, beams = score.shape
    raw = np.concatenate([np.zeros(offset, np.float16), logits.reshape(-1)])
    lb, sb, db = ctx.upload(raw), ctx.upload(score), None if done is None else ctx.upload(done)
    n = groups * picks * 4
    outs = [alloc_with_canary(ctx, n) for _ in range(4)]
    if in_place:
        os_, od = sb, db
    else:
        os_, od = outs[0], outs[3] if done is not None else None
    ctx.beam_select(groups, beams, vocab, lb + 2 * offset, logits.shape[-1], sb, db, eos, picks, os_, outs[1], outs[2], od)
    ctx.sync()
    got = [ctx.download(o, (groups, picks), t) if o else None for o, t in ((os_, np.float32), (outs[1], np.int32), (outs[2], np.int32), (od, np.int32))]
    for o in outs:
        check_canary(ctx, o, n)
    if not in_place:
        assert np.array_equal(ctx.download(sb, score.shape, np.float32), score, equal_nan=True)
    for b in (lb, sb, *outs, *([db] if db else [])):
        ctx.free(b)
    return got


def check(got, logits, vocab, score, done, eos, picks, what=""):
    worst = 0.0
    for g in range(len(score)):
        want, token, parent, near = br.best_continuations(logits[g, :, :vocab], score[g], None if done is None else done[g], eos, picks)
        assert near > NEAR or near == 0, (what, g, near)
        assert np.array_equal(got[1][g], token) and np.array_equal(got[2][g], parent), (what, g, got[1][g], token, got[2][g], parent)
        there = token >= 0
        assert (got[0][g][~there] == -np.inf).all()
        # the result's rounding (half a step, 2^-24 of it), and the logarithm of a sum whose terms have 32 bits: 2^-21 of the sum at most
        off = np.abs(got[0][g][there].astype(np.float64) - want[there])
        bound = 2.0 ** -24 * np.abs(want[there]) + 2.0 ** -21
        if off.size:
            worst = max(worst, (off / bound).max())
        assert (off <= bound).all(), (what, g, off, bound)
        if got[3] is not None:
            assert np.array_equal(got[3][g], ((token == eos) & there).astype(np.int32))
    report(f"beams {what}: worst error {worst:.2f} of its bound")


def draw(groups, beams, vocab, seed, pad=0, spread=2.5):
    rng = np.random.default_rng(seed)
    logits = (rng.standard_normal((groups, beams, vocab + pad)) * spread).astype(np.float16)
    logits[..., vocab:] = 1000
    score = -np.cumsum(rng.random((groups, beams)), axis=1).astype(np.float32)
    return logits, score


SHAPES = [(1, 4, 49152, 4, 0), (3, 5, 65535, 10, 65), (2, 1, 1, 1, 0), (2, 3, 7, 5, 0), (1, 1, 100, 32, 3), (5, 32, 333, 32, 1), (2, 8, 151936, 16, 0), (40, 4, 1000, 8, 0), (1, 2, 31, 32, 0),
          (300, 2, 257, 3, 7), (1, 1, 1000003, 20, 0)]


@pytest.mark.parametrize("groups,beams,vocab,picks,pad", SHAPES)
def test_picks(nnb, ctx, groups, beams, vocab, picks, pad):
    logits, score = draw(groups, beams, vocab, 91, pad)
    for offset in (0, 1):      # (rows that begin at an odd value)
        got = run(nnb, ctx, logits, vocab, score, None, -1, picks, offset=offset)
        check(got, logits, vocab, score, None, -1, picks, f"{groups}x{beams} of {vocab}")
    again = run(nnb, ctx, logits, vocab, score, None, -1, picks, offset=1)     # (the same call: where the rows begin decides which values are added up first)
    assert all(np.array_equal(a, b) for a, b in zip(got[:3], again[:3]))


@pytest.mark.parametrize("groups,beams,vocab,picks", [(1, 4, 49152, 4), (6, 7, 5000, 7), (3, 16, 2049, 16), (2, 32, 40, 32)])
def test_beams_that_have_ended(nnb, ctx, groups, beams, vocab, picks):
    logits, score = draw(groups, beams, vocab, 92)
    rng = np.random.default_rng(93)
    done = rng.integers(0, 3, (groups, beams)).astype(np.int32) * rng.integers(0, 2, (groups, beams)).astype(np.int32)
    done[0, 0] = 5
    logits[done != 0] = np.nan            # not looked at
    for eos in (0, vocab - 1):
        logits[0, -1, eos] = 12 if done[0, -1] == 0 else np.nan     # an end among the picks
        for in_place in (False, True):
            got = run(nnb, ctx, logits, vocab, score, done, eos, picks, in_place)
            check(got, logits, vocab, score, done, eos, picks, f"ended, {groups}x{beams} of {vocab}")
    # all have ended: as many candidates as beams
    done[:] = 1
    got = run(nnb, ctx, logits, vocab, score, done, 3, 32)
    check(got, logits, vocab, score, done, 3, 32, "all ended")
    assert (got[1][:, beams:] == -1).all() and (got[2][:, :beams] == np.argsort(-score, axis=1, kind="stable")).all()


def test_ends_without_flags(nnb, ctx):
    """out_done alone: which of the picks are ends."""
    logits, score = draw(2, 3, 500, 94)
    logits[:, 1, 77] = 11
    lb, sb = ctx.upload(logits), ctx.upload(score)
    outs = [ctx.alloc(2 * 6 * 4) for _ in range(4)]
    ctx.beam_select(2, 3, 500, lb, 0, sb, None, 77, 6, *outs)
    ctx.sync()
    got = [ctx.download(o, (2, 6), t) for o, t in zip(outs, (np.float32, np.int32, np.int32, np.int32))]
    check(got, logits, 500, score, None, 77, 6, "ends")
    assert (got[3] == (got[1] == 77)).all() and got[3].any()
    for b in (lb, sb, *outs):
        ctx.free(b)


@pytest.mark.parametrize("vocab", [9, 5000, 70000])
def test_ties(nnb, ctx, vocab):
    """Equal totals: the lowest beam, then the lowest token.  Equal rows and scores, equal logits, both zeros, nothing but one value."""
    rng = np.random.default_rng(95)
    row = rng.integers(-3, 4, vocab).astype(np.float16)                # few different values
    zeros = np.where(rng.random(vocab) < 0.5, 0.0, -0.0).astype(np.float16)
    logits = np.stack([np.stack([row, row, row]), np.stack([zeros, zeros, zeros]), np.full((3, vocab), 2.0, np.float16),
                       np.stack([np.full(vocab, -1.0), np.full(vocab, 7.0), np.full(vocab, 65504.0)]).astype(np.float16)])
    score = np.array([[-1, -1, -1], [-2, -1, -1], [-1, -1, -1], [-0.5, -0.5, -0.5]], np.float32)
    for picks in (1, 3, 9, 32):
        got = run(nnb, ctx, logits, vocab, score, None, -1, picks)
        check(got, logits, vocab, score, None, -1, picks, f"ties of {vocab}")


@pytest.mark.parametrize("vocab", [50, 33000])
def test_values_that_are_not_numbers(nnb, ctx, vocab):
    """Masked logits are never picked; rows with a NaN or an infinity, rows without a logit and beams without a score have no candidates."""
    rng = np.random.default_rng(96)
    logits, score = draw(8, 3, vocab, 97)
    logits[0, :, 5:] = -np.inf                                          # five tokens of each beam are left
    logits[1, 0] = -np.inf
    logits[2, 1, vocab // 2] = np.nan
    logits[3, 2, vocab - 1] = np.inf
    score[4, 0] = -np.inf
    score[5, 1] = np.nan
    logits[6] = -np.inf                                                 # none at all
    score[7] = [0, -np.inf, -np.inf]                                    # the first step: one beam
    logits[7, 0, rng.integers(0, vocab, 20)] = -65504
    for picks in (3, 20):
        got = run(nnb, ctx, logits, vocab, score, None, -1, picks)
        check(got, logits, vocab, score, None, -1, picks, "not numbers")
    assert (got[1][6] == -1).all() and (got[2][7][got[2][7] >= 0] == 0).all() and (got[1][0] >= 0).sum() == 15


@pytest.mark.parametrize("order", ["up", "down", "late", "wide"])
def test_orders_of_logits(nnb, ctx, order):
    """Rows whose values rise or fall all along, whose best ones come last or lie together, and values as far apart as fp16 has them."""
    vocab, beams = 60001, 2
    rng = np.random.default_rng(98)
    x = np.sort(rng.standard_normal((1, beams, vocab)) * 3, axis=-1)
    if order == "down":
        x = x[..., ::-1]
    elif order == "late":
        x = rng.permuted(x, axis=-1)
        x[..., -40:] += 8
    elif order == "wide":
        x = rng.permuted(x, axis=-1) * 15000
        x = np.clip(x, -65504, 65504)
    logits, score = np.ascontiguousarray(x).astype(np.float16), np.array([[-1.25, -1.7]], np.float32)
    for picks in (1, 8, 32):
        got = run(nnb, ctx, logits, vocab, score, None, -1, picks)
        check(got, logits, vocab, score, None, -1, picks, order)


def test_rows_beyond_32_bits(nnb, ctx):
    """Rows that lie more than 2^32 bytes apart."""
    stride, vocab = (1 << 31) + 1001, 3000
    logits, score = draw(1, 2, vocab, 99)
    buf = ctx.alloc(2 * (stride + vocab))
    for i in range(2):
        row = np.ascontiguousarray(logits[0, i])
        nnb._check(ctx.L.nn_buf_write(ctx.h, buf, 2 * stride * i, row.ctypes.data, row.nbytes))
        ctx.sync()
    sb, outs = ctx.upload(score), [ctx.alloc(64) for _ in range(3)]
    ctx.beam_select(1, 2, vocab, buf, stride, sb, None, -1, 4, *outs, None)
    ctx.sync()
    got = [ctx.download(o, (1, 4), t) for o, t in zip(outs, (np.float32, np.int32, np.int32))] + [None]
    check(got, logits, vocab, score, None, -1, 4, "far rows")
    for b in (buf, sb, *outs):
        ctx.free(b)


@pytest.mark.parametrize("vocab,beams", [(200003, 1), (400000, 2), (1000000, 1), (30000, 24)])
def test_equal_values_in_many_places(nnb, ctx, vocab, beams):
    """More equal values than a block compares at once, among the shares' largest ones and within shares: the first tokens of them."""
    rng = np.random.default_rng(101)
    flat = np.full(vocab, 0.25, np.float16)
    few = (rng.integers(0, 2, vocab) * 3).astype(np.float16)
    edge = np.where(np.arange(vocab) % 9000 < 20, 4.0, rng.integers(-2, 4, vocab)).astype(np.float16)      # twenty in a row, in every segment
    rows = np.stack([flat, few, edge])
    logits = np.ascontiguousarray(np.repeat(rows[:, None], beams, 1))
    score = np.repeat([[-0.5], [-1.0], [-1.5]], beams, 1).astype(np.float32)
    for picks in (8, 31, 32):
        got = run(nnb, ctx, logits, vocab, score, None, -1, picks)
        check(got, logits, vocab, score, None, -1, picks, f"equal values of {vocab}")


def test_scores_that_are_not_finite(nnb, ctx):
    """An infinite score is none, of a beam that goes on and of one that has ended."""
    logits, score = draw(2, 4, 700, 102)
    done = np.array([[0, 0, 1, 1], [1, 0, 0, 0]], np.int32)
    score[0, 1] = score[0, 2] = score[1, 0] = np.inf
    score[1, 2] = -np.inf
    got = run(nnb, ctx, logits, 700, score, done, 9, 6)
    none = np.where(np.isfinite(score), score, -np.inf).astype(np.float32)
    check(got, logits, 700, none, np.where(np.isfinite(score), done, 0), 9, 6, "scores that are not finite")
    assert not np.isin(got[2][0], (1, 2)).any() and not np.isin(got[2][1], (0, 2)).any()


@pytest.mark.parametrize("groups,beams,vocab,picks", [(1, 16, 49152, 10), (1, 16, 49152, 11), (1, 21, 49152, 8), (1, 22, 49152, 8), (98, 1, 49152, 7), (99, 1, 49152, 7), (4, 16, 1000, 8), (4, 17, 1000, 8),
                                                   (1, 2, 500000, 2), (37, 4, 32000, 1)])
def test_few_and_many_segments(nnb, ctx, groups, beams, vocab, picks):
    """Calls on both sides of what decides whether rows' or segments' candidates are joined: some beams ended, without a score or with a NaN, results in place; the next call
    finds lists of another one's."""
    for seed in (111, 112):
        logits, score = draw(groups, beams, vocab, seed)
        rng = np.random.default_rng(seed)
        done = (rng.random((groups, beams)) < 0.2).astype(np.int32)
        score[rng.random((groups, beams)) < 0.1] = -np.inf
        bad = rng.random((groups, beams)) < 0.1
        logits[bad, rng.integers(0, vocab)] = np.nan
        for in_place in (False, True)[:1 + (picks == beams)]:
            got = run(nnb, ctx, logits, vocab, score, done, vocab // 2, picks, in_place)
            check(got, logits, vocab, score, done, vocab // 2, picks, f"{groups}x{beams} of {vocab}, {picks} picks")
