"""The beam selection where a thread goes through several rounds of its segment: maxima that rise from round to round, shares' places behind the first round, shares of
many values, and the segment's last place."""
import numpy as np
import pytest

from beam_rounds import KINDS, SHAPES, best_of, rows_of
from helpers import report
from test_beam_bound_cpu import logarithm_off, stated

pytestmark = pytest.mark.gpu

FAR = 1 << 22


@pytest.mark.parametrize("groups,beams,vocab,picks,offset", [(*s[:4], o) for s in SHAPES for o in (0, 1)[:1 + (s[2] <= FAR)]])
def test_many_rounds(nnb, ctx, groups, beams, vocab, picks, offset):
    far = vocab > FAR      # (two different rows in all)
    rng = np.random.default_rng(141)
    score = -np.cumsum(rng.random((len(KINDS), beams)), axis=1).astype(np.float32)
    kinds, wanted = [], []
    if far:
        two = [rows_of("up", 1, vocab, 142)[0], rows_of("few", 1, vocab, 143)[0]]
        rows = [two[b % 2] for b in range(beams)]
        kinds, groups_of = [rows], [0]
        half = [best_of([r], [0.0], picks) for r in two]
        total = np.concatenate([np.float64(score[0, b]) + half[b % 2][0] for b in range(beams)])
        token, parent = np.concatenate([half[b % 2][1] for b in range(beams)]), np.repeat(np.arange(beams), picks)
        order = np.lexsort((token, parent, -total))
        near = min(abs(total[a] - total[c]) for a, c in zip(order[:picks], order[1:]) if parent[a] != parent[c])
        order = order[:picks]
        wanted.append((total[order], token[order], parent[order], near))
    else:
        for k, kind in enumerate(KINDS):
            kinds.append(rows_of(kind, beams, vocab, 144 + k))
            wanted.append(best_of(kinds[-1], score[k], picks))
        groups_of = [g % len(KINDS) for g in range(groups)]
    assert all(w[3] > stated() for w in wanted), [w[3] for w in wanted]
    lb = ctx.alloc(2 * (groups * beams * vocab + offset))
    for g, k in enumerate(groups_of):
        for b in range(beams):
            row = kinds[k][b]
            nnb._check(ctx.L.nn_buf_write(ctx.h, lb, 2 * (offset + (g * beams + b) * vocab), row.ctypes.data, row.nbytes))
        ctx.sync()
    sb, outs = ctx.upload(np.stack([score[k] for k in groups_of])), [ctx.alloc(4 * groups * picks) for _ in range(3)]
    ctx.beam_select(groups, beams, vocab, lb + 2 * offset, 0, sb, None, -1, picks, *outs, None)
    ctx.sync()
    got = [ctx.download(o, (groups, picks), t) for o, t in zip(outs, (np.float32, np.int32, np.int32))]
    for b in (lb, sb, *outs):
        ctx.free(b)
    worst = 0.0
    for g, k in enumerate(groups_of):
        total, token, parent, _ = wanted[k]
        assert np.array_equal(got[1][g], token) and np.array_equal(got[2][g], parent), (g, "far" if far else KINDS[k], got[1][g], token, got[2][g], parent)
        # the result's rounding (half a step, 2^-24 of it), the logarithm's bound, and 2^-40 for what is done in 64 bits
        off, bound = np.abs(got[0][g].astype(np.float64) - total), 2.0 ** -24 * np.abs(total) + logarithm_off(vocab) + 2.0 ** -40
        worst = max(worst, (off / bound).max())
        assert (off <= bound).all(), (g, off, bound)
    report(f"rounds {groups}x{beams} of {vocab}: worst error {worst:.2f} of its bound")
