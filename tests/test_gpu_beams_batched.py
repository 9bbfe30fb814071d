"""The beam selection where rows have several segments and are joined one by one."""
import numpy as np
import pytest

from test_gpu_beams import check, draw

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("groups,beams,vocab,picks", [(64, 8, 151936, 16), (40, 8, 60001, 8)])
def test_the_same_call_again_and_again(nnb, ctx, groups, beams, vocab, picks):
    """The last block of each row and of each group is another one every time; all of them see all that the others have written."""
    logits, score = draw(1, beams, vocab, 121)
    lb = ctx.alloc(2 * groups * beams * vocab)
    for g in range(groups):      # (each group has the first one's rows, begun one value later)
        row = np.roll(logits, g, axis=-1)
        nnb._check(ctx.L.nn_buf_write(ctx.h, lb, 2 * beams * vocab * g, row.ctypes.data, row.nbytes))
        ctx.sync()
    sb, outs = ctx.upload(np.repeat(score, groups, 0)), [ctx.alloc(4 * groups * picks) for _ in range(3)]
    first = None
    for turn in range(60):
        ctx.beam_select(groups, beams, vocab, lb, 0, sb, None, -1, picks, *outs, None)
        ctx.sync()
        got = [ctx.download(o, (groups, picks), t) for o, t in zip(outs, (np.float32, np.int32, np.int32))]
        if turn == 0:
            for g in (0, 1, groups - 1):
                check([x[g:g + 1] for x in got] + [None], np.roll(logits, g, axis=-1), vocab, score, None, -1, picks, f"group {g} of {groups}")
            first = got
        assert all(np.array_equal(a, b) for a, b in zip(got, first)), turn
    for b in (lb, sb, *outs):
        ctx.free(b)


@pytest.mark.parametrize("groups,beams,vocab,picks", [(1, 8, 5000, 5), (2, 8, 60001, 9), (60, 8, 60001, 9)])
def test_rows_without_numbers(nnb, ctx, groups, beams, vocab, picks):
    """Rows of nothing but NaN, of NaN where one warp, one round or one segment reads, of infinities, and of no logit until the last token."""
    logits, score = draw(1, beams, vocab, 122)
    x = logits[0]
    x[0] = np.nan
    x[1] = -np.float16(np.nan)
    x[2, 256:512] = np.nan
    x[3, vocab // 2:] = np.nan
    x[4] = np.inf
    x[5] = -np.inf
    x[5, -1] = 3
    x[6, :vocab - 3] = -np.inf
    lb, sb = ctx.upload(np.repeat(logits, groups, 0)), ctx.upload(np.repeat(score, groups, 0))
    outs = [ctx.alloc(4 * groups * picks) for _ in range(3)]
    ctx.beam_select(groups, beams, vocab, lb, 0, sb, None, -1, picks, *outs, None)
    ctx.sync()
    got = [ctx.download(o, (groups, picks), t) for o, t in zip(outs, (np.float32, np.int32, np.int32))]
    for g in range(groups):
        check([a[g:g + 1] for a in got] + [None], logits, vocab, score, None, -1, picks, "without numbers")
    assert set(got[2][0][got[2][0] >= 0]) <= {5, 6, 7}
    for b in (lb, sb, *outs):
        ctx.free(b)
