"""Attention of new tokens over the paged key/value cache against the formula in 64 bits."""
import numpy as np
import pytest

import kv_reference as ref
from helpers import alloc_with_canary, check_canary, report

pytestmark = pytest.mark.gpu

HEADS = {"mha": (3, 3), "gqa3": (9, 3), "gqa7": (14, 2), "mqa": (8, 1), "mqa40": (40, 1)}
# (new rows, length) of each sequence
BATCHES = {
    "one": [(1, 1)],
    "tokens": [(1, 700), (1, 1), (1, 16), (1, 129), (1, 64)],
    "drafts": [(5, 300), (3, 3), (0, 77), (5, 65), (1, 513)],
    "chunks": [(130, 130), (40, 700), (257, 300), (0, 0), (17, 1000)],
    "prompt": [(400, 400)],
    "negative": [(5, 3), (2, 0), (1, 20)],     # rows with positions below 0 see nothing
}


def run_attention(nnb, ctx, c, q, new, lengths=None, scale=None, window=0, sinks=0, extra=0, **bounds):
    """out [rows + extra, heads, D] as fp16 bits; rows behind the last sequence keep what they held."""
    rows, hq, D = q.shape
    n = (rows + extra) * hq * D * 2
    qb, out = ctx.upload(np.concatenate([q, np.zeros((extra, hq, D), np.float16)])), alloc_with_canary(ctx, n)
    ctx.attention(c.handle, c.batch(new, lengths, extra_rows=extra, **bounds), hq, qb, 0, out, 0, scale or D ** -0.5, window, sinks)
    got = ctx.download(out, (rows + extra, hq, D), np.float16)
    check_canary(ctx, out, n)
    for b in (qb, out):
        ctx.free(b)
    return got


def check_attention(c, got, q, seqs, scale, window, sinks, what=""):
    hq, D = q.shape[1:]
    group, row, worst = hq // c.kv_heads, 0, 0.0
    for i, (new, length) in enumerate(seqs):
        k, v = c.sequence("k", i, length), c.sequence("v", i, length)
        pos = np.arange(length - new, length)
        for h in range(hq):
            want, spread, most, steep = ref.attend(q[row:row + new, h].astype(np.float64), k[:, h // group], v[:, h // group], pos, scale, window, sinks)
            bound = ref.attention_bound(want, spread, most, steep, length, D)
            have = got[row:row + new, h].astype(np.float64)
            assert np.array_equal(np.isfinite(have), np.isfinite(want)), (what, i, h, np.argwhere(np.isfinite(have) != np.isfinite(want))[:4])
            fine = np.isfinite(want)
            off = np.abs(have - want)[fine] / bound[fine]
            if off.size:
                worst = max(worst, off.max())
                assert off.max() <= 1, (what, i, h, off.max(), np.argwhere(np.where(fine, np.abs(have - want), 0) > np.where(fine, bound, 1))[:4])
        row += new
    report(f"attention {what}: worst error {worst:.2f} of its bound")


@pytest.mark.parametrize("window,sinks", [(0, 0), (48, 0), (48, 4), (1, 0), (200, 70)])
@pytest.mark.parametrize("batch", BATCHES)
@pytest.mark.parametrize("fmt,D,page,heads", [("fp16", 64, 16, "gqa3"), ("int8", 64, 64, "gqa7"), ("fp8", 64, 256, "mha"), ("fp16", 128, 128, "mqa"),
                                              ("int8", 128, 32, "mqa40"), ("fp8", 128, 16, "gqa3"), ("fp16", 64, 64, "mqa40"), ("fp8", 64, 32, "mqa")])
def test_attention(nnb, ctx, fmt, D, page, heads, batch, window, sinks):
    seqs = BATCHES[batch]
    hq, hk = HEADS[heads]
    c = ref.Cache(nnb, ctx, fmt, [n for _, n in seqs], hk, D, page, seed=11)
    q = np.random.default_rng(12).standard_normal((sum(n for n, _ in seqs), hq, D)).astype(np.float16)
    new = [n for n, _ in seqs]
    got = run_attention(nnb, ctx, c, q, new, window=window, sinks=sinks, extra=3)
    ctx.sync()
    assert (got[len(q):].view(np.uint16) == 0x7E7E).all()          # rows behind the last sequence
    check_attention(c, got, q, seqs, D ** -0.5, window, sinks, f"{fmt} D{D} {heads} {batch} window {window}")
    again = run_attention(nnb, ctx, c, q, new, window=window, sinks=sinks, extra=3)
    assert np.array_equal(got.view(np.uint16), again.view(np.uint16))
    c.close()
