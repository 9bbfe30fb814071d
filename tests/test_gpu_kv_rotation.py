"""Rotated writes, bit for bit: up to 128 dims, keys without queries, queries to another buffer, many rows, positions behind the tables."""
import numpy as np
import pytest

import kv_reference as ref
from helpers import alloc_with_canary, check_canary
from test_gpu_kv_cache import _positions, _stored, _values

pytestmark = pytest.mark.gpu


def _tables(length, rotary):
    angle = np.arange(length)[:, None] * 10000.0 ** (-2.0 * np.arange(rotary // 2) / rotary)
    return np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)


def _check_cells(c):
    got = c.read_back()
    for name in got:
        want = c.host[name]
        if name.endswith("scale"):
            have = got[name].view(np.float16)
            assert np.array_equal(have, want, equal_nan=True), name
        else:
            assert np.array_equal(got[name], want), name


# rows to a warp each need more than 592 of them (2368 where a row is wide)
@pytest.mark.parametrize("seqs", [[(1, 300)], [(40, 60), (0, 5), (3, 3), (1, 129)], [(900, 900), (1700, 1800)]])
@pytest.mark.parametrize("fmt,D,rotary,hq,hk", [("fp16", 128, 128, 8, 2), ("int8", 128, 128, 32, 8), ("fp8", 128, 128, 4, 4), ("int8", 128, 96, 2, 1), ("fp8", 128, 112, 7, 7),
                                                ("fp16", 64, 48, 3, 3), ("int8", 64, 16, 9, 3), ("fp8", 64, 64, 14, 2)])
def test_rotation(nnb, ctx, fmt, D, rotary, hq, hk, seqs):
    page, rng = 32, np.random.default_rng(71)
    c = ref.Cache(nnb, ctx, fmt, [n for _, n in seqs], hk, D, page, seed=72)
    rows, pos = sum(n for n, _ in seqs), _positions(seqs)
    q, k, v = (_values(rng, rows, h, D) for h in (hq, hk, hk))
    cos, sin = _tables(max(n for _, n in seqs), rotary)
    up = [ctx.upload(a) for a in (cos, sin, q, k, v)]
    out = alloc_with_canary(ctx, q.nbytes)
    b = c.batch([n for n, _ in seqs])
    ctx.rope_kv_write(c.handle, b, up[0], up[1], len(cos), rotary, hq, up[2], 0, out, 0, up[3], 0, up[4], 0)
    ctx.sync()
    turned_q, turned_k = (ref.rotated(t, cos[pos], sin[pos], rotary) for t in (q, k))
    assert np.array_equal(ctx.download(out, q.shape, np.uint16), turned_q.view(np.uint16))
    assert np.array_equal(ctx.download(up[2], q.shape, np.uint16), q.view(np.uint16))        # (the operands stay)
    check_canary(ctx, out, q.nbytes)
    _stored(c, seqs, turned_k, v)
    _check_cells(c)
    # keys alone give the same cells
    for name in "kv":
        ctx.upload(np.zeros_like(c.host[name]), c.dev[name])
    ctx.rope_kv_write(c.handle, b, up[0], up[1], len(cos), rotary, 0, None, 0, None, 0, up[3], 0, up[4], 0)
    ctx.sync()
    fresh = {n: np.zeros_like(c.host[n]) for n in "kv"}
    for i, (new, n) in enumerate(seqs):
        for p in range(n - new, n):
            at = c.table[i, p // page], slice(None), p % page
            for name in "kv":
                fresh[name][at] = c.host[name][at]
    c.host.update(fresh)
    _check_cells(c)
    c.close()
    for t in (*up, out):
        ctx.free(t)


@pytest.mark.parametrize("fmt,D", [("fp16", 64), ("int8", 128)])
@pytest.mark.parametrize("rows", [6, 3000])
def test_positions_behind_the_tables(nnb, ctx, fmt, D, rows):
    """They are reported, neither their queries nor their cells are written; the rows in front of them are."""
    hq, hk, page, length, inside = 2, 1, 16, rows + 10, 10 + rows // 2
    c = ref.Cache(nnb, ctx, fmt, [length], hk, D, page, seed=73)
    rng = np.random.default_rng(74)
    q, k, v = (rng.standard_normal((rows, h, D)).astype(np.float16) for h in (hq, hk, hk))
    cos, sin = _tables(inside, D)
    up = [ctx.upload(a) for a in (cos, sin, q, k, v)]
    out = alloc_with_canary(ctx, q.nbytes)
    ctx.rope_kv_write(c.handle, c.batch([rows]), up[0], up[1], inside, D, hq, up[2], 0, out, 0, up[3], 0, up[4], 0)
    with pytest.raises(nnb.NNError) as e:
        ctx.sync()
    assert e.value.code == nnb.NN_ERR_ARG
    good = rows // 2                                       # rows with positions 10 .. inside - 1
    got = ctx.download(out, q.shape, np.uint16)
    pos = np.arange(10, inside)
    assert np.array_equal(got[:good], ref.rotated(q[:good], cos[pos], sin[pos], D).view(np.uint16)) and (got[good:] == 0x7E7E).all()
    check_canary(ctx, out, q.nbytes)
    _stored(c, [(good, inside)], ref.rotated(k[:good], cos[pos], sin[pos], D), v[:good])
    _check_cells(c)
    c.close()
    for t in (*up, out):
        ctx.free(t)
