"""Writes of many rows of many heads, at the row counts where one kernel takes over from the other: queries, cells and scales bit by bit."""
import numpy as np
import pytest

import kv_reference as ref
from helpers import alloc_with_canary, check_canary

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["fp16", "int8", "fp8"])
@pytest.mark.parametrize("q_heads,heads,D,rotary,rows", [(*shape, rows) for shape in ((16, 8, 128, 128), (48, 8, 64, 32)) for rows in (2368, 2369, 2960, 2961, 4736, 4737)]
                         + [(2, 1, 64, 64, 592), (2, 1, 64, 64, 593)])
def test_row_counts(nnb, ctx, fmt, q_heads, heads, D, rotary, rows):
    rng = np.random.default_rng(161 + rows)
    P, before, behind = 256, 3, 2
    n, pages = rows - before - behind, -(-rows // P)
    q, k, v = (rng.standard_normal((rows, h, D)).astype(np.float16) for h in (q_heads, heads, heads))
    for x in (q, k, v):
        x[:before], x[rows - behind:] = 7, 7
    k[before, 0], v[before + 1, heads - 1, 5], k[rows - behind - 1, heads - 1, 3] = 0, np.inf, 65504
    angle = np.arange(pages * P)[:, None] * np.linspace(0.01, 1, rotary // 2)
    cos, sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
    table, cell = rng.permutation(pages).astype(np.int32), np.float16 if fmt == "fp16" else np.uint8
    size = pages * heads * P * D
    cells = [alloc_with_canary(ctx, size * np.dtype(cell).itemsize) for _ in range(2)]
    scales = [alloc_with_canary(ctx, size // D * 2) for _ in range(2)] if fmt != "fp16" else [None, None]
    c = ctx.kv_cache(fmt, pages, P, heads, D, *cells, *scales)
    up = [ctx.upload(np.ascontiguousarray(x)) for x in (q.view(np.uint16), k.view(np.uint16), v.view(np.uint16), cos, sin, np.array([before, before + n], np.int32), np.array([n], np.int32), table)]
    out = alloc_with_canary(ctx, q.nbytes)
    b = nnb.KVBatch(1, rows, n, pages * P, pages, *up[5:])
    ctx.rope_kv_write(c, b, up[3], up[4], pages * P, rotary, q_heads, up[0], 0, out, 0, up[1], 0, up[2], 0)
    ctx.sync()
    mine, where = slice(before, before + n), np.arange(n)
    turned_q, turned_k = (ref.rotated(x[mine], cos[where], sin[where], rotary) for x in (q, k))
    got = ctx.download(out, q.shape, np.uint16)
    assert np.array_equal(got[mine], turned_q.view(np.uint16))
    assert (got[:before] == 0x7E7E).all() and (got[before + n:] == 0x7E7E).all()      # as they were
    for x, cb, sb in ((turned_k, cells[0], scales[0]), (v[mine], cells[1], scales[1])):
        have = ctx.download(cb, (pages, heads, P, D), cell)[table[where // P], :, where % P]
        if fmt == "fp16":
            assert np.array_equal(have.view(np.uint16), x.view(np.uint16))
            continue
        codes, scale = ref.quantised(x, fmt)
        have_scale = ctx.download(sb, (pages, heads, P), np.uint16)[table[where // P], :, where % P]
        assert np.array_equal(have_scale.view(np.float16), scale, equal_nan=True) and np.array_equal(have, np.ascontiguousarray(codes).view(np.uint8))
    check_canary(ctx, out, q.nbytes)
    for cb, sb in zip(cells, scales):
        check_canary(ctx, cb, size * np.dtype(cell).itemsize)
        if sb:
            check_canary(ctx, sb, size // D * 2)
    c.close()
    for x in (*up, out, *cells, *[s for s in scales if s]):
        ctx.free(x)
