"""Writes to the caches of one to 1500 sequences, most of them with few new rows or none, and rows before the first and behind the last one."""
import numpy as np
import pytest

import kv_reference as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt,heads,D", [("fp16", 2, 64), ("int8", 2, 64), ("fp8", 8, 128)])
@pytest.mark.parametrize("seqs", [1, 31, 32, 33, 64, 65, 96, 128, 129, 1500])
def test_rows_find_their_sequences(nnb, ctx, fmt, heads, D, seqs):
    rng = np.random.default_rng(121 + seqs)
    lengths = rng.integers(3, 40, seqs)
    new = np.where(rng.random(seqs) < 0.5, 0, rng.integers(1, 4, seqs))
    new[rng.integers(0, seqs)] = 3
    if seqs > 100:
        new[5:80] = 0          # a whole stretch of them
    cache = ref.Cache(nnb, ctx, fmt, list(lengths), heads, D, 16, seed=122)
    before, behind = 2, 3
    start = before + np.concatenate([[0], np.cumsum(new)])
    rows = int(start[-1]) + behind
    b = cache.batch(list(new), extra_rows=behind, row_start=start)
    k, v = (rng.standard_normal((rows, heads, D)).astype(np.float16) for _ in range(2))
    kb, vb = ctx.upload(k.view(np.uint16)), ctx.upload(v.view(np.uint16))
    ctx.kv_write(cache.handle, b, kb, 0, vb, 0)
    ctx.sync()
    for name, x in (("k", k), ("v", v)):
        codes, scale = (x.view(np.uint16), None) if fmt == "fp16" else ref.quantised(x, fmt)
        for i in range(seqs):
            for j in range(new[i]):
                p = lengths[i] - new[i] + j
                cache.host[name][cache.table[i, p // 16], :, p % 16] = codes[start[i] + j]
                if scale is not None:
                    cache.host[name + "_scale"][cache.table[i, p // 16], :, p % 16] = scale[start[i] + j]
    got = cache.read_back()
    for name, a in got.items():
        assert np.array_equal(a.view(np.uint8), np.ascontiguousarray(cache.host[name]).view(np.uint8)), (fmt, seqs, name)
    # the same rows at positions of their own: all keys turned by one angle, as if each sequence had the position 1
    cos, sin = (np.ascontiguousarray(f(np.arange(2)[:, None] * np.linspace(0.1, 1, D // 2)), np.float32) for f in (np.cos, np.sin))
    up = [ctx.upload(a) for a in (np.ones(rows, np.int32), cos, sin)]
    ctx.rope_kv_write_at(cache.handle, b, up[0], up[1], up[2], 2, D, 0, None, 0, None, 0, kb, 0, vb, 0)
    ctx.sync()
    turned = ref.rotated(k, cos[np.ones(rows, int)], sin[np.ones(rows, int)], D)
    codes, scale = (turned.view(np.uint16), None) if fmt == "fp16" else ref.quantised(turned, fmt)
    for i in range(seqs):
        for j in range(new[i]):
            p = lengths[i] - new[i] + j
            cache.host["k"][cache.table[i, p // 16], :, p % 16] = codes[start[i] + j]
            if scale is not None:
                cache.host["k_scale"][cache.table[i, p // 16], :, p % 16] = scale[start[i] + j]
    got = cache.read_back()
    for name, a in got.items():
        assert np.array_equal(a.view(np.uint8), np.ascontiguousarray(cache.host[name]).view(np.uint8)), (fmt, seqs, name, "turned")
    cache.close()
    for x in (kb, vb, *up):
        ctx.free(x)
