"""The paged key/value cache: rotated and quantised writes and the read back, bit for bit."""
import numpy as np
import pytest

import kv_reference as ref
from helpers import alloc_with_canary, check_canary

pytestmark = pytest.mark.gpu

# (new rows, length) of the sequences: one token, a prompt from its start, none at all, chunks that end inside and at the end of pages
BATCHES = {
    "one": [(1, 1)],
    "token": [(1, 700)],
    "ragged": [(3, 40), (0, 9), (17, 17), (1, 64), (33, 129), (0, 0), (5, 48)],
    "many": [(1 + i % 3, 20 + 7 * i) for i in range(150)],
}


def _values(rng, rows, heads, D):
    """Rows of all magnitudes, with zeros, the largest and the smallest values."""
    x = (rng.standard_normal((rows, heads, D)) * np.exp2(rng.integers(-20, 12, (rows, heads, 1)))).astype(np.float16)
    flat = x.reshape(-1, D)
    flat[0] = 0
    if len(flat) > 3:
        flat[1, 5], flat[2] = 65504.0, 2.0 ** -24
        flat[3, ::2] = -65504.0
    return x


def _write(ctx, c, batch, x, rope):
    up = {n: ctx.upload(np.ascontiguousarray(a)) for n, a in x.items()}
    if rope:
        ctx.rope_kv_write(c.handle, batch, up["cos"], up["sin"], len(x["cos"]), rope, x["q"].shape[1], up["q"], 0, up["q"], 0, up["k"], 0, up["v"], 0)
    else:
        ctx.kv_write(c.handle, batch, up["k"], 0, up["v"], 0)
    q = ctx.download(up["q"], x["q"].shape, np.float16)
    for b in up.values():
        ctx.free(b)
    return q


def _positions(batch):
    return np.concatenate([np.arange(n - new, n) for new, n in batch]).astype(int)


def _stored(c, batch, k, v):
    """The host's copy with the new rows in it."""
    row = 0
    for name, x in (("k", k), ("v", v)):
        codes, scale = (x.view(np.uint16), None) if c.fmt == "fp16" else ref.quantised(x, c.fmt)
        row = 0
        for i, (new, n) in enumerate(batch):
            for p in range(n - new, n):
                at = c.table[i, p // c.page], slice(None), p % c.page
                c.host[name][at] = codes[row]
                if scale is not None:
                    c.host[name + "_scale"][at] = scale[row]
                row += 1


@pytest.mark.parametrize("rope", [0, 32, 64])
@pytest.mark.parametrize("batch", BATCHES)
@pytest.mark.parametrize("fmt,D,page,heads", [("fp16", 64, 16, (9, 3)), ("int8", 64, 32, (14, 2)), ("fp8", 64, 256, (4, 4)), ("fp16", 128, 64, (8, 1)),
                                              ("int8", 128, 16, (7, 7)), ("fp8", 128, 128, (32, 8))])
def test_write_and_read_back(nnb, ctx, fmt, D, page, heads, batch, rope):
    seqs = BATCHES[batch]
    c = ref.Cache(nnb, ctx, fmt, [n for _, n in seqs], heads[1], D, page, seed=3)
    rng = np.random.default_rng(5)
    rows = sum(n for n, _ in seqs)
    x = {"q": _values(rng, rows, heads[0], D), "k": _values(rng, rows, heads[1], D), "v": _values(rng, rows, heads[1], D)}
    pos = _positions(seqs)
    k, q = x["k"], x["q"]
    if rope:
        angle = np.arange(max(n for _, n in seqs))[:, None] * 10000.0 ** (-2.0 * np.arange(rope // 2) / rope)
        x["cos"], x["sin"] = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
        k, q = (ref.rotated(t, x["cos"][pos], x["sin"][pos], rope) for t in (k, q))
    b = c.batch([n for n, _ in seqs])
    got_q = _write(ctx, c, b, x, rope)
    assert np.array_equal(got_q.view(np.uint16), q.view(np.uint16))
    _stored(c, seqs, k, x["v"])
    got = c.read_back()
    for name in "kv":
        if fmt != "fp16":
            want = c.host[name + "_scale"]
            have = got[name + "_scale"].view(np.float16)
            assert np.array_equal(np.isnan(have), np.isnan(want)) and np.array_equal(have[~np.isnan(want)], want[~np.isnan(want)]), name
        assert np.array_equal(got[name], c.host[name]), name          # (every cell: those that are not written too)
    # the read back of the same rows, and of every position
    for new in ([n for n, _ in seqs], [n for _, n in seqs]):
        total = sum(new)
        n = total * heads[1] * D * 2
        ko, vo = alloc_with_canary(ctx, n), alloc_with_canary(ctx, n)
        ctx.kv_read(c.handle, c.batch(new), ko, 0, vo, 0)
        for name, buf in (("k", ko), ("v", vo)):
            have = ctx.download(buf, (total, heads[1], D), np.float16)
            want = np.concatenate([c.sequence(name, i, length)[length - m:] for i, (m, (_, length)) in enumerate(zip(new, seqs))])
            assert np.array_equal(have, want.astype(np.float16), equal_nan=True), name
            check_canary(ctx, buf, n)
            ctx.free(buf)
    c.close()


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_rows_with_infinities_or_nans_read_back_as_nan(nnb, ctx, fmt):
    D, H = 64, 2
    c = ref.Cache(nnb, ctx, fmt, [20], H, D, 16, seed=1)
    rng = np.random.default_rng(2)
    x = {"q": np.zeros((4, 2, D), np.float16), "k": rng.standard_normal((4, H, D)).astype(np.float16), "v": rng.standard_normal((4, H, D)).astype(np.float16)}
    x["k"][0, 1, 63], x["k"][2, 0, 7], x["v"][3, 1, 0] = np.inf, np.nan, -np.inf
    b = c.batch([4])
    _write(ctx, c, b, x, 0)
    ko, vo = ctx.alloc(4 * H * D * 2), ctx.alloc(4 * H * D * 2)
    ctx.kv_read(c.handle, b, ko, 0, vo, 0)
    k, v = (ctx.download(t, (4, H, D), np.float16) for t in (ko, vo))
    bad_k, bad_v = np.zeros((4, H), bool), np.zeros((4, H), bool)
    bad_k[0, 1] = bad_k[2, 0] = bad_v[3, 1] = True
    for got, bad in ((k, bad_k), (v, bad_v)):
        assert np.isnan(got[bad]).all() and np.isfinite(got[~bad]).all()
    for t in (ko, vo):
        ctx.free(t)
    c.close()


@pytest.mark.parametrize("fmt", ["fp16", "int8"])
def test_columns_of_one_buffer_and_rows_behind_the_last_sequence(nnb, ctx, fmt):
    """q, k and v as columns of a fused projection's output, rotated in place; rows that belong to no sequence stay as they are."""
    D, hq, hk, seqs, spare = 64, 6, 2, [(3, 50), (4, 4)], 5
    c = ref.Cache(nnb, ctx, fmt, [n for _, n in seqs], hk, D, 16, seed=4)
    rng = np.random.default_rng(6)
    width = (hq + 2 * hk) * D
    pitch = width + 24
    x = rng.standard_normal((7 + spare, pitch)).astype(np.float16)
    pos = _positions(seqs)
    angle = np.arange(50)[:, None] * 10000.0 ** (-np.arange(0, D, 2) / D)
    cos, sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
    buf, cb, sb = ctx.upload(x), ctx.upload(cos), ctx.upload(sin)
    b = c.batch([n for n, _ in seqs], extra_rows=spare)
    ctx.rope_kv_write(c.handle, b, cb, sb, 50, D, hq, buf, pitch, buf, pitch, buf + hq * D * 2, pitch, buf + (hq + hk) * D * 2, pitch)
    got = ctx.download(buf, x.shape, np.float16)
    want = x.copy()
    want[:7, : hq * D] = ref.rotated(x[:7, : hq * D].reshape(7, hq, D), cos[pos], sin[pos], D).reshape(7, -1)
    assert np.array_equal(got, want)
    k = ref.rotated(x[:7, hq * D:(hq + hk) * D].reshape(7, hk, D), cos[pos], sin[pos], D)
    _stored(c, seqs, k, np.ascontiguousarray(x[:7, (hq + hk) * D:width].reshape(7, hk, D)))
    have = c.read_back()
    for name in "kv":
        assert np.array_equal(have[name], c.host[name])
    out = ctx.upload(x)                                   # the read back into columns
    ctx.kv_read(c.handle, b, out + 8 * 2, pitch, out + (8 + hk * D) * 2, pitch)
    got = ctx.download(out, x.shape, np.float16)
    want = x.copy()
    for name, at in (("k", 8), ("v", 8 + hk * D)):
        want[:7, at:at + hk * D] = np.concatenate([c.sequence(name, i, n)[n - m:] for i, (m, n) in enumerate(seqs)]).astype(np.float16).reshape(7, -1)
    assert np.array_equal(got, want)
    for t in (buf, cb, sb, out):
        ctx.free(t)
    c.close()


@pytest.mark.parametrize("fmt", ["fp16", "fp8"])
def test_pages_and_lengths_out_of_range(nnb, ctx, fmt):
    """Bad page numbers, lengths and positions: reported by the next sync, their rows left out, everything else done."""
    D, H = 64, 1
    c = ref.Cache(nnb, ctx, fmt, [40, 40], H, D, 16, seed=8, fill=False)
    rng = np.random.default_rng(9)
    x = {"q": np.zeros((4, 1, D), np.float16), "k": rng.standard_normal((4, H, D)).astype(np.float16), "v": rng.standard_normal((4, H, D)).astype(np.float16)}
    ko, vo = ctx.alloc(4 * H * D * 2), ctx.alloc(4 * H * D * 2)

    def expect(batch, good, seqs, table):
        with pytest.raises(nnb.NNError) as e:
            _write(ctx, c, batch, x, 0)
        assert e.value.code == nnb.NN_ERR_ARG and "out of range" in str(e.value)
        keep = c.table
        c.table = table
        row = 0
        for i, (m, n) in enumerate(seqs):
            for p in range(n - m, n):
                if good[row]:
                    for name in "kv":
                        codes, scale = (x[name].view(np.uint16), None) if fmt == "fp16" else ref.quantised(x[name], fmt)
                        c.host[name][table[i, p // 16], :, p % 16] = codes[row]
                        if scale is not None:
                            c.host[name + "_scale"][table[i, p // 16], :, p % 16] = scale[row]
                row += 1
        have = c.read_back()
        for name in "kv":
            assert np.array_equal(have[name], c.host[name])
        ctx.kv_read(c.handle, batch, ko, 0, vo, 0)
        with pytest.raises(nnb.NNError):
            ctx.sync()
        got = ctx.download(ko, (4, H, D), np.float16)
        assert not got[~np.asarray(good)].any() and got[np.asarray(good)].any(axis=(1, 2)).all()
        c.table = keep

    for bad in (-1, c.pages, 1 << 30, -(1 << 31)):
        table = c.table.copy()
        table[1, 2] = bad                                           # positions 32..47 of the second sequence
        expect(c.batch([1, 3], [40, 34], table=table), [True, True, False, False], [(1, 40), (3, 34)], table)
    expect(c.batch([2, 2], [40, 1]), [True, True, False, True], [(2, 40), (2, 1)], c.table)      # position -1
    big = c.batch([2, 2], [40, 41], max_len=40)                     # longer than max_len
    expect(big, [True, True, False, False], [(2, 40), (2, 40)], c.table)
    ctx.kv_write(c.handle, c.batch([0, 0]), ko, 0, vo, 0)           # and the context stays usable
    ctx.sync()
    for t in (ko, vo):
        ctx.free(t)
    c.close()


def test_cells_beyond_two_to_the_32_bytes(nnb, ctx):
    """Page numbers whose cells lie more than 4 GiB into a buffer."""
    D, H, page = 128, 8, 256
    pages = (5 << 30) // (page * H * D * 2)
    k, v = ctx.alloc(5 << 30), ctx.alloc(5 << 30)
    cache = ctx.kv_cache("fp16", pages, page, H, D, k, v)
    rng = np.random.default_rng(3)
    x = rng.standard_normal((2, H, D)).astype(np.float16)
    up = [ctx.upload(a) for a in (np.array([0, 2], np.int32), np.array([258], np.int32), np.array([[0, pages - 1]], np.int32), x, x)]
    b = nnb.KVBatch(1, 2, 2, 512, 2, *up[:3])
    ctx.kv_write(cache, b, up[3], 0, up[4], 0)
    at = (pages - 1) * page * H * D * 2
    for buf in (k, v):
        got = ctx.download(buf, (H, page, D), np.float16, offset=at)
        assert np.array_equal(got[:, :2].transpose(1, 0, 2), x)
    ko, vo = ctx.alloc(x.nbytes), ctx.alloc(x.nbytes)
    ctx.kv_read(cache, b, ko, 0, vo, 0)
    assert np.array_equal(ctx.download(ko, x.shape, np.float16), x) and np.array_equal(ctx.download(vo, x.shape, np.float16), x)
    cache.close()
    for t in (*up, k, v, ko, vo):
        ctx.free(t)
