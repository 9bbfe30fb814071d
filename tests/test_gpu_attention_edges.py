"""Attention over the paged cache where it can go wrong: cells that are not finite, bad tables, shared pages, columns, very long, very many."""
import threading

import numpy as np
import pytest

import kv_reference as ref
from test_gpu_attention import check_attention, run_attention

pytestmark = pytest.mark.gpu

# one token, drafts and chunks: each takes a way of its own through the kernels
SHAPES = {"token": [(1, 150), (1, 90)], "drafts": [(5, 150), (3, 90)], "chunk": [(150, 150), (40, 90)], "long chunk": [(140, 900), (260, 300)]}


def _queries(seqs, hq, D, seed=12):
    return np.random.default_rng(seed).standard_normal((sum(n for n, _ in seqs), hq, D)).astype(np.float16)


def _poke(c, name, seq, pos, head, dim, value):
    """A value into a cell of the cache: into its row's scale where the cells are codes."""
    page, slot = c.table[seq, pos // c.page], pos % c.page
    if c.fmt == "fp16":
        c.host[name].view(np.float16)[page, head, slot, dim] = value
    else:
        c.host[name + "_scale"][page, head, slot] = value


def _upload(c):
    for name in "kv":
        c.ctx.upload(c.host[name], c.dev[name])
        if c.fmt != "fp16":
            c.ctx.upload(c.host[name + "_scale"].view(np.uint16), c.dev[name + "_scale"])


@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 2)])
@pytest.mark.parametrize("shape", list(SHAPES))
@pytest.mark.parametrize("fmt,D", [("fp16", 64), ("fp16", 128), ("int8", 64), ("int8", 128), ("fp8", 64), ("fp8", 128)])
def test_cells_that_are_not_finite(nnb, ctx, fmt, D, shape, window, sinks):
    """Infinities and NaNs in keys and values: rows that see them give what the formula gives, the others are not touched by them."""
    seqs, hq, hk = SHAPES[shape], 4, 2
    c = ref.Cache(nnb, ctx, fmt, [n for _, n in seqs], hk, D, 16, seed=21)
    for i, (_, n) in enumerate(seqs):
        for name, pos, head, dim, value in (("v", n - 2, 0, 5, np.nan), ("k", n - 4, 1, 9, np.inf), ("v", 20, 1, D - 1, -np.inf), ("k", n // 2, 0, 0, np.nan)):
            _poke(c, name, i, pos, head, dim, value)
    _upload(c)
    q = _queries(seqs, hq, D)
    got = run_attention(nnb, ctx, c, q, [n for n, _ in seqs], window=window, sinks=sinks)
    ctx.sync()
    check_attention(c, got, q, seqs, D ** -0.5, window, sinks, f"not finite {fmt} D{D} {shape} window {window}")
    c.close()


@pytest.mark.parametrize("fmt", ["fp16", "int8"])
@pytest.mark.parametrize("new", [1, 140])
def test_long_rows_of_nans(nnb, ctx, fmt, new):
    """Every row of a long sequence sees an infinite value: computed once more from the formula, without a wait that takes it for a standstill."""
    seqs, D = [(new, 20000)], 64
    c = ref.Cache(nnb, ctx, fmt, [20000], 1, D, 256, seed=22)
    _poke(c, "v", 0, 19999 - new, 0, 3, np.inf if fmt == "fp16" else np.nan)
    _upload(c)
    q = _queries(seqs, 4, D)
    got = run_attention(nnb, ctx, c, q, [new])
    ctx.sync()
    if fmt == "fp16":       # (dims without the infinity are as exact as ever)
        assert (got[..., 3] == np.inf).all()
        c.host["v"].view(np.float16)[c.table[0, (19999 - new) // 256], 0, (19999 - new) % 256, 3] = 0
        got[..., 3] = 0
        k, v = c.sequence("k", 0, 20000), c.sequence("v", 0, 20000)
        for i in (0, new - 1):
            want, spread, most, steep = ref.attend(q[i].astype(np.float64), k[:, 0], v[:, 0], [20000 - new + i] * 4, D ** -0.5, 0, 0)
            want[:, 3] = 0
            assert (np.abs(got[i] - want) <= ref.attention_bound(want, spread, most, steep, 20000, D)).all()
    else:
        assert np.isnan(got).all()
    c.close()


@pytest.mark.parametrize("fmt,D", [("fp16", 64), ("int8", 128)])
@pytest.mark.parametrize("shape", ["token", "drafts", "long chunk"])
def test_bad_pages_are_reported_and_hidden(nnb, ctx, fmt, D, shape):
    seqs, hq, hk, page = SHAPES[shape], 4, 2, 32
    c = ref.Cache(nnb, ctx, fmt, [n for _, n in seqs], hk, D, page, seed=23)
    q = _queries(seqs, hq, D)
    new = [n for n, _ in seqs]
    for bad in (-1, c.pages, 1 << 30, -(1 << 31)):
        table = c.table.copy()
        table[0, 1] = bad                          # positions 32 .. 63 of the first sequence
        with pytest.raises(nnb.NNError) as e:
            run_attention(nnb, ctx, c, q, new, table=table)
        assert e.value.code == nnb.NN_ERR_ARG and "out of range" in str(e.value)
    # their keys count as hidden: the same result as with cells there whose scores are far below the others'
    out = ctx.alloc(q.nbytes)
    qb = ctx.upload(q)
    ctx.attention(c.handle, c.batch(new, table=table), hq, qb, 0, out, 0, D ** -0.5)
    with pytest.raises(nnb.NNError):
        ctx.sync()
    got = ctx.download(out, q.shape, np.float16)
    row = 0
    for i, (n, length) in enumerate(seqs):
        k, v = c.sequence("k", i, length), c.sequence("v", i, length)
        for t in range(n):
            p = length - n + t
            keep = np.array([x for x in range(p + 1) if i or not 32 <= x < 64])
            for h in range(hq):
                want, spread, most, steep = ref.attend(q[row + t:row + t + 1, h].astype(np.float64), k[keep, h // 2], v[keep, h // 2], [length], D ** -0.5, 0, 0)
                assert (np.abs(got[row + t, h] - want) <= ref.attention_bound(want, spread, most, steep, length, D)).all()
        row += n
    got = run_attention(nnb, ctx, c, q, new)         # and the context stays usable
    ctx.sync()
    check_attention(c, got, q, seqs, D ** -0.5, 0, 0)
    for b in (out, qb):
        ctx.free(b)
    c.close()


@pytest.mark.parametrize("max_new", [1, 200])
def test_row_starts_that_do_not_ascend(nnb, ctx, max_new):
    """Reported, nothing is computed and nothing beyond the operands is touched; lengths out of range spoil their own sequence alone."""
    seqs, hq, hk, D = [(40, 300), (40, 200), (40, 120), (40, 64)], 2, 1, 64
    c = ref.Cache(nnb, ctx, "fp16", [n for _, n in seqs], hk, D, 64, seed=24)
    q = _queries(seqs, hq, D)
    for starts in ([0, 160, 0, 160, 160], [0, 160, 80, 40, 160], [160, 0, 160, 0, 160]):
        with pytest.raises(nnb.NNError) as e:
            run_attention(nnb, ctx, c, q, None, row_start=starts, max_new=max_new)
        assert e.value.code == nnb.NN_ERR_ARG
    for lengths in ([300, 200, 120, 1 << 30], [300, 200, 120, -5]):
        qb, out = ctx.upload(q), ctx.alloc(q.nbytes)
        ctx.attention(c.handle, c.batch([40] * 4, lengths, max_new=max_new, max_len=300), hq, qb, 0, out, 0, D ** -0.5)
        with pytest.raises(nnb.NNError):
            ctx.sync()
        check_attention(c, ctx.download(out, q.shape, np.float16), q, seqs[:3], D ** -0.5, 0, 0)
        for b in (qb, out):
            ctx.free(b)
    c.close()


@pytest.mark.parametrize("shape", list(SHAPES))
def test_shared_pages_columns_and_rows_before_the_first(nnb, ctx, shape):
    """A common prefix in the same pages, q and out as columns of wider buffers, rows before row_start[0]."""
    seqs, hq, hk, D, page, before = SHAPES[shape], 6, 2, 64, 16, 3
    c = ref.Cache(nnb, ctx, "int8", [n for _, n in seqs], hk, D, page, seed=25)
    c.table[1, :2] = c.table[0, :2]
    c.table[1, 3] = c.table[1, 2]                   # the same page twice in a sequence
    rows, pitch, opitch = sum(n for n, _ in seqs) + before, (hq + 2 * hk) * D + 8, hq * D + 16
    x = np.random.default_rng(3).standard_normal((rows, pitch)).astype(np.float16)
    ob = np.full((rows, opitch), 0x7E7E, np.uint16)
    qb, out = ctx.upload(x), ctx.upload(ob)
    starts = before + np.concatenate([[0], np.cumsum([n for n, _ in seqs])])
    ctx.attention(c.handle, c.batch([n for n, _ in seqs], row_start=starts), hq, qb, pitch, out + 16, opitch, D ** -0.5)
    got = ctx.download(out, ob.shape, np.uint16)
    rest = got.copy()
    rest[before:, 8:8 + hq * D] = 0x7E7E
    assert (rest == 0x7E7E).all()
    check_attention(c, np.ascontiguousarray(got[before:, 8:8 + hq * D]).view(np.float16).reshape(-1, hq, D), x[before:, :hq * D].reshape(-1, hq, D), seqs, D ** -0.5, 0, 0,
                    f"columns {shape}")
    for b in (qb, out):
        ctx.free(b)
    c.close()


@pytest.mark.parametrize("fmt,D,hq,hk", [("fp16", 64, 12, 4), ("int8", 128, 8, 1), ("fp8", 64, 24, 1), ("fp8", 128, 2, 2), ("int8", 64, 20, 1), ("fp16", 128, 300, 2)])
def test_one_long_sequence_and_many_short_ones(nnb, ctx, fmt, D, hq, hk):
    """An item cut over all blocks next to many that are not; more sequences than a warp counts at once; groups of 3 to 150 heads."""
    seqs = [(1, 9000)] + [(1 + i % 3, 1 + (37 * i) % 140) for i in range(75)] + [(0, 50)] * 5 + [(2, 700)]
    c = ref.Cache(nnb, ctx, fmt, [n for _, n in seqs], hk, D, 16, seed=26)
    q = _queries(seqs, hq, D)
    for max_new in (1, 64):                         # (fewer than there are: served all the same)
        got = run_attention(nnb, ctx, c, q, [n for n, _ in seqs], max_new=max_new, extra=1)
        ctx.sync()
        check_attention(c, got, q, seqs, D ** -0.5, 0, 0, f"many {fmt} D{D} {hq}/{hk} max_new {max_new}")
    c.close()


@pytest.mark.parametrize("scale,size", [(1.0, 30.0), (1e-3, 1.0), (0.125, 6e4), (50.0, 8.0)])
@pytest.mark.parametrize("shape", ["token", "chunk"])
@pytest.mark.parametrize("fmt", ["fp16", "fp8"])
def test_steep_and_flat_scores(nnb, ctx, fmt, shape, scale, size):
    """Scores up to 1e11 (one key takes all) and next to none."""
    seqs, hq, hk, D = SHAPES[shape], 2, 1, 64
    c = ref.Cache(nnb, ctx, fmt, [n for _, n in seqs], hk, D, 16, seed=27)
    q = (np.clip(_queries(seqs, hq, D).astype(np.float32), -1, 1) * size).astype(np.float16)
    got = run_attention(nnb, ctx, c, q, [n for n, _ in seqs], scale=scale)
    ctx.sync()
    check_attention(c, got, q, seqs, scale, 0, 0, f"scale {scale} size {size} {fmt} {shape}")
    c.close()


@pytest.mark.parametrize("window,sinks", [(2 ** 31 - 1, 2 ** 31 - 1), (1, 2 ** 31 - 1), (2 ** 31 - 1, 1), (33, 1000)])
@pytest.mark.parametrize("shape", ["drafts", "long chunk"])
def test_windows_and_sinks_beyond_the_sequence(nnb, ctx, shape, window, sinks):
    seqs, hq, hk, D = SHAPES[shape], 2, 1, 64
    c = ref.Cache(nnb, ctx, "fp16", [n for _, n in seqs], hk, D, 64, seed=28)
    q = _queries(seqs, hq, D)
    got = run_attention(nnb, ctx, c, q, [n for n, _ in seqs], window=window, sinks=sinks)
    ctx.sync()
    check_attention(c, got, q, seqs, D ** -0.5, window, sinks, f"window {window} sinks {sinks} {shape}")
    c.close()


def test_no_rows_and_too_much_work(nnb, ctx):
    c = ref.Cache(nnb, ctx, "int8", [10, 10], 1, 64, 16, seed=29)
    b = c.batch([0, 0])
    ctx.attention(c.handle, b, 1, None, 0, None, 0, 1.0)                 # no rows: nothing to do
    q, out = ctx.alloc(4096), ctx.alloc(4096)
    before = ctx.launch_count()
    b = c.batch([0, 0], extra_rows=4)
    ctx.attention(c.handle, b, 1, q, 0, out, 0, 1.0)                     # rows of no sequence
    ctx.sync()
    assert ctx.launch_count() - before == 1
    huge = nnb.KVBatch(1 << 12, 4, 1, 1 << 30, 1 << 26, b.row_start, b.kv_len, b.page_table)
    with pytest.raises(nnb.NNError) as e:                                # (refused before anything is read)
        ctx.attention(c.handle, huge, 1, q, 0, out, 0, 1.0)
    assert e.value.code in (nnb.NN_ERR_UNSUPPORTED, nnb.NN_ERR_ARG)
    for t in (q, out):
        ctx.free(t)
    c.close()


@pytest.mark.parametrize("fmt,new", [("fp16", 2), ("fp16", 200), ("int8", 1)])
def test_cells_beyond_two_to_the_32_bytes(nnb, ctx, fmt, new):
    """Page numbers whose cells lie more than 4 GiB into a buffer (and more than 2^31 values)."""
    D, H, page, length = 128, 8, 256, 300
    eb = 2 if fmt == "fp16" else 1
    pages = (5 << 30) // (page * H * D * eb)
    k, v = ctx.alloc(5 << 30), ctx.alloc(5 << 30)
    scales = [None, None] if eb == 2 else [ctx.alloc(pages * page * H * 2) for _ in range(2)]
    cache = ctx.kv_cache(fmt, pages, page, H, D, k, v, *scales)
    rng = np.random.default_rng(3)
    x = {n: rng.standard_normal((length, H, D)).astype(np.float16) for n in "kv"}
    up = [ctx.upload(a) for a in (np.array([0, length], np.int32), np.array([0, new], np.int32), np.array([length], np.int32), np.array([[pages - 1, pages - 2]], np.int32), x["k"], x["v"])]
    ctx.kv_write(cache, nnb.KVBatch(1, length, length, 512, 2, up[0], up[2], up[3]), up[4], 0, up[5], 0)
    q = _queries([(new, length)], H, D)
    qb, out = ctx.upload(q), ctx.alloc(q.nbytes)
    ctx.attention(cache, nnb.KVBatch(1, new, new, 512, 2, up[1], up[2], up[3]), H, qb, 0, out, 0, D ** -0.5)
    got = ctx.download(out, q.shape, np.float16)

    class Plain:
        kv_heads = H

        def sequence(self, name, i, n):
            if fmt == "fp16":
                return x[name].astype(np.float64)
            codes, scale = ref.quantised(x[name], fmt)
            return ref.code_values(codes, fmt) * scale.astype(np.float64)[..., None]

    check_attention(Plain(), got, q, [(new, length)], D ** -0.5, 0, 0, f"far cells {fmt}")
    cache.close()
    for t in (*up, k, v, qb, out, *[s for s in scales if s]):
        ctx.free(t)


def test_from_another_thread(nnb, ctx):
    """A thread that has made no call on the device before."""
    seqs, D = SHAPES["drafts"], 64
    c = ref.Cache(nnb, ctx, "int8", [n for _, n in seqs], 2, D, 16, seed=30)
    q = _queries(seqs, 4, D)
    got = []
    t = threading.Thread(target=lambda: got.append(run_attention(nnb, ctx, c, q, [n for n, _ in seqs])))
    t.start()
    t.join()
    check_attention(c, got[0], q, seqs, D ** -0.5, 0, 0, "another thread")
    c.close()


def test_a_cache_of_another_context(nnb, ctx):
    """A handle may be used by every context of its device; each has its own workspace, so their calls may run at the same time."""
    seqs, D = [(1, 3000), (1, 70)], 64
    c = ref.Cache(nnb, ctx, "fp16", [n for _, n in seqs], 1, D, 64, seed=31)
    q = _queries(seqs, 8, D)
    want = run_attention(nnb, ctx, c, q, [1, 1])
    other = nnb.Context()
    b = c.batch([1, 1])
    ctx.sync()
    bufs = [(x, x.upload(q), x.alloc(q.nbytes)) for x in (ctx, other)]
    for _ in range(30):
        for x, qb, out in bufs:
            x.attention(c.handle, b, 8, qb, 0, out, 0, D ** -0.5)
    for x, qb, out in bufs:
        assert np.array_equal(x.download(out, q.shape, np.uint16), want.view(np.uint16))
    other.close()
    for b in bufs[0][1:]:
        ctx.free(b)
    c.close()


@pytest.mark.parametrize("fmt,D", [("fp16", 64), ("int8", 128)])
def test_recorded_calls_of_both_kinds_take_new_batches(nnb, ctx, fmt, D):
    """A chunk, tokens and a read back in one recording, replayed while row starts and lengths change between replays (sequences without rows
    too): the bits of separate calls, whose counters and partial results they share."""
    lengths, hq, hk, rows, spare = [900, 333, 64, 2000], 8, 2, 220, 0x7E7E
    c = ref.Cache(nnb, ctx, fmt, lengths, hk, D, 32, seed=33)
    q = np.random.default_rng(34).standard_normal((rows, hq, D)).astype(np.float16)
    qb, outs, reads = ctx.upload(q), [ctx.alloc(q.nbytes) for _ in range(2)], [ctx.alloc(rows * hk * D * 2) for _ in range(2)]
    start, lens = ctx.alloc(4 * 5), ctx.alloc(4 * 4)
    batches = [nnb.KVBatch(4, rows, m, c.table.shape[1] * 32, c.table.shape[1], start, lens, ctx.upload(c.table)) for m in (200, 1)]

    def call():
        for b, out in zip(batches, outs):
            ctx.attention(c.handle, b, hq, qb, 0, out, 0, D ** -0.5)
        ctx.kv_read(c.handle, batches[0], reads[0], 0, reads[1], 0)

    def results():
        return [ctx.download(b, (rows, w, D), np.uint16) for b, w in (*((o, hq) for o in outs), *((r, hk) for r in reads))]

    ctx.plan_begin()
    call()
    plan = ctx.plan_end()
    for new, now in (([200, 1, 0, 5], [900, 333, 64, 2000]), ([1, 1, 1, 1], [1, 200, 64, 1999]), ([0, 0, 0, 0], [5, 5, 5, 5]), ([0, 220, 0, 0], [9, 333, 0, 7]), ([3, 64, 64, 64], [700, 64, 64, 2000])):
        ctx.upload(np.concatenate([[0], np.cumsum(new)]).astype(np.int32), start)
        ctx.upload(np.asarray(now, np.int32), lens)
        got = []
        for replay in (False, True):
            for b, w in (*((o, hq) for o in outs), *((r, hk) for r in reads)):
                ctx.upload(np.full((rows, w, D), spare, np.uint16), b)
            ctx.plan_launch(plan) if replay else call()
            got.append(results())
        for a, b in zip(*got):
            assert np.array_equal(a, b)
        total = sum(new)
        for out in got[0][:2]:
            assert (out[total:] == spare).all()
            check_attention(c, out.view(np.float16), q, list(zip(new, now)), D ** -0.5, 0, 0, f"replay {new}")
    c.close()
    for b in (qb, *outs, *reads, start, lens):
        ctx.free(b)
