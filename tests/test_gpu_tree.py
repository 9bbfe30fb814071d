"""Drafted trees: their layout, the write at given positions and the attention over the cache, against host loops and the formula in 64 bits."""
import numpy as np
import pytest

import branch_reference as br
import kv_reference as ref
from helpers import alloc_with_canary, check_canary, report

pytestmark = pytest.mark.gpu

HEADS = {"mha": (3, 3), "gqa3": (9, 3), "gqa7": (14, 2), "mqa": (8, 1), "mqa40": (40, 1)}
# (drafted tokens, length) of each sequence
BATCHES = {
    "one": [(1, 1)],
    "few": [(1, 700), (5, 300), (8, 8), (0, 50), (2, 65)],
    "some": [(26, 700), (33, 65), (31, 31), (32, 129)],
    "many": [(64, 1000), (130, 500), (64, 64), (1, 90), (200, 263)],
    "negative": [(5, 3), (2, 0), (1, 20)],      # more rows than positions: those that are not there are not seen
}


def queries(rows, hq, D, seed=12):
    return np.random.default_rng(seed).standard_normal((rows, hq, D)).astype(np.float16)


def run_tree(nnb, ctx, c, q, new, masks, words, extra=0, **bounds):
    """out [rows + extra, heads, D]; rows behind the last sequence keep what they held."""
    rows, hq, D = q.shape
    n = (rows + extra) * hq * D * 2
    bits = np.concatenate([br.words_of(masks, words), np.full((extra, words), 0xFFFFFFFF, np.uint32)])
    qb, mb, out = ctx.upload(np.concatenate([q, np.zeros((extra, hq, D), np.float16)])), ctx.upload(bits), alloc_with_canary(ctx, n)
    ctx.attention_tree(c.handle, c.batch(new, extra_rows=extra, **bounds), hq, qb, 0, out, 0, D ** -0.5, words, mb)
    got = ctx.download(out, (rows + extra, hq, D), np.float16)
    check_canary(ctx, out, n)
    for b in (qb, mb, out):
        ctx.free(b)
    return got


def check_tree(c, got, q, seqs, masks, what=""):
    hq, D = q.shape[1:]
    group, row, worst = hq // c.kv_heads, 0, 0.0
    for i, (new, length) in enumerate(seqs):
        k, v = c.sequence("k", i, length), c.sequence("v", i, length)
        keys = [br.tree_keys(m, new, length) for m in masks[row:row + new]]
        for h in range(hq):
            want, spread, most, steep = br.attend_keys(q[row:row + new, h].astype(np.float64), k[:, h // group], v[:, h // group], D ** -0.5, keys)
            bound = ref.attention_bound(want, spread, most, steep, length, D)
            have = got[row:row + new, h].astype(np.float64)
            assert np.array_equal(np.isfinite(have), np.isfinite(want)), (what, i, h, np.argwhere(np.isfinite(have) != np.isfinite(want))[:4])
            fine = np.isfinite(want)
            with np.errstate(invalid="ignore"):
                off = np.abs(have - want)[fine] / bound[fine]
            if off.size:
                worst = max(worst, off.max())
                assert off.max() <= 1, (what, i, h, off.max())
        row += new
    report(f"tree {what}: worst error {worst:.2f} of its bound")


def trees_of(seqs, seed, kind="tree"):
    rng = np.random.default_rng(seed)
    masks = []
    for n, _ in seqs:
        if kind == "tree":
            masks += br.masks_of(br.random_tree(n, rng))[0]
        elif kind == "chain":
            masks += [(2 << i) - 1 for i in range(n)]
        else:   # anything: rows without themselves, with later ones, without any, bits behind the last token
            masks += [0 if rng.random() < 0.2 else int.from_bytes(rng.bytes(2 + n // 8), "little") for _ in range(n)]
    return masks


@pytest.mark.parametrize("kind", ["tree", "any"])
@pytest.mark.parametrize("batch", BATCHES)
@pytest.mark.parametrize("fmt,D,page,heads", [("fp16", 64, 16, "gqa3"), ("int8", 64, 64, "gqa7"), ("fp8", 64, 256, "mha"), ("fp16", 128, 128, "mqa"),
                                              ("int8", 128, 32, "mqa40"), ("fp8", 128, 16, "gqa3"), ("fp16", 64, 64, "mqa40"), ("fp8", 64, 32, "mqa")])
def test_tree_attention(nnb, ctx, fmt, D, page, heads, batch, kind):
    seqs = BATCHES[batch]
    hq, hk = HEADS[heads]
    words = -(-max(n for n, _ in seqs) // 32)
    c = ref.Cache(nnb, ctx, fmt, [n for _, n in seqs], hk, D, page, seed=11)
    new = [n for n, _ in seqs]
    q, masks = queries(sum(new), hq, D), trees_of(seqs, 5, kind)
    masks = [m & (1 << 32 * words) - 1 for m in masks]
    got = run_tree(nnb, ctx, c, q, new, masks, words, extra=3)
    ctx.sync()
    assert (got[len(q):].view(np.uint16) == 0x7E7E).all()          # rows behind the last sequence
    check_tree(c, got, q, seqs, masks, f"{fmt} D{D} {heads} {batch} {kind}")
    again = run_tree(nnb, ctx, c, q, new, masks, words, extra=3)
    assert np.array_equal(got.view(np.uint16), again.view(np.uint16))
    # the kernel that the batch's bound picks, and masks that are wider than need be
    wide = run_tree(nnb, ctx, c, q, new, masks, words + 2, max_new=1 if max(new) > 1 else 64)
    ctx.sync()
    check_tree(c, wide, q, seqs, masks, f"{fmt} D{D} {heads} {batch} {kind}, other kernel")
    c.close()


@pytest.mark.parametrize("fmt,D", [("fp16", 64), ("int8", 128)])
@pytest.mark.parametrize("n", [1, 6, 150])
def test_a_chain_is_a_draft(nnb, ctx, fmt, D, n):
    """A tree that is a chain gives the bits of the attention of new tokens one behind the other: the same kernel, the same keys."""
    seqs = [(n, 400), (n, n + 7)]
    c = ref.Cache(nnb, ctx, fmt, [x for _, x in seqs], 2, D, 32, seed=21)
    q = queries(2 * n, 4, D)
    got = run_tree(nnb, ctx, c, q, [n, n], trees_of(seqs, 0, "chain"), -(-n // 32))
    out = ctx.alloc(q.nbytes)
    qb = ctx.upload(q)
    ctx.attention(c.handle, c.batch([n, n]), 4, qb, 0, out, 0, D ** -0.5)
    want = ctx.download(out, q.shape, np.float16)
    if n <= 8:      # (one item of the work for each head: tiles and splits are the same)
        assert np.array_equal(got.view(np.uint16), want.view(np.uint16))
    check_tree(c, got, q, seqs, trees_of(seqs, 0, "chain"), "chain")
    check_tree(c, want, q, seqs, trees_of(seqs, 0, "chain"), "draft")
    for b in (out, qb):
        ctx.free(b)
    c.close()


@pytest.mark.parametrize("n", [7, 64, 150])
@pytest.mark.parametrize("fmt,D", [("fp16", 64), ("fp16", 128), ("int8", 64), ("int8", 128), ("fp8", 64), ("fp8", 128)])
def test_cells_that_are_not_finite(nnb, ctx, fmt, D, n):
    """Infinities and NaNs, in the sequence and in drafted tokens: rows that see them give what the formula gives, the others are not touched by them."""
    seqs, hq, hk = [(n, 300), (n, n + 5)], 4, 2
    c = ref.Cache(nnb, ctx, fmt, [x for _, x in seqs], hk, D, 16, seed=22)
    for i, (_, length) in enumerate(seqs):
        for name, pos, head, dim, value in (("v", length - n + 3, 0, 5, np.nan), ("k", length - n + 4, 1, 9, np.inf), ("v", 2, 1, D - 1, -np.inf), ("k", length - n + 1, 0, 0, np.nan)):
            page, slot = c.table[i, pos // c.page], pos % c.page
            if fmt == "fp16":
                c.host[name].view(np.float16)[page, head, slot, dim] = value
            else:
                c.host[name + "_scale"][page, head, slot] = value
    for name in "kv":
        ctx.upload(c.host[name], c.dev[name])
        if fmt != "fp16":
            ctx.upload(c.host[name + "_scale"].view(np.uint16), c.dev[name + "_scale"])
    q, masks = queries(2 * n, hq, D), trees_of(seqs, 8)
    got = run_tree(nnb, ctx, c, q, [n, n], masks, -(-n // 32))
    ctx.sync()
    check_tree(c, got, q, seqs, masks, f"not finite {fmt} D{D} {n}")
    c.close()


@pytest.mark.parametrize("fmt,D,hq,hk,n", [("int8", 64, 8, 1, 16), ("fp16", 128, 4, 1, 64)])
def test_long_sequences(nnb, ctx, fmt, D, hq, hk, n):
    seqs = [(n, 40001)]
    c = ref.Cache(nnb, ctx, fmt, [40001], hk, D, 256, seed=23)
    q, masks = queries(n, hq, D), trees_of(seqs, 9)
    got = run_tree(nnb, ctx, c, q, [n], masks, 2)
    ctx.sync()
    check_tree(c, got, q, seqs, masks, f"long {fmt}")
    c.close()


@pytest.mark.parametrize("max_new", [1, 200])
def test_bad_sequences_are_left_out(nnb, ctx, max_new):
    """More new rows than a mask has bits, bad lengths, bad pages, row starts that do not ascend: reported, and the context stays usable."""
    seqs, D = [(40, 120), (20, 90)], 64
    words = max(1, -(-max_new // 32))
    c = ref.Cache(nnb, ctx, "fp16", [n for _, n in seqs], 1, D, 16, seed=24)
    q, masks = queries(60, 2, D), trees_of(seqs, 3)
    with pytest.raises(nnb.NNError) as e:
        run_tree(nnb, ctx, c, q, [40, 20], [m & 0xFFFFFFFF for m in masks], 1, max_new=1)      # 40 rows, 32 bits
        ctx.sync()
    assert e.value.code == nnb.NN_ERR_ARG and "out of range" in str(e.value)
    n = 60 * 2 * D * 2
    qb, mb, out = ctx.upload(q), ctx.upload(br.words_of([m & 0xFFFFFFFF for m in masks], 1)), alloc_with_canary(ctx, n)
    ctx.attention_tree(c.handle, c.batch([40, 20], max_new=1), 2, qb, 0, out, 0, D ** -0.5, 1, mb)
    with pytest.raises(nnb.NNError):
        ctx.sync()
    got = ctx.download(out, q.shape, np.float16)
    assert (got[:40].view(np.uint16) == 0x7E7E).all()
    kk, vv = c.sequence("k", 1, 90), c.sequence("v", 1, 90)
    for h in range(2):
        want, spread, most, steep = br.attend_keys(q[40:, h].astype(np.float64), kk[:, 0], vv[:, 0], D ** -0.5, [br.tree_keys(m & 0xFFFFFFFF, 20, 90) for m in masks[40:]])
        assert (np.abs(got[40:, h] - want) <= ref.attention_bound(want, spread, most, steep, 90, D)).all()
    table = c.table.copy()
    table[0, 1] = c.pages
    for bad in (dict(table=table), dict(row_start=[0, 50, 40]), dict(row_start=[0, 40, 1 << 30]), dict(lengths=[120, 1 << 29])):
        new = [40, 20]
        start = bad.pop("row_start", None)
        b = c.batch(new, max_new=max_new, row_start=None, **bad)
        if start:
            s = ctx.upload(np.asarray(start, np.int32))
            c.kept.append(s)
            b.row_start = s
        mw = ctx.upload(br.words_of([m & (1 << 32 * 7) - 1 for m in masks], 7))
        ctx.attention_tree(c.handle, b, 2, qb, 0, out, 0, D ** -0.5, 7, mw)
        with pytest.raises(nnb.NNError) as e:
            ctx.sync()
        assert e.value.code == nnb.NN_ERR_ARG
        check_canary(ctx, out, n)
        ctx.free(mw)
    good = run_tree(nnb, ctx, c, q, [40, 20], masks, 7, max_new=max_new)
    ctx.sync()
    check_tree(c, good, q, seqs, masks, "after bad ones")
    for b in (qb, mb, out):
        ctx.free(b)
    c.close()


@pytest.mark.parametrize("sizes", [[1], [26], [0, 33, 5, 0], [64, 100, 1], [1024, 700], [32, 31]])
def test_layout(nnb, ctx, sizes):
    rng = np.random.default_rng(31)
    lengths = [n + int(rng.integers(0, 50)) for n in sizes]
    trees = [br.random_tree(n, rng) for n in sizes]
    if sizes[0] == 1024:
        trees[0] = [i - 1 for i in range(1024)]        # a chain, and one without edges
        trees[1] = [-1] * 700
    rows, words = sum(sizes), -(-max(sizes) // 32)
    start = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
    up = [ctx.upload(np.asarray(a, np.int32)) for a in (start, lengths, sum(trees, []) or [0])]
    mask, pos = alloc_with_canary(ctx, (rows + 2) * words * 4), alloc_with_canary(ctx, (rows + 2) * 4)
    b = nnb.KVBatch(len(sizes), rows + 2, max(sizes), max(lengths) + 1, 0, up[0], up[1], None)
    ctx.tree_layout(b, ctx.upload(np.asarray(sum(trees, []) + [77, 77], np.int32), ctx.alloc(4 * rows + 8)), words, mask, pos)
    ctx.sync()
    want = [br.masks_of(t) for t in trees]
    got = ctx.download(mask, (rows + 2, words), np.uint32)
    assert np.array_equal(got[:rows], br.words_of(sum((m for m, _ in want), []), words))
    assert (got[rows:] == 0x7E7E7E7E).all()
    at = ctx.download(pos, (rows + 2,), np.int32)
    assert np.array_equal(at[:rows], np.concatenate([[ln - n + d for d in ds] for (_, ds), n, ln in zip(want, sizes, lengths)]).astype(np.int32))
    assert (at[rows:] == 0x7E7E7E7E).all()
    check_canary(ctx, mask, (rows + 2) * words * 4)
    check_canary(ctx, pos, (rows + 2) * 4)
    for x in (*up, mask, pos):
        ctx.free(x)


def test_layout_of_bad_trees(nnb, ctx):
    """A parent that does not come before its child counts as none; sequences that are too long or whose numbers are bad are left as they are."""
    up = lambda a: ctx.upload(np.asarray(a, np.int32))  # noqa: E731
    parent = up([-1, 0, 2, -5, 1 << 30] + [-1] * 35)
    mask, pos = ctx.upload(np.full(40, 9, np.int32)), ctx.upload(np.full(40, 9, np.int32))
    start, lens = up([0, 5, 40]), up([10, 40])
    ctx.tree_layout(nnb.KVBatch(2, 40, 32, 100, 0, start, lens, None), parent, 1, mask, pos)      # the second has 35 rows
    with pytest.raises(nnb.NNError) as e:
        ctx.sync()
    assert e.value.code == nnb.NN_ERR_ARG
    m, p = ctx.download(mask, (40,), np.int32), ctx.download(pos, (40,), np.int32)
    assert list(m[:5]) == [1, 3, 4, 8, 16] and list(p[:5]) == [5, 6, 5, 5, 5] and (m[5:] == 9).all() and (p[5:] == 9).all()
    for lengths in ([4, 90], [-1, 90], [101, 90]):    # fewer positions than rows; out of range
        ctx.upload(np.asarray(lengths, np.int32), lens)
        ctx.tree_layout(nnb.KVBatch(1, 40, 32, 100, 0, start, lens, None), parent, 1, mask, pos)
        with pytest.raises(nnb.NNError):
            ctx.sync()
    ctx.sync()
    for b in (parent, mask, pos, start, lens):
        ctx.free(b)


@pytest.mark.parametrize("fmt,D,rotary", [("fp16", 64, 64), ("int8", 128, 32), ("fp8", 64, 64)])
@pytest.mark.parametrize("new", [[5, 0, 17], [700, 5]])
def test_write_at_positions(nnb, ctx, fmt, D, rotary, new):
    """The rotation goes by the given positions, the cells by the rows' own; rows whose position is out of the tables' range are left out."""
    lengths = [n + 9 for n in new]
    hq, hk, rows, table_len = 6, 2, sum(new), 800
    rng = np.random.default_rng(41)
    c = ref.Cache(nnb, ctx, fmt, lengths, hk, D, 16, seed=42)
    q, k, v = (rng.standard_normal((rows, h, D)).astype(np.float16) for h in (hq, hk, hk))
    angle = np.arange(table_len)[:, None] * 10000.0 ** (-np.arange(0, rotary, 2) / rotary)
    cos, sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
    pos = rng.integers(0, table_len, rows).astype(np.int32)
    up = [ctx.upload(a) for a in (cos, sin, q, k, v)]
    qo = alloc_with_canary(ctx, q.nbytes)
    for bad in (False, True):
        if bad:
            pos[[0, rows // 2, rows - 1]] = [-1, table_len, -(1 << 31)]
        pb = ctx.upload(pos)
        ctx.rope_kv_write_at(c.handle, c.batch(new), pb, up[0], up[1], table_len, rotary, hq, up[2], 0, qo, 0, up[3], 0, up[4], 0)
        if bad:
            with pytest.raises(nnb.NNError):
                ctx.sync()
        ctx.sync()
        there = (pos >= 0) & (pos < table_len)
        at = np.where(there, pos, 0)
        if bad:   # what lay there stays: rows of the first pass
            at = np.where(there, pos, before)
        want_q, want_k = ref.rotated(q, cos[at], sin[at], rotary), ref.rotated(k, cos[at], sin[at], rotary)
        got_q = ctx.download(qo, q.shape, np.float16)
        assert np.array_equal(got_q.view(np.uint16), want_q.view(np.uint16))
        row = 0
        for i, (n, length) in enumerate(zip(new, lengths)):
            for j in range(n):
                p = length - n + j
                page, slot = c.table[i, p // 16], p % 16
                for name, x in (("k", want_k[row]), ("v", v[row])):
                    if fmt == "fp16":
                        c.host[name][page, :, slot] = x.view(np.uint16)
                    else:
                        c.host[name][page, :, slot], c.host[name + "_scale"][page, :, slot] = ref.quantised(x, fmt)
                row += 1
        got = c.read_back()
        for name in got:
            assert np.array_equal(got[name].view(np.uint8), c.host[name].view(np.uint8)), name
        before = pos.copy()
        ctx.free(pb)
    check_canary(ctx, qo, q.nbytes)
    for b in (*up, qo):
        ctx.free(b)
    c.close()
