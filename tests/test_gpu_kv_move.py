"""Cells that move to earlier positions, and beams that take over their parents' sequences: every byte of the caches against host loops."""
import numpy as np
import pytest

import kv_reference as ref

pytestmark = pytest.mark.gpu

LAYERS = {"one fp16": [("fp16", 2, 64)], "three int8": [("int8", 3, 64)] * 3, "mixed": [("fp16", 1, 128), ("fp8", 5, 64), ("int8", 2, 128)], "many": [("int8", 1, 64)] * 70}


class Layers:
    """Caches of several layers over the same pages, random bytes in every cell."""

    def __init__(self, nnb, ctx, kinds, pages, page, seed):
        rng = np.random.default_rng(seed)
        self.ctx, self.page, self.host, self.dev, self.handles = ctx, page, [], [], []
        for fmt, heads, D in kinds:
            eb = 2 if fmt == "fp16" else 1
            host = {n: rng.integers(0, 256, (pages, heads, page, D * eb), dtype=np.uint8) for n in "kv"}
            if fmt != "fp16":
                host.update({n + "_scale": rng.integers(0, 1 << 16, (pages, heads, page), dtype=np.uint16) for n in "kv"})
            dev = {n: ctx.upload(a) for n, a in host.items()}
            self.host.append(host)
            self.dev.append(dev)
            self.handles.append(ctx.kv_cache(fmt, pages, page, heads, D, dev["k"], dev["v"], dev.get("k_scale"), dev.get("v_scale")))

    def move(self, pairs):
        """((page, slot) to, from) pairs, as if all were read first."""
        for host in self.host:
            for name, a in host.items():
                new = [(to, a[f[0], :, f[1]].copy()) for to, f in pairs]
                for (page, slot), x in new:
                    a[page, :, slot] = x

    def check(self, what=""):
        for i, (host, dev) in enumerate(zip(self.host, self.dev)):
            for name, a in host.items():
                got = self.ctx.download(dev[name], a.shape, a.dtype)
                assert np.array_equal(got, a), (what, i, name, np.argwhere(got != a)[:3])

    def close(self):
        self.ctx.sync()
        for h in self.handles:
            h.close()
        for dev in self.dev:
            for b in dev.values():
                self.ctx.free(b)


def place(table, s, p, page):
    return int(table[s, p // page]), p % page


@pytest.mark.parametrize("kinds", LAYERS)
@pytest.mark.parametrize("page", [16, 64, 256])
def test_moves(nnb, ctx, kinds, page):
    rng = np.random.default_rng(61)
    # rows, length before, length after
    seqs = [(1, 40, 7), (5, 60, 31), (0, 3, 3), (300, 900, 450), (16, 16, 16), (700, 1500, 701)]
    need = [-(-n // page) for _, n, _ in seqs]
    pages = sum(need) + 2
    order, table = rng.permutation(pages), np.full((len(seqs), max(need) + 1), -9, np.int32)
    for i, n in enumerate(need):
        table[i, :n], order = order[:n], order[n:]
    layers = Layers(nnb, ctx, LAYERS[kinds], pages, page, 62)
    source, pairs = [], []
    for i, (n, before, after) in enumerate(seqs):
        base = after - n
        at = np.sort(rng.choice(np.arange(base, before), n, replace=False)) if n != 700 else np.arange(base + 1, base + 701)     # (each to its neighbour's place)
        source += list(at)
        pairs += [(place(table, i, base + j, page), place(table, i, int(p), page)) for j, p in enumerate(at)]
    start = np.concatenate([[0], np.cumsum([n for n, _, _ in seqs])]).astype(np.int32)
    up = [ctx.upload(np.ascontiguousarray(a, np.int32)) for a in (start, [a for _, _, a in seqs], table, source + [5, 5])]
    b = nnb.KVBatch(len(seqs), len(source) + 2, 700, table.shape[1] * page, table.shape[1], *up[:3])     # (two rows behind the last sequence)
    for _ in range(2):     # (a second time moves on from what the first one left)
        ctx.kv_move(layers.handles, b, up[3])
        ctx.sync()
        layers.move(pairs)
        layers.check(kinds)
    ctx.kv_move([], b, up[3])
    ctx.sync()
    layers.close()
    for x in up:
        ctx.free(x)


def test_bad_moves_are_left_out(nnb, ctx):
    page, pages = 16, 8
    layers = Layers(nnb, ctx, [("int8", 2, 64), ("fp16", 1, 128)], pages, page, 63)
    table = np.array([[3, 1, 5, 99], [0, 2, -1, 4]], np.int32)
    # sequence 0, rows for positions 10 .. 15: before the row; a bad page (48 .. 63); at the end of the tables; not ascending; good ones
    source = [9, 50, 64, 60, 20, 33] + [3, 40, 49]
    up = [ctx.upload(np.ascontiguousarray(a, np.int32)) for a in ([0, 6, 9], [16, 5], table, source)]
    b = nnb.KVBatch(2, 9, 6, 64, 4, *up[:3])
    ctx.kv_move(layers.handles, b, up[3])
    with pytest.raises(nnb.NNError) as e:
        ctx.sync()
    assert e.value.code == nnb.NN_ERR_ARG and "out of range" in str(e.value)
    # row 4's source 20 is not above row 3's 60; row 5's 33 is above row 4's; sequence 1: 3 -> 2, then a bad page, then 49 -> 4
    layers.move([((3, 15), (5, 1)), ((0, 2), (0, 3)), ((0, 4), (4, 1))])
    layers.check()
    for bad in (dict(lens=[-1, 5]), dict(lens=[65, 5]), dict(lens=[5, 2])):     # out of range, or fewer positions than rows
        ctx.upload(np.asarray(bad["lens"], np.int32), up[1])
        ctx.upload(np.asarray([20] * 6 + [0] * 3, np.int32), up[3])
        ctx.kv_move(layers.handles, nnb.KVBatch(1, 9, 6, 64, 4, *up[:3]), up[3])
        if bad["lens"][0] != 5:
            with pytest.raises(nnb.NNError):
                ctx.sync()
        else:
            with pytest.raises(nnb.NNError):
                ctx.sync()
        layers.check()
    layers.close()
    for x in up:
        ctx.free(x)


def beam_tables(rng, groups, beams, lengths, page, extra=1):
    """Tables whose full pages are shared at random and whose others are each beam's own."""
    width = max(n // page for n in lengths) + 1 + extra
    pages = groups * beams * width
    table = rng.permutation(pages).astype(np.int32).reshape(groups * beams, width)
    for g, n in enumerate(lengths):
        for i in range(n // page):
            rows = slice(g * beams, (g + 1) * beams)
            table[rows, i] = table[rows, i][rng.integers(0, beams, beams)]
    return table, pages


def reorder_host(layers, table, lengths, beams, parents, page):
    old = table.copy()
    pairs = []
    for s in range(len(table)):
        g = s // beams
        p = parents[s] if parents[s] >= 0 else s % beams
        n, t = lengths[g], g * beams + p
        table[s, :n // page] = old[t, :n // page]
        if p != s % beams:
            pairs += [((int(old[s, n // page]), x), (int(old[t, n // page]), x)) for x in range(n % page)]
    layers.move(pairs)


@pytest.mark.parametrize("kinds", LAYERS)
@pytest.mark.parametrize("beams", [1, 2, 5, 8, 9, 16, 32])
def test_reorders(nnb, ctx, kinds, beams):
    rng = np.random.default_rng(71 + beams)
    page = 32 if beams < 9 else 16
    lengths = [0, 1, page, 5 * page + 7, 3 * page - 1]
    groups = len(lengths)
    table, pages = beam_tables(rng, groups, beams, lengths, page)
    layers = Layers(nnb, ctx, LAYERS[kinds], pages, page, 72)
    kv_len = ctx.upload(np.repeat(lengths, beams).astype(np.int32))
    tb = ctx.upload(table)
    b = nnb.KVBatch(groups * beams, 0, 0, table.shape[1] * page, table.shape[1], None, kv_len, tb)
    for turn in range(4):
        parents = rng.integers(-1, beams, groups * beams).astype(np.int32)
        if turn == 1:      # a cycle through all beams
            parents = np.tile(np.roll(np.arange(beams), 1), groups).astype(np.int32)
        if turn == 2:
            parents[:] = 0
        pb = ctx.upload(parents)
        ctx.kv_reorder(layers.handles, b, beams, pb)
        ctx.sync()
        reorder_host(layers, table, lengths, beams, parents, page)
        layers.check((kinds, beams, turn))
        assert np.array_equal(ctx.download(tb, table.shape, np.int32), table)
        ctx.free(pb)
    layers.close()
    for x in (kv_len, tb):
        ctx.free(x)


@pytest.mark.parametrize("what", ["parent", "parent below", "length", "lengths differ", "length below", "page", "read page", "same page"])
def test_bad_groups_are_left_as_they_are(nnb, ctx, what):
    rng = np.random.default_rng(81)
    beams, page, lengths = 3, 16, [40, 37, 55]
    table, pages = beam_tables(rng, 3, beams, lengths, page)
    layers = Layers(nnb, ctx, LAYERS["mixed"], pages, page, 82)
    lens, parents = np.repeat(lengths, beams).astype(np.int32), np.array([1, 1, 0, 2, 0, 1, 0, 0, 2], np.int32)
    good = (table.copy(), lens.copy(), parents.copy())
    if what == "parent":
        parents[4] = beams
    elif what == "parent below":
        parents[4] = -2
    elif what == "length":
        lens[3:6] = table.shape[1] * page + 1
    elif what == "lengths differ":
        lens[5] = 36
    elif what == "length below":
        lens[3:6] = -1
    elif what == "page":
        table[4, 2] = pages
    elif what == "read page":
        table[5, 2] = -1
        parents[5] = -1      # not written, but the third beam's cells are asked for
        parents[3] = 2
    else:
        table[4, 2] = table[3, 2]
    tb, kb, pb = ctx.upload(table), ctx.upload(lens), ctx.upload(parents)
    b = nnb.KVBatch(9, 0, 0, table.shape[1] * page, table.shape[1], None, kb, tb)
    ctx.kv_reorder(layers.handles, b, beams, pb)
    with pytest.raises(nnb.NNError) as e:
        ctx.sync()
    assert e.value.code == nnb.NN_ERR_ARG and "out of range" in str(e.value)
    ctx.sync()
    for g in (0, 2):       # the others are served
        part = table[g * beams:(g + 1) * beams]
        reorder_host(layers, part, [lengths[g]], beams, parents[g * beams:(g + 1) * beams], page)
    layers.check(what)
    assert np.array_equal(ctx.download(tb, table.shape, np.int32), table)
    layers.close()
    for x in (tb, kb, pb):
        ctx.free(x)


def test_pages_that_one_layer_does_not_have(nnb, ctx):
    """Layers with more pages than others: what the smallest does not have is bad in all of them."""
    page = 16
    large, small = (Layers(nnb, ctx, [(fmt, 2, 64)], n, page, 83) for fmt, n in (("fp16", 8), ("int8", 4)))
    both = large.handles + small.handles
    # a sequence in both, one with a page that only the first has
    table = np.array([[0, 1], [2, 5]], np.int32)
    up = [ctx.upload(np.ascontiguousarray(a, np.int32)) for a in ([0, 1, 2], [10, 10], table, [20, 20], [30, 30], [1, 0])]
    ctx.kv_move(both, nnb.KVBatch(2, 2, 1, 32, 2, *up[:3]), up[3])
    with pytest.raises(nnb.NNError):
        ctx.sync()
    for layers in (large, small):
        layers.move([((0, 9), (1, 4))])
        layers.check()
    ctx.kv_reorder(both, nnb.KVBatch(2, 0, 0, 32, 2, None, up[4], up[2]), 2, up[5])     # (the beams change places)
    with pytest.raises(nnb.NNError):
        ctx.sync()
    for layers in (large, small):
        layers.check()
        layers.close()
    assert np.array_equal(ctx.download(up[2], table.shape, np.int32), table)
    for x in up:
        ctx.free(x)
