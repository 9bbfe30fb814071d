"""Drafted trees and beams as a decode loop uses them: several layers, several steps, eager and recorded."""
import ctypes
import threading

import numpy as np
import pytest

import branch_reference as br
import kv_reference as ref
from test_gpu_beams import draw
from test_gpu_tree import check_tree

pytestmark = pytest.mark.gpu


def _rope_tables(n, D):
    angle = np.arange(n)[:, None] * 10000.0 ** (-np.arange(0, D, 2) / D)
    return np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)


def _read_all(nnb, ctx, c, lengths, table):
    """Every position of every sequence as bits, read back by the library."""
    n = sum(lengths)
    k, v = (ctx.alloc(n * c.kv_heads * c.D * 2) for _ in range(2))
    ctx.kv_read(c.handle, c.batch(lengths, lengths, table=table), k, 0, v, 0)
    ctx.sync()
    got = [ctx.download(b, (n, c.kv_heads, c.D), np.uint16) for b in (k, v)]
    for b in (k, v):
        ctx.free(b)
    return got


@pytest.mark.parametrize("recorded", [False, True])
@pytest.mark.parametrize("fmt,D,hq,hk,nodes", [("int8", 64, 9, 3, [26, 7]), ("fp16", 128, 8, 2, [13, 64]), ("fp8", 64, 4, 4, [1, 40])])
def test_a_tree_is_drafted_checked_and_its_path_kept(nnb, ctx, fmt, D, hq, hk, nodes, recorded):
    """Layout, writes and attention in two layers; then a path's cells move behind the sequence, and the caches are those of a decode loop that wrote the path's
    tokens one behind the other."""
    layers, page, prefix = 2, 16, [37, 90]
    lengths = [p + n for p, n in zip(prefix, nodes)]
    rows, words = sum(nodes), -(-max(nodes) // 32)
    rng = np.random.default_rng(51)
    trees = [br.random_tree(n, rng) for n in nodes]
    masks, depth = zip(*(br.masks_of(t) for t in trees))
    table_len = 160
    cos, sin = _rope_tables(table_len, D)
    caches = [ref.Cache(nnb, ctx, fmt, lengths, hk, D, page, seed=60) for i in range(layers)]       # (layers share their page numbers)
    line = [ref.Cache(nnb, ctx, fmt, lengths, hk, D, page, seed=60) for i in range(layers)]      # the same contents
    q, k, v = ([rng.standard_normal((rows, h, D)).astype(np.float16) for _ in range(layers)] for h in (hq, hk, hk))
    up = lambda a: ctx.upload(np.ascontiguousarray(a))  # noqa: E731
    cb, sb, parent = up(cos), up(sin), up(np.array(sum(trees, []), np.int32))
    mask, pos, out, q_out = ctx.alloc(rows * words * 4), ctx.alloc(rows * 4), [ctx.alloc(rows * hq * D * 2) for _ in range(layers)], [ctx.alloc(rows * hq * D * 2) for _ in range(layers)]
    qb, kb, vb = ([up(x) for x in xs] for xs in (q, k, v))
    batches = [c.batch(nodes) for c in caches]

    def step():
        ctx.tree_layout(batches[0], parent, words, mask, pos)
        for i, c in enumerate(caches):
            ctx.rope_kv_write_at(c.handle, batches[i], pos, cb, sb, table_len, D, hq, qb[i], 0, q_out[i], 0, kb[i], 0, vb[i], 0)
            ctx.attention_tree(c.handle, batches[i], hq, q_out[i], 0, out[i], 0, D ** -0.5, words, mask)

    if recorded:
        ctx.plan_begin()
        step()
        plan = ctx.plan_end()
        for _ in range(2):
            ctx.plan_launch(plan)
        ctx.sync()
        ctx.L.nn_plan_free(plan)
    else:
        step()
    ctx.sync()
    # the attention's rows against the formula, with the cells that the writes have left
    at = np.concatenate([np.array(d) + p for d, p in zip(depth, prefix)])
    for i, c in enumerate(caches):
        got = c.read_back()
        for name in got:
            c.host[name] = got[name].view(c.host[name].dtype)
        turned = ref.rotated(q[i], cos[at], sin[at], D)
        assert np.array_equal(ctx.download(q_out[i], q[i].shape, np.uint16), turned.view(np.uint16))
        check_tree(c, ctx.download(out[i], q[i].shape, np.float16), turned, list(zip(nodes, lengths)), sum(masks, []), f"layer {i} {fmt}")
    # the deepest path of each tree is kept
    source, kept = [], []
    for t, d, p in zip(trees, depth, prefix):
        path, node = [], int(np.argmax(d))
        while node >= 0:
            path.insert(0, node)
            node = t[node]
        kept.append(path)
        source += [p + x for x in path]
    after = [p + len(path) for p, path in zip(prefix, kept)]
    src = up(np.array(source, np.int32))
    ctx.kv_move([c.handle for c in caches], caches[0].batch([len(x) for x in kept], after), src)
    # the loop that has no tree
    first = 0
    row_of = []
    for n, path in zip(nodes, kept):
        row_of += [first + x for x in path]
        first += n
    for i, c in enumerate(line):
        ql, kl, vl = (up(np.ascontiguousarray(x[i][row_of])) for x in (q, k, v))
        ctx.rope_kv_write(c.handle, c.batch([len(x) for x in kept], after), cb, sb, table_len, D, hq, ql, 0, ql, 0, kl, 0, vl, 0)
        ctx.sync()
        a, b = _read_all(nnb, ctx, caches[i], after, caches[i].table), _read_all(nnb, ctx, c, after, c.table)
        assert all(np.array_equal(x, y) for x, y in zip(a, b)), i
        # and the next token sees the same
        nxt, o1, o2 = up(q[i][:2]), ctx.alloc(2 * hq * D * 2), ctx.alloc(2 * hq * D * 2)
        ctx.attention(caches[i].handle, caches[i].batch([1, 1], after), hq, nxt, 0, o1, 0, D ** -0.5)
        ctx.attention(c.handle, c.batch([1, 1], after), hq, nxt, 0, o2, 0, D ** -0.5)
        ctx.sync()
        assert np.array_equal(ctx.download(o1, (2, hq, D), np.uint16), ctx.download(o2, (2, hq, D), np.uint16))
        for x in (ql, kl, vl, nxt, o1, o2):
            ctx.free(x)
    for x in (cb, sb, parent, mask, pos, src, *out, *q_out, *qb, *kb, *vb):
        ctx.free(x)
    for c in (*caches, *line):
        c.close()


@pytest.mark.parametrize("recorded", [False, True])
@pytest.mark.parametrize("fmt,page,prompt", [("fp16", 16, 14), ("int8", 32, 64), ("fp8", 16, 1)])
def test_beams_keep_their_histories(nnb, ctx, fmt, page, prompt, recorded):
    """Selection, reordering and a write for each beam, step after step: every beam's cells are those of its own tokens from the prompt on."""
    groups, beams, vocab, steps, hk, D, layers = 3, 4, 50, 9, 2, 64, 2
    seqs = groups * beams
    rng = np.random.default_rng(71)
    words = rng.standard_normal((layers, 2, vocab, hk, D)).astype(np.float16)      # what a token writes into a layer's keys and values
    lengths = [prompt + steps] * seqs
    caches = [ref.Cache(nnb, ctx, fmt, lengths, hk, D, page, seed=72 + i, fill=False) for i in range(layers)]
    table = caches[0].table.copy()
    for c in caches:                                                               # layers share their page numbers
        c.table[:] = table
    prompts = rng.integers(0, vocab, (groups, prompt))
    up = lambda a: ctx.upload(np.ascontiguousarray(a))  # noqa: E731
    tb, lens = up(table), up(np.zeros(seqs, np.int32))
    starts = up(np.arange(seqs + 1, dtype=np.int32))
    score = up(np.zeros((groups, beams), np.float32))
    done = up(np.zeros((groups, beams), np.int32))
    token, parent, logits = up(np.zeros(seqs, np.int32)), up(np.zeros(seqs, np.int32)), ctx.alloc(seqs * vocab * 2)
    new = [[ctx.alloc(seqs * hk * D * 2) for _ in range(2)] for _ in range(layers)]
    one = nnb.KVBatch(seqs, seqs, 1, table.shape[1] * page, table.shape[1], starts, lens, tb)
    # the prompt goes to the first beam of each group, and from there to all
    for i, c in enumerate(caches):
        rows = [up(words[i, j][prompts].reshape(-1, hk, D)) for j in range(2)]
        first = np.ascontiguousarray(table[::beams])
        fb = up(first)
        b = nnb.KVBatch(groups, groups * prompt, prompt, table.shape[1] * page, table.shape[1], up(np.arange(0, groups * prompt + 1, prompt, dtype=np.int32)),
                        up(np.full(groups, prompt, np.int32)), fb)
        ctx.kv_write(c.handle, b, rows[0], 0, rows[1], 0)
        ctx.sync()
    ctx.upload(np.full(seqs, prompt, np.int32), lens)
    ctx.upload(np.zeros(seqs, np.int32), parent)
    ctx.kv_reorder([c.handle for c in caches], one, beams, parent)
    ctx.sync()
    history = [[list(p) for _ in range(beams)] for p in prompts]
    host_score, host_done = np.full((groups, beams), -np.inf, np.float32), np.zeros((groups, beams), np.int32)
    host_score[:, 0] = 0                                                           # the first step: one beam counts
    ctx.upload(host_score, score)

    def choose():
        ctx.beam_select(groups, beams, vocab, logits, 0, score, done, 3, beams, score, token, parent, done)
        ctx.kv_reorder([c.handle for c in caches], one, beams, parent)

    def write():
        for i, c in enumerate(caches):
            ctx.kv_write(c.handle, one, new[i][0], 0, new[i][1], 0)

    plans = []
    if recorded:
        for f in (choose, write):
            ctx.plan_begin()
            f()
            plans.append(ctx.plan_end())
    for step in range(steps):
        x = (rng.standard_normal((groups, beams, vocab)) * 2).astype(np.float16)
        x[..., 3] = 4 if step == 4 else -5                                          # some beams end
        ctx.upload(x, logits)
        ctx.plan_launch(plans[0]) if recorded else choose()
        ctx.sync()
        got = [ctx.download(b, (groups, beams), t) for b, t in ((score, np.float32), (token, np.int32), (parent, np.int32), (done, np.int32))]
        for g in range(groups):
            want, tok, par, near = br.best_continuations(x[g], host_score[g], host_done[g], 3, beams)
            assert near > 2.0 ** -19 and (tok >= 0).all()
            assert np.array_equal(got[1][g], tok) and np.array_equal(got[2][g], par), (step, g)
            assert np.allclose(got[0][g], want, rtol=2.0 ** -23, atol=2.0 ** -20)
            history[g] = [history[g][p] + [int(t)] for p, t in zip(par, tok)]
            host_done[g] = tok == 3
        host_score = got[0]
        assert np.array_equal(got[3], host_done)
        # the chosen tokens' rows behind the sequences
        for i in range(layers):
            for j in range(2):
                ctx.upload(words[i, j][got[1].reshape(-1)], new[i][j])
        ctx.upload(np.full(seqs, prompt + step + 1, np.int32), lens)
        ctx.plan_launch(plans[1]) if recorded else write()
        ctx.sync()
        now = ctx.download(tb, table.shape, np.int32)
        n = prompt + step + 1
        for i, c in enumerate(caches):
            k, v = _read_all(nnb, ctx, c, [n] * seqs, now)
            for j, rows in enumerate((k, v)):
                want = words[i, j][np.array(history).reshape(-1)]
                if fmt != "fp16":
                    codes, sc = ref.quantised(want, fmt)
                    want = (ref.code_values(codes, fmt) * sc.astype(np.float64)[..., None]).astype(np.float16)
                assert np.array_equal(rows.view(np.float16), want.reshape(rows.shape)), (step, i, j)      # (values: -0 reads back as 0 from int8)
    assert len({tuple(r) for r in now[:beams].tolist()}) == beams                   # each has pages of its own at the end
    for p in plans:
        ctx.L.nn_plan_free(p)
    for b in (tb, lens, starts, score, done, token, parent, logits, *sum(new, [])):
        ctx.free(b)
    for c in caches:
        c.close()


def test_two_recordings_of_a_context_take_turns(nnb, ctx):
    """Two recorded selections of other sizes share the context's workspace, with eager calls between them."""
    sets = []
    for groups, beams, vocab, picks in ((5, 3, 30011, 6), (40, 8, 700, 8)):
        x, score = draw(groups, beams, vocab, 81)
        lb, sb = ctx.upload(x), ctx.upload(score)
        outs = [ctx.alloc(groups * picks * 4) for _ in range(3)]
        call = lambda a=(groups, beams, vocab, lb, 0, sb, None, -1, picks, *outs, None): ctx.beam_select(*a)  # noqa: E731
        call()
        ctx.sync()
        want = [ctx.download(o, (groups, picks), np.int32) for o in outs]
        ctx.plan_begin()
        call()
        sets.append((call, ctx.plan_end(), outs, want, (lb, sb)))
    for turn in range(6):
        for call, plan, outs, want, _ in sets:
            for o in outs:
                ctx.L.nn_buf_fill(ctx.h, o, 0x55, want[0].nbytes)
            ctx.plan_launch(plan) if turn % 3 else call()
        ctx.sync()
        for _, _, outs, want, _ in sets:
            assert all(np.array_equal(ctx.download(o, w.shape, np.int32), w) for o, w in zip(outs, want)), turn
    for _, plan, outs, _, bufs in sets:
        ctx.L.nn_plan_free(plan)
        for b in (*outs, *bufs):
            ctx.free(b)


def test_contexts_side_by_side(nnb, ctx):
    """Two contexts of a GPU, each in a thread of its own: workspaces, streams and status words are each context's."""
    problems, results = [], {}

    def work(i):
        try:
            with nnb.Context(0) as c:
                x, score = draw(6, 4, 20001 + i, 90 + i)
                lb, sb, outs = c.upload(x), c.upload(score), [c.alloc(6 * 8 * 4) for _ in range(3)]
                cache = ref.Cache(nnb, c, "int8", [300, 120], 2, 64, 32, seed=91 + i)
                masks = [(2 << j) - 1 for j in range(20)] + [(2 << j) - 1 for j in range(9)]
                q, mb, o = c.upload(np.random.default_rng(i).standard_normal((29, 4, 64)).astype(np.float16)), c.upload(br.words_of(masks, 1)), c.alloc(29 * 4 * 64 * 2)
                b = cache.batch([20, 9])
                seen = set()
                for _ in range(30):
                    c.beam_select(6, 4, 20001 + i, lb, 0, sb, None, -1, 8, *outs, None)
                    c.attention_tree(cache.handle, b, 4, q, 0, o, 0, 0.125, 1, mb)
                    c.sync()
                    seen.add(tuple(c.download(x, (6, 8), np.int32).tobytes() for x in outs) + (c.download(o, (29, 4, 64), np.uint16).tobytes(),))
                results[i] = seen
                want = [br.best_continuations(x[g], score[g], None, -1, 8) for g in range(6)]
                got = c.download(outs[1], (6, 8), np.int32)
                assert all(np.array_equal(got[g], want[g][1]) for g in range(6))
                cache.close()
        except Exception as e:      # noqa: BLE001
            problems.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not problems, problems
    assert all(len(results[i]) == 1 for i in range(2))      # the same bits each time


def test_calls_are_counted_and_take_places_in_the_profile(nnb, built_lib, ctx):
    before = ctx.launch_count()
    b = nnb.KVBatch(0, 0, 0, 0, 0, None, None, None)
    assert ctx.L.nn_kv_move(ctx.h, None, 0, ctypes.byref(b), None) == 0
    assert ctx.L.nn_beam_select(ctx.h, 0, 4, 10, None, 0, None, None, -1, 4, None, None, None, None) == 0
    assert ctx.launch_count() == before                     # nothing to do, nothing launched
    x, score = draw(1, 2, 300, 99)
    lb, sb, outs = ctx.upload(x), ctx.upload(score), [ctx.alloc(16) for _ in range(3)]
    ctx.beam_select(1, 2, 300, lb, 0, sb, None, -1, 2, *outs, None)
    ctx.sync()
    assert ctx.launch_count() == before + 1
    for o in (lb, sb, *outs):
        ctx.free(o)
