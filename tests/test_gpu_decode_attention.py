"""The decode step with its attention: rotation, cache and attention between the projections, run together over several tokens, called one by one and recorded."""
import importlib

import numpy as np
import pytest

import kv_reference as ref
from helpers import check_close
from oracle import cpu

pytestmark = pytest.mark.gpu

SHAPE = ("tiny-attention", 576, 2, 576, 192, 1536, 4100)     # 9 query heads to 3 of the cache, 64 dims


def _step(ctx, M, seed=7, lengths=None, cache="int8", page=16, window=0, sinks=0, keep=False):
    synth, dstep = (importlib.import_module("adreno_llms_b200." + m) for m in ("synth", "decode_step"))
    lengths = lengths or [37, 0, 130][:M]
    return dstep.DecodeStep(ctx, synth.ModelShape(*SHAPE), "int8", M=M, n_sets=1, seed=seed, keep_host=keep, norm=True, chained=True,
                            attention=dict(lengths=lengths, cache=cache, page=page, window=window, sinks=sinks))


def _close(step):
    step.ctx.sync()
    step.attention.close()
    for st in step.sets:
        for w in st.values():
            w.release()


def _read(step):
    sh, M, c = step.shape, step.M, step.ctx
    return {n: c.download(b, (M, w), np.uint16).view(np.float16)
            for n, b, w in (("q", step.q, sh.q_dim), ("out", step.attention.out, sh.q_dim), ("resid", step.resid, sh.hidden), ("logits", step.logits, sh.vocab))}


def _check_last_layer(step, got, window, sinks):
    """What the last layer left behind, tightly: the new cells are what its k and v make, its output what the formula makes of its queries and its cache."""
    at, c, M, D, page = step.attention, step.ctx, step.M, 64, 16
    fmt = at.cache
    pages = at.table.size
    held = {}
    for name, cells, scales, rows in (("k", 0, 2, step.k), ("v", 1, 3, step.v)):
        bufs = at.buffers[-1]
        new = c.download(rows, (M, 3, D), np.uint16).view(np.float16)
        if name == "k":
            new = ref.rotated(new, at.cos_host[at.lengths], at.sin_host[at.lengths], D)
        codes = c.download(bufs[cells], (pages, 3, page, D), np.uint16 if fmt == "fp16" else np.uint8)
        scale = None if fmt == "fp16" else c.download(bufs[scales], (pages, 3, page), np.float16)
        want = (new.view(np.uint16), None) if fmt == "fp16" else ref.quantised(new, fmt)
        for s, p in enumerate(at.lengths):
            cell = at.table[s, p // page], slice(None), p % page
            assert np.array_equal(codes[cell], want[0][s]) and (scale is None or np.array_equal(scale[cell], want[1][s]))
            where = np.arange(p + 1)
            row = at.table[s, where // page], slice(None), where % page
            held[name, s] = codes[row].view(np.float16).astype(np.float64) if fmt == "fp16" else ref.code_values(codes[row], fmt) * scale[row].astype(np.float64)[..., None]
    for s, p in enumerate(at.lengths):
        for head in range(9):
            want, spread, most, steep = ref.attend(got["q"][s].reshape(9, 1, D)[head].astype(np.float64), held["k", s][:, head // 3], held["v", s][:, head // 3], [p], D ** -0.5,
                                                   window, sinks)
            have = got["out"][s].reshape(9, D)[head]
            assert (np.abs(have - want[0]) <= ref.attention_bound(want, spread, most, steep, p + 1, D)[0]).all(), (s, head)


@pytest.mark.parametrize("M", [1, 3])
@pytest.mark.parametrize("cache,window,sinks", [("fp16", 0, 0), ("int8", 0, 0), ("fp8", 0, 0), ("int8", 20, 4)])
def test_steps_follow_a_plain_chain(nnb, ctx, cache, window, sinks, M):
    """Four tokens of each sequence: a host chain of plain operators keeps its own cache beside the device's."""
    step = _step(ctx, M, cache=cache, window=window, sinks=sinks, keep=True)
    at, h, D = step.attention, step.host, 64
    starts = np.concatenate([[0], np.cumsum(at.lengths)])
    held = [[[h[f"cache.{layer}"][i][starts[s]:starts[s + 1]].reshape(-1, 3, D) for s in range(M)] if f"cache.{layer}" in h else [np.zeros((0, 3, D), np.float16)] * M
             for i in range(2)] for layer in range(2)]

    def seen(rows):
        if cache == "fp16":
            return rows.astype(np.float64)
        codes, scale = ref.quantised(rows, cache)
        return ref.code_values(codes, cache) * scale.astype(np.float64)[..., None]

    for token in range(4):
        if token == 2:
            step.record()
        step.reset_residual()
        step.enqueue(0) if token < 2 else step.launch(0)
        ctx.sync()
        got = _read(step)
        r, pos = step.resid0.copy(), at.lengths
        for layer in range(2):
            x = cpu.rmsnorm(r, h["gamma"], step.eps)
            q, k, v = (cpu.linear("int8", x, *h[f"qkv.{layer}.{j}"]).reshape(M, -1, D) for j in range(3))
            q, k = (ref.rotated(t, at.cos_host[pos], at.sin_host[pos], D) for t in (q, k))
            out = np.zeros((M, 9, D))
            for s in range(M):
                for i, new in ((0, k), (1, v)):
                    held[layer][i][s] = np.concatenate([held[layer][i][s], new[s:s + 1]])
                ks, vs = seen(held[layer][0][s]), seen(held[layer][1][s])
                for head in range(9):
                    out[s, head] = ref.attend(q[s:s + 1, head].astype(np.float64), ks[:, head // 3], vs[:, head // 3], [pos[s]], D ** -0.5, window, sinks)[0]
            out = out.astype(np.float16).reshape(M, -1)
            r = cpu.linear_residual("int8", out, *h[f"o_add.{layer}.0"], r)
            act = cpu.linear_swiglu("int8", cpu.rmsnorm(r, h["gamma"], step.eps), *h[f"gate_up.{layer}.0"], *h[f"gate_up.{layer}.1"])
            r = cpu.linear_residual("int8", act, *h[f"down_add.{layer}.0"], r)
        logits = cpu.linear("int8", r, *h["lm_head.-1.0"])
        what = f"{cache} M{M} token {token}"
        # The chain's own tolerances, 3e-3 of a value.  Codes add to them: a difference d of two values moves them to different codes, a step s apart,
        # with the probability d / s, which is an error of sqrt(s d) in the mean square.  s of a row of 64 normal values is 3 / 127 of their
        # deviation (int8) or on average 0.09 of a value (e4m3, 2^-4 to 2^-3): with d = 3e-3 sqrt(s d) is 8.4e-3 and 1.65e-2.
        more = {"fp16": 0.0, "int8": 8.4e-3, "fp8": 1.65e-2}[cache]
        for name, want, tol in (("q", q.reshape(M, -1), 3e-3 + more), ("out", out, 3e-3 + more), ("resid", r, 2e-3 + more), ("logits", logits, 3e-3 + more)):
            check_close(got[name], want, tol=tol, what=f"{name} {what}")
        _check_last_layer(step, got, window, sinks)
        at.advance()
    _close(step)


@pytest.mark.parametrize("M,cache", [(1, "int8"), (3, "fp16")])
def test_a_recording_takes_new_lengths_and_pages(nnb, ctx, M, cache):
    """One recording replayed while lengths grow and pages are moved gives the bits of calls made one by one; two recordings of a context take turns with
    their shared workspace."""
    lengths = [700, 15, 64][:M]
    eager, first, second = (_step(ctx, M, cache=cache, lengths=lengths) for _ in range(3))
    for s in (first, second):
        s.record()
    for token in range(6):
        for s in (eager, first, second):
            s.reset_residual()
        eager.enqueue(0)
        want = _read(eager)
        for s in (first, second):
            s.launch(0)
        for s in (first, second):
            got = _read(s)
            for name in want:
                assert np.array_equal(got[name].view(np.uint16), want[name].view(np.uint16)), (name, token)
        assert np.isfinite(want["logits"]).all()
        for s in (eager, first, second):
            s.attention.advance()
        if token == 2:      # a page of the first sequence is moved in one of them: both buffers, scales too, and the table
            at = first.attention
            page, row = 16, 3 * 64 * (2 if cache == "fp16" else 1)
            old, new = int(at.table[0, 1]), int(at.table[0, -1])     # (its last page has not been reached)
            for bufs in at.buffers:
                for b, size in zip(bufs, [page * row] * 2 + [page * 3 * 2] * 2):
                    if b:
                        ctx.upload(ctx.download(b, (size,), np.uint8, offset=old * size), b + new * size)
                        ctx.upload(np.full(size, 0x7E if cache == "fp16" else 0xFF, np.uint8), b + old * size)
            at.table[0, 1], at.table[0, -1] = new, old
            ctx.upload(at.table, at.table_dev)
    for s in (eager, first, second):
        _close(s)


def test_attention_needs_a_chained_step(nnb, ctx):
    synth, dstep = (importlib.import_module("adreno_llms_b200." + m) for m in ("synth", "decode_step"))
    with pytest.raises(ValueError):
        dstep.DecodeStep(ctx, synth.ModelShape(*SHAPE), "int8", attention=dict(lengths=[4]))
