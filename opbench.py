"""Time one operator on one GPU:  python opbench.py --fmt q4 --n 28672 --k 8192 --m 1
                                python opbench.py --op attention --cache int8 --seqs 16 --new 1 --len 4096 --heads 16 --kv-heads 8 --dim 64
                                python opbench.py --op attention_tree --cache fp8 --seqs 8 --new 64 --len 8192 --heads 32 --kv-heads 8 --dim 128
                                python opbench.py --op beam_select --seqs 64 --beams 8 --picks 16 --vocab 151936

Prints one JSON line: microseconds per launch (CUDA events around `reps` back-to-back launches
that rotate through enough weight copies to exceed L2), algorithmic GB/s and TFLOP/s.  Weights are
seeded synthetic tensors quantised the way the offline tools of the reference do it.  With
--reps 1..4 and --copies 1 it is also a small, self-ending command to put under a profiler.
"""
import argparse
import importlib
import importlib.util
import json
import os
import sys

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
PKG = os.path.join(HERE, "adreno-llms_b200")


def load_pkg():
    name = "adreno_llms_b200"
    if name in sys.modules:
        return sys.modules[name]
    spec = importlib.util.spec_from_file_location(name, os.path.join(PKG, "__init__.py"), submodule_search_locations=[PKG])
    mod = importlib.util.module_from_spec(spec)
    sys.modules[name] = mod
    spec.loader.exec_module(mod)
    return mod


def cache_op(pkg, ctx, args, l2, rng):
    """One call on a paged cache, rotating through enough caches to exceed the L2."""
    S, n, ln, hq, hk, D, P = args.seqs, args.new, args.len, args.heads, args.kv_heads, args.dim, args.page
    per_seq, eb, scaled = -(-ln // P), 2 if args.cache == "fp16" else 1, args.cache != "fp16"
    cells = S * per_seq * P * hk
    nbytes = 2 * cells * (D * eb + (2 if scaled else 0))
    copies = args.copies if args.copies > 0 else int(max(1, min(64, -(-2 * l2 // nbytes) + 1)))
    table = ctx.upload(rng.permutation(S * per_seq).astype(np.int32))
    up = lambda a: ctx.upload(np.ascontiguousarray(a))  # noqa: E731
    lens = up(np.full(S, ln, np.int32))
    batch = lambda m: pkg.KVBatch(S, S * m, m, ln, per_seq, up(np.arange(0, S * m + 1, m, dtype=np.int32)), lens, table)  # noqa: E731
    full, b = batch(ln), batch(n)
    rows = [up(np.tile(rng.standard_normal((min(S * ln, 4096), hk * D)).astype(np.float16), (-(-S * ln // 4096), 1))[:S * ln].view(np.uint16)) for _ in range(2)]
    caches = []
    for _ in range(copies):
        bufs = [ctx.alloc(cells * D * eb) for _ in range(2)] + ([ctx.alloc(cells * 2) for _ in range(2)] if scaled else [None, None])
        caches.append(ctx.kv_cache(args.cache, S * per_seq, P, hk, D, *bufs))
        ctx.kv_write(caches[-1], full, rows[0], 0, rows[1], 0)
    q = up(rng.standard_normal((S * n, hq * D)).astype(np.float16).view(np.uint16))
    out = ctx.alloc(S * n * hq * D * 2)
    angle = np.arange(ln)[:, None] * 10000.0 ** (-np.arange(0, D, 2) / D)
    cos, sin = up(np.cos(angle).astype(np.float32)), up(np.sin(angle).astype(np.float32))
    seen = [min(p + 1, args.window) + min(args.sinks, max(0, p + 1 - args.window)) if args.window else p + 1 for p in range(ln - n, ln)]
    keys = min(ln, args.window + n - 1 + args.sinks) if args.window else ln
    cell_row = D * eb + (2 if scaled else 0)
    # drafted trees of two branches to a token; rows that move up over as many others; beams of which the odd ones take over their neighbours' sequences
    tree = [(1 << j) | (1 << j // 2) | 1 for j in range(n)] if args.op == "attention_tree" else []
    words = -(-n // 32)
    mask = up(np.tile(np.array([[m >> 32 * w & 0xFFFFFFFF for w in range(words)] for m in tree], np.uint32).reshape(-1), S)) if tree else None
    source = up(np.tile(np.arange(ln - n, ln, dtype=np.int32), S))
    parent = up((np.arange(S, dtype=np.int32) % args.beams) & ~1)
    if args.op == "kv_move":
        b.kv_len = up(np.full(S, max(n, ln - n), np.int32))

    def run(i):
        c = caches[i % copies]
        if args.op == "attention":
            ctx.attention(c, b, hq, q, 0, out, 0, D ** -0.5, args.window, args.sinks)
        elif args.op == "attention_tree":
            ctx.attention_tree(c, b, hq, q, 0, out, 0, D ** -0.5, words, mask)
        elif args.op == "kv_move":
            ctx.kv_move([c], b, source)
        elif args.op == "kv_reorder":
            ctx.kv_reorder([c], b, args.beams, parent)
        elif args.op == "kv_write":
            ctx.rope_kv_write(c, b, cos, sin, ln, D, hq, q, 0, out, 0, rows[0], 0, rows[1], 0)
        else:
            ctx.kv_read(c, b, rows[0], 0, rows[1], 0)

    for i in range(args.warmup):
        run(i)
    e0, e1 = ctx.event(), ctx.event()
    ctx.sync()
    l0 = ctx.launch_count()
    ctx.record(e0)
    for i in range(args.reps):
        run(i)
    ctx.record(e1)
    us = ctx.elapsed_ms(e0, e1) * 1e3 / args.reps
    ctx.sync()
    moved = {"attention": S * 2 * hk * keys * cell_row + 4 * S * n * hq * D, "kv_write": S * n * (2 * hk * (cell_row + 2 * D) + 4 * hq * D + 4 * D),
             "kv_read": S * n * 2 * hk * (cell_row + 2 * D), "attention_tree": S * 2 * hk * ln * cell_row + 4 * S * n * hq * D,
             "kv_move": S * n * 4 * hk * cell_row, "kv_reorder": (S // 2) * (8 * (ln // P) + (ln % P) * 4 * hk * cell_row)}[args.op]
    flops = 4.0 * S * hq * D * sum(seen) if args.op == "attention" else 4.0 * S * hq * D * n * (ln - n + 1) if args.op == "attention_tree" else 0.0
    print(json.dumps({"op": args.op, "cache": args.cache, "seqs": S, "new": n, "len": ln, "heads": hq, "kv_heads": hk, "dim": D, "page": P, "window": args.window,
                      "sinks": args.sinks, "us_per_call": round(us, 3), "algorithmic_bytes": moved, "gbps": round(moved / (us * 1e-6) / 1e9, 1),
                      "tflops": round(flops / (us * 1e-6) / 1e12, 2), "kernels_per_call": (ctx.launch_count() - l0) / args.reps, "caches": copies}), flush=True)
    for c in caches:
        c.close()
    ctx.close()
    return 0


def beam_op(ctx, args, l2, rng):
    """The selection of each group's best continuations, rotating through enough logits to exceed the L2."""
    G, B, V, n = args.seqs, args.beams, args.vocab, args.picks
    nbytes = 2 * G * B * V
    copies = args.copies if args.copies > 0 else int(max(1, min(64, -(-2 * l2 // nbytes) + 1)))
    logits = [ctx.upload((rng.standard_normal((G * B, V)) * 2.5).astype(np.float16)) for _ in range(copies)]
    score = ctx.upload(-np.cumsum(rng.random((G, B)), axis=1).astype(np.float32))
    outs = [ctx.alloc(4 * G * n) for _ in range(3)]

    def run(i):
        ctx.beam_select(G, B, V, logits[i % copies], 0, score, None, -1, n, *outs, None)

    for i in range(args.warmup):
        run(i)
    e0, e1 = ctx.event(), ctx.event()
    ctx.sync()
    ctx.record(e0)
    for i in range(args.reps):
        run(i)
    ctx.record(e1)
    us = ctx.elapsed_ms(e0, e1) * 1e3 / args.reps
    ctx.sync()
    print(json.dumps({"op": args.op, "groups": G, "beams": B, "vocab": V, "picks": n, "us_per_call": round(us, 3), "algorithmic_bytes": nbytes,
                      "gbps": round(nbytes / (us * 1e-6) / 1e9, 1), "copies": copies}), flush=True)
    ctx.close()
    return 0


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--fmt", default="int8", choices=["fp16", "int8", "q4"])
    ap.add_argument("--n", type=int, default=151936)
    ap.add_argument("--k", type=int, default=896)
    ap.add_argument("--m", type=int, default=1)
    ap.add_argument("--op", default="linear", choices=["linear", "add", "swiglu", "kv_write", "kv_read", "attention", "attention_tree", "kv_move", "kv_reorder", "beam_select"])
    ap.add_argument("--cache", default="fp16", choices=["fp16", "int8", "fp8"], help="cells of the key/value cache")
    ap.add_argument("--seqs", type=int, default=1, help="sequences (kv_reorder: all beams of all groups; beam_select: groups)")
    ap.add_argument("--beams", type=int, default=4)
    ap.add_argument("--picks", type=int, default=4)
    ap.add_argument("--vocab", type=int, default=49152)
    ap.add_argument("--new", type=int, default=1, help="new tokens of each sequence")
    ap.add_argument("--len", type=int, default=4096, help="positions of each sequence, the new tokens included")
    ap.add_argument("--heads", type=int, default=16)
    ap.add_argument("--kv-heads", type=int, default=8)
    ap.add_argument("--dim", type=int, default=64, choices=[64, 128])
    ap.add_argument("--page", type=int, default=64)
    ap.add_argument("--window", type=int, default=0)
    ap.add_argument("--sinks", type=int, default=0)
    ap.add_argument("--reps", type=int, default=200)
    ap.add_argument("--warmup", type=int, default=5)
    ap.add_argument("--copies", type=int, default=0, help="resident weight copies (0: enough to exceed twice the L2)")
    ap.add_argument("--device", type=int, default=0)
    args = ap.parse_args()
    pkg = load_pkg()
    synth = importlib.import_module("adreno_llms_b200.synth")
    ctx = pkg.Context(args.device)
    _, l2, _ = ctx.device_info()
    rng = np.random.default_rng(1)
    if args.op == "beam_select":
        return beam_op(ctx, args, l2, rng)
    if args.op in ("kv_write", "kv_read", "attention", "attention_tree", "kv_move", "kv_reorder"):
        return cache_op(pkg, ctx, args, l2, rng)
    fmt, N, K, M = args.fmt, args.n, args.k, args.m
    blk = min(N, 2048)   # timing does not depend on the values: quantise a block of rows and repeat it
    W, s = synth.weight(fmt, blk, K, rng)
    rep = (N + blk - 1) // blk
    W = np.tile(W, (rep, 1))[:N]
    if s is not None:
        s = np.tile(s, (rep, 1) if s.ndim == 2 else rep)[:N]
    nbytes = W.nbytes + (0 if s is None else s.nbytes)
    nw = 2 if args.op == "swiglu" else 1
    copies = args.copies if args.copies > 0 else int(max(2, min(256, -(-2 * l2 // (nbytes * nw)) + 1)))
    ws = [[pkg.QuantWeight(ctx, fmt, W, s) for _ in range(nw)] for _ in range(copies)]
    x = ctx.upload(synth.activations(M, K, rng).view(np.uint16))
    out = ctx.upload(synth.activations(M, N, rng).view(np.uint16))

    def run(i):
        w = ws[i % copies]
        if args.op == "linear":
            ctx.linear(M, N, K, x, w[0].buf, out)
        elif args.op == "add":
            ctx.linear_add(M, N, K, x, w[0].buf, out)
        else:
            ctx.fused_gate_up_silu(M, N, K, x, w[0].buf, w[1].buf, out)

    for i in range(args.warmup):
        run(i)
    a, b = ctx.event(), ctx.event()
    ctx.sync()
    l0 = ctx.launch_count()
    ctx.record(a)
    for i in range(args.reps):
        run(i)
    ctx.record(b)
    ms = ctx.elapsed_ms(a, b)
    us = ms * 1e3 / args.reps
    algo = nw * synth.linear_bytes(fmt, N, K, M) - (nw - 1) * (2 * M * K + 2 * M * N)
    print(json.dumps({"op": args.op, "fmt": fmt, "N": N, "K": K, "M": M, "us_per_launch": round(us, 3),
                      "algorithmic_bytes": algo, "gbps": round(algo / (us * 1e-6) / 1e9, 1),
                      "tflops": round(2.0 * nw * M * N * K / (us * 1e-6) / 1e12, 2),
                      "kernels_per_call": (ctx.launch_count() - l0) / args.reps, "weight_copies": copies}), flush=True)
    ctx.close()
    return 0


if __name__ == "__main__":
    sys.exit(main())
