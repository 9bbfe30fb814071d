"""Several continuations of a sequence over the paged key/value cache, as timed cases: drafted tokens that form a tree, and beams.

  draft    nn_tree_layout and nn_rope_kv_write_at: from the drafted tokens' parents, which of them each one sees and its position; queries and keys
           are rotated to these positions, keys and values go into the cache.  A cache of 8 bits is read back with nn_kv_read.
  tree     nn_attention_tree: each drafted token attends to the sequence before the draft, to its ancestors and to itself.
  move     nn_kv_move: cells of all layers go to earlier positions of their sequences: those of a draft's accepted path behind the sequence, or those
           behind turns of a conversation that are dropped.
  select   nn_beam_select: the best continuations of each group of beams, from the logits of every beam and the beams' scores.
  reorder  nn_kv_reorder: every beam takes over its parent's sequence in the caches of all layers: the page table's entries of full pages, and the
           cells of the page that is not full.

A cache's pages are [page][kv head][slot][dim], their scales [page][kv head][slot] in fp16; here those of all layers are one tensor.  `run` computes the
operators in their plain form (elementary torch operations in 32 bits, the beams' scores in 64) where `own` is false, and calls the library where it
is true.
"""
import importlib.util
import math
import os
import random
import sys

import torch

own = False

CELL_BYTES = {"fp16": 2, "int8": 1, "fp8": 1}    # bytes of a cell
CODES = {"int8": 127.0, "fp8": 448.0}              # the largest code
ROPE_BASE = 10000.0


def listed():
    return [
        # a small tree for one user of the 135M shape: latency
        dict(name="draft_135m_int8_1x26", op="draft", fmt="int8", seqs=1, new=26, len=700, q_heads=9, kv_heads=3, dim=64, page=16),
        # trees of many users, ragged, into an 8-bit cache
        dict(name="draft_fp8_64x64", op="draft", fmt="fp8", seqs=64, new=64, len=2048, q_heads=32, kv_heads=8, dim=128, page=64),
        # the same small tree over the sequence: latency
        dict(name="tree_135m_int8_1x26", op="tree", fmt="int8", seqs=1, new=26, len=700, q_heads=9, kv_heads=3, dim=64, page=16),
        # trees of a few users, fp16, heads in groups of 7
        dict(name="tree_500m_fp16_8x15", op="tree", fmt="fp16", seqs=8, new=15, len=4096, q_heads=14, kv_heads=2, dim=64, page=64),
        # a serving batch: trees of 64 tokens over an 8-bit cache
        dict(name="tree_fp8_32x64_8k", op="tree", fmt="fp8", seqs=32, new=64, len=8192, q_heads=32, kv_heads=8, dim=128, page=64),
        # an accepted path of one user, all layers: latency
        dict(name="move_135m_int8_5", op="move", fmt="int8", kind="accept", seqs=1, new=5, tree=26, len=700, kv_heads=3, dim=64, page=16, layers=30),
        # the oldest turns of 8 conversations go, all layers
        dict(name="move_500m_fp16_8x2048", op="move", fmt="fp16", kind="drop", seqs=8, new=2048, tree=0, len=5000, kv_heads=2, dim=64, page=64, layers=24),
        # four beams of one user: latency
        dict(name="select_135m_1x4", op="select", groups=1, beams=4, vocab=49152, picks=8, pad=0, done=False),
        # eight users, some of whose beams have ended; an odd vocabulary in padded rows
        dict(name="select_8x5_odd", op="select", groups=8, beams=5, vocab=65535, picks=5, pad=65, done=True),
        # a serving batch with the largest vocabulary
        dict(name="select_500m_64x8", op="select", groups=64, beams=8, vocab=151936, picks=16, pad=0, done=False),
        # four beams of one user, all layers: latency
        dict(name="reorder_135m_int8_1x4", op="reorder", fmt="int8", groups=1, beams=4, len=700, kv_heads=3, dim=64, page=16, layers=30),
        # a serving batch, all layers
        dict(name="reorder_500m_fp16_16x8", op="reorder", fmt="fp16", groups=16, beams=8, len=2000, kv_heads=2, dim=64, page=128, layers=24),
    ]


def _log_uniform(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


MOST_POOL = 24 * 16 * (2000 // 128 + 1 + 3 * 8) * 128 * 2 * 64   # values of keys of all beams' pages in all layers, as the largest listed reorder has


def _within(c):
    """Whether a case costs no more than the largest listed one of its operator."""
    most = [work(x) for x in listed() if x["op"] == c["op"]]
    if c["op"] == "reorder" and c["layers"] * c["groups"] * (c["len"] // c["page"] + 1 + 3 * c["beams"]) * c["page"] * c["kv_heads"] * c["dim"] > MOST_POOL:
        return False
    return all(work(c)[k] <= max(w[k] for w in most) for k in ("bytes", "flops"))


def _shrunk(c, keys):
    """The case with its largest of these numbers halved, until it is within the range."""
    while not _within(c):
        key = max(keys, key=lambda k: c[k] / (64 if k == "new" else 1))
        key = key if c[key] > 1 else "len"
        c[key] = (c[key] + 1) // 2
        if "tree" in c:
            c["len"] = max(c["len"], c["tree"], 2 * c["new"])
    return c


def draw(rng):
    op = rng.choice(("draft", "tree", "tree", "tree", "move", "select", "select", "reorder"))
    if op == "select":
        beams = rng.randint(1, 16)
        return _shrunk(dict(op=op, groups=int(_log_uniform(rng, 1, 65)), beams=beams, vocab=int(_log_uniform(rng, 100, 151937)), picks=rng.choice((beams, 2 * beams)),
                            pad=rng.choice((0, 0, 1, 13)), done=rng.random() < 0.4), ("groups",))
    c = dict(op=op, fmt=rng.choice(("fp16", "int8", "fp8")), kv_heads=rng.randint(1, 8), dim=rng.choice((64, 64, 128)), page=rng.choice((16, 32, 64, 128, 256)))
    if op == "reorder":
        c.update(groups=int(_log_uniform(rng, 1, 17)), beams=rng.randint(2, 16), len=int(_log_uniform(rng, 16, 4097)), layers=int(_log_uniform(rng, 1, 33)))
        return _shrunk(c, ("groups", "layers"))
    c["seqs"] = int(_log_uniform(rng, 1, 65)) if rng.random() < 0.6 else 1
    if op == "move":
        c.update(kind=rng.choice(("accept", "drop")), layers=int(_log_uniform(rng, 1, 33)))
        c["new"] = rng.randint(1, 16) if c["kind"] == "accept" else int(_log_uniform(rng, 16, 2049))
        c["tree"] = c["new"] * rng.randint(2, 8) if c["kind"] == "accept" else 0
        c["len"] = (c["tree"] if c["tree"] else 2 * c["new"]) + int(_log_uniform(rng, 1, 1025))
        return _shrunk(c, ("seqs", "layers"))
    c["q_heads"] = c["kv_heads"] * rng.choice((1, 2, 3, 4, 7, 8))
    c["new"] = int(_log_uniform(rng, 1, 65)) if rng.random() < 0.85 else int(_log_uniform(rng, 64, 300))
    c["len"] = c["new"] + int(_log_uniform(rng, 1, 32768 if op == "tree" else 4096))
    return _shrunk(c, ("seqs", "new"))


def _lengths(c):
    """[(new tokens, length)] of the sequences: one as the case says, several ragged, down to half of it."""
    if c["seqs"] == 1:
        return [(c["new"], c["len"])]
    got = []
    for i in range(c["seqs"]):
        new = max(1, c["new"] - (i * 104729) % (c["new"] // 2 + 1)) if c["new"] > 16 else c["new"]
        got.append((new, max(c["len"] - (i * 7919) % (c["len"] // 2 + 1), 2 * new if c.get("kind") == "drop" else max(new, c.get("tree", 0)))))
    return got


def _beam_lengths(c):
    """Positions of each group's beams."""
    return [max(1, c["len"] - (i * 7919) % (c["len"] // 2 + 1)) for i in range(c["groups"])]


def _parents_of_beams(c, i):
    """Group i's: some beams stay, the others go on from one of them.  (What a beam that stays holds does not change, so that a second pass changes nothing.)"""
    rng = random.Random(1000 * i + c["beams"])
    stay = rng.sample(range(c["beams"]), rng.randint(1, c["beams"] - 1))
    return [b if b in stay else rng.choice(stay) for b in range(c["beams"])]


def work(case):
    c = case
    if c["op"] == "select":
        rows = c["groups"] * c["beams"]
        return {"bytes": rows * (2 * c["vocab"] + 4 + (4 if c["done"] else 0)) + c["groups"] * c["picks"] * (12 + (4 if c["done"] else 0)), "flops": 3.0 * rows * c["vocab"]}
    D, hk, cell, scale = c["dim"], c["kv_heads"], CELL_BYTES[c["fmt"]], 0 if c["fmt"] == "fp16" else 2
    cells = 2 * hk * (D * cell + scale)                       # of a position of a layer, keys and values
    if c["op"] == "reorder":
        b = 0
        for i, n in enumerate(_beam_lengths(c)):
            moved = [(x, p) for x, p in enumerate(_parents_of_beams(c, i)) if x != p]
            b += 8 * len(moved) * (n // c["page"]) + (len(moved) + len({p for _, p in moved})) * (n % c["page"]) * cells * c["layers"] + 4 * 2 * c["beams"]
        return {"bytes": b, "flops": 0}
    rows = sum(n for n, _ in _lengths(c))
    if c["op"] == "move":
        return {"bytes": rows * (2 * cells * c["layers"] + 4) + 4 * (2 * c["seqs"] + 1) + sum(8 * (-(-n // c["page"])) for n, _ in _lengths(c)), "flops": 0}
    meta = 4 * (2 * c["seqs"] + 1) + sum(4 * (-(-n // c["page"])) for _, n in _lengths(c)) + rows * 4 * (-(-c["new"] // 32))
    hq = c["q_heads"]
    if c["op"] == "draft":
        b = rows * (2 * D * (2 * hq + 2 * hk) + cells) + rows * 2 * D * 4 // 2 + rows * 8
        if scale:
            b += rows * (cells + 2 * 2 * hk * D)              # read back
        return {"bytes": b + meta, "flops": 3.0 * rows * D * (hq + hk)}
    pairs = sum(n * (length - n) + n for n, length in _lengths(c))   # (the sequence before the draft, and each token itself)
    return {"bytes": sum(length for _, length in _lengths(c)) * cells + rows * 2 * 2 * hq * D + meta, "flops": 4.0 * D * hq * pairs}


# ---- the library ---------------------------------------------------------------------------------
def _package():
    name = "adreno_llms_b200"
    if name not in sys.modules:
        path = os.path.join(os.getcwd(), "adreno-llms_b200", "__init__.py")
        spec = importlib.util.spec_from_file_location(name, path, submodule_search_locations=[os.path.dirname(path)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    return sys.modules[name]


_context = None


def _ctx():
    """The process's one context, as a serving program keeps it."""
    global _context
    if _context is None:
        torch.cuda.init()
        _context = _package().Context(torch.cuda.current_device())
    return _context


def _p(t):
    return None if t is None else t.data_ptr()


class _State:
    handles = ()

    def __del__(self):
        for h in self.handles:
            h.close()


# ---- inputs ----------------------------------------------------------------------------------------
def _fill(fmt, codes, scales, gen):
    """Every cell of a cache from N(0, 1) rows, by the cache's own rule, some pages at a time."""
    codes, scales = codes.flatten(0, 1), None if scales is None else scales.flatten(0, 1)
    pages, H, P, D = codes.shape
    step = max(1, (1 << 26) // (H * P * D))
    for a in range(0, pages, step):
        n = min(step, pages - a)
        x = torch.randn((n, H, P, D), generator=gen, device="cuda", dtype=torch.float16)
        if fmt == "fp16":
            codes[a:a + n] = x
        else:
            codes[a:a + n], scales[a:a + n] = _quantise(x, fmt)


def _make_caches(s, pages, layers, gen):
    """Keys, values and scales of all layers, and with the library a handle for each layer."""
    c = s.case
    D, hk, P, fmt = c["dim"], c["kv_heads"], c["page"], c["fmt"]
    cells = {"fp16": torch.float16, "int8": torch.int8, "fp8": torch.float8_e4m3fn}[fmt]
    s.k, s.v = (torch.zeros((layers, pages, hk, P, D), dtype=cells, device="cuda") for _ in range(2))
    s.k_scale = s.v_scale = None
    if fmt != "fp16":
        s.k_scale, s.v_scale = (torch.zeros((layers, pages, hk, P), dtype=torch.float16, device="cuda") for _ in range(2))
    _fill(fmt, s.k, s.k_scale, gen)
    _fill(fmt, s.v, s.v_scale, gen)
    if own:
        s.handles = [_ctx().kv_cache(fmt, pages, P, hk, D, *(_p(None if t is None else t[i]) for t in (s.k, s.v, s.k_scale, s.v_scale))) for i in range(layers)]


def _make_batch(s, rows, most, row_start):
    s.batch = None
    if own:   # the batch's description, which a serving program keeps
        s.batch = _package().KVBatch(s.table.shape[0], rows, most, s.table.shape[1] * s.case["page"], s.table.shape[1], _p(row_start), _p(s.kv_len), _p(s.table))


def _prepare_select(s, gen):
    c = s.case
    rows = c["groups"] * c["beams"]
    s.logits = (2.5 * torch.randn((rows, c["vocab"] + c["pad"]), generator=gen, device="cuda")).half()
    s.score = -torch.rand((c["groups"], c["beams"]), generator=gen, device="cuda").cumsum(1)
    s.done = s.out_done = None
    s.eos = -1
    if c["done"]:
        s.eos = 2
        s.done = (torch.rand((c["groups"], c["beams"]), generator=gen, device="cuda") < 0.3).int()
        s.out_done = torch.zeros((c["groups"], c["picks"]), dtype=torch.int32, device="cuda")
    s.out_score = torch.zeros((c["groups"], c["picks"]), device="cuda")
    s.token, s.parent = (torch.zeros((c["groups"], c["picks"]), dtype=torch.int32, device="cuda") for _ in range(2))


def _prepare_reorder(s, gen):
    """A group's beams share the pages of their prompt; behind it each has three pages of its own, of which the last but one is not full."""
    c = s.case
    G, B, P = c["groups"], c["beams"], c["page"]
    lengths = _beam_lengths(c)
    full = [n // P for n in lengths]
    width = max(full) + 2
    pages = sum(max(0, f - 1) for f in full) + 3 * G * B
    order = torch.randperm(pages, generator=gen, device="cuda").tolist()
    table = torch.full((G * B, width), -1, dtype=torch.int32)
    for i, f in enumerate(full):
        shared = [order.pop() for _ in range(max(0, f - 1))]
        for b in range(B):
            table[i * B + b, :f + 2] = torch.tensor((shared + [order.pop() for _ in range(3)])[-(f + 2):], dtype=torch.int32)
    s.table = table.cuda()
    s.kv_len = torch.tensor([n for n in lengths for _ in range(B)], dtype=torch.int32, device="cuda")
    s.parent = torch.tensor([p for i in range(G) for p in _parents_of_beams(c, i)], dtype=torch.int32, device="cuda")
    _make_caches(s, pages, c["layers"], gen)
    _make_batch(s, 0, 0, None)


def _tree(n, rng):
    """Parents of n drafted tokens: each goes on from one of the eight before it, or begins at the sequence's end."""
    return [-1 if i == 0 or rng.random() < 0.1 else rng.randrange(max(0, i - 8), i) for i in range(n)]


def _prepare_rows(s, gen, seed):
    """What draft, tree and move share: sequences with their pages anywhere."""
    c = s.case
    D, hk, P, op = c["dim"], c["kv_heads"], c["page"], c["op"]
    lengths = _lengths(c)
    need = [-(-length // P) for _, length in lengths]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=gen, device="cuda").tolist()
    table = torch.full((len(lengths), max(need)), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    starts = [0]
    for n, _ in lengths:
        starts.append(starts[-1] + n)
    rng = random.Random(seed)
    s.rows, s.new, s.len = starts[-1], max(n for n, _ in lengths), max(length for _, length in lengths)
    s.table = table.cuda()
    s.row_start = torch.tensor(starts, dtype=torch.int32, device="cuda")
    ends = [length for _, length in lengths]
    if op == "move":   # rows come from further on: the first of an accepted path from its own place already, a dropped part's successors from behind it
        source = []
        ends = []
        for n, length in lengths:
            if c["kind"] == "drop":
                source += range(length - n, length)
                ends.append(rng.randint(n, length - n))
            else:
                base = length - c["tree"]
                source += [base] + sorted(rng.sample(range(base + n, length), n - 1))
                ends.append(base + n)
        s.source = torch.tensor(source, dtype=torch.int32, device="cuda")
    s.kv_len = torch.tensor(ends, dtype=torch.int32, device="cuda")
    _make_caches(s, pages, c.get("layers", 1), gen)
    _make_batch(s, s.rows, s.new, s.row_start)
    if op == "move":
        return
    hq = c["q_heads"]
    rows = lambda heads: torch.randn((s.rows, heads, D), generator=gen, device="cuda", dtype=torch.float16)  # noqa: E731
    empty = lambda heads: torch.zeros((s.rows, heads, D), device="cuda", dtype=torch.float16)  # noqa: E731
    s.words = -(-s.new // 32)
    trees = [_tree(n, rng) for n, _ in lengths]
    s.parent = torch.tensor([p for t in trees for p in t], dtype=torch.int32, device="cuda")
    s.mask = torch.zeros((s.rows, s.words), dtype=torch.int32, device="cuda")
    if op == "draft":
        s.q, s.new_k, s.new_v, s.q_out = rows(hq), rows(hk), rows(hk), empty(hq)
        s.position = torch.zeros(s.rows, dtype=torch.int32, device="cuda")
        angle = torch.arange(s.len, dtype=torch.float64)[:, None] * ROPE_BASE ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
        s.cos, s.sin = angle.cos().float().cuda(), angle.sin().float().cuda()
        s.k_out = s.v_out = None
        if c["fmt"] != "fp16":
            s.k_out, s.v_out = empty(hk), empty(hk)
        return
    s.q, s.out = rows(hq), empty(hq)
    words = []   # the masks are made once in a step, for the attention of all layers
    for t in trees:
        seen = []
        for i, p in enumerate(t):
            seen.append((seen[p] if p >= 0 else 0) | 1 << i)
        words += [[(m >> 32 * w & 0xFFFFFFFF) - (1 << 32 if m >> 32 * w & 0x80000000 else 0) for w in range(s.words)] for m in seen]
    s.mask.copy_(torch.tensor(words, dtype=torch.int32))


def prepare(case, seed):
    s = _State()
    s.case = dict(case)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    if case["op"] == "select":
        _prepare_select(s, gen)
    elif case["op"] == "reorder":
        _prepare_reorder(s, gen)
    else:
        _prepare_rows(s, gen, seed)
    return s


# ---- the plain form --------------------------------------------------------------------------------
def _quantise(x, fmt):
    """Codes and fp16 scales of rows of fp16 values: the scale is the smallest fp16 that takes the row's largest value to the largest code."""
    x = x.float()
    most = x.abs().amax(dim=-1)
    h = (most / CODES[fmt]).half()
    h = torch.where(h.float() * CODES[fmt] < most, (h.view(torch.int16) + 1).view(torch.float16), h)   # (the product is exact)
    h = torch.where(most > 0, h, torch.ones_like(h))
    y = x / h.float()[..., None]
    return (y.round().clamp(-127, 127).to(torch.int8) if fmt == "int8" else y.to(torch.float8_e4m3fn)), h


def _places(s):
    """Sequence, index among its new rows, position, page and slot of every row."""
    row = torch.arange(s.rows, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s.row_start, row, right=True) - 1
    index = row - s.row_start[seq]
    pos = s.kv_len[seq] - s.row_start[seq + 1] + row
    page = s.table[seq, (pos // s.case["page"]).long()].long()
    return seq, index.long(), pos.long(), page, (pos % s.case["page"]).long()


def _bytes(t):
    """Codes without their type, which indexing does not know."""
    return t.view(torch.uint8) if t.element_size() == 1 else t


def _cells(codes, scales, page, slot):
    """fp32 values of a layer's cells at (page, slot): [..., kv head, dim]."""
    if scales is None:
        return codes[page, :, slot].float()
    return _bytes(codes)[page, :, slot].view(codes.dtype).float() * scales[page, :, slot].float()[..., None]


def _rotated(x, cos, sin):
    a, b = x.float().chunk(2, dim=-1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1).half()


def _plain_draft(s):
    c = s.case
    seq, index, _, page, slot = _places(s)
    S, T, W = c["seqs"], s.new, s.words
    # With P the matrix of parents, strictly below the diagonal, the sum of its powers is the inverse of 1 - P: a token's row has a 1 for itself and each ancestor.
    less = torch.eye(T, device="cuda").repeat(S, 1, 1)
    child = s.parent >= 0
    less[seq[child], index[child], s.parent[child].long()] = -1.0
    seen = torch.linalg.solve_triangular(less, torch.eye(T, device="cuda").expand(S, T, T), upper=False, unitriangular=True)[seq, index]   # [rows, T]
    s.position.copy_(s.kv_len[seq] - (s.row_start[seq + 1] - s.row_start[seq]) + seen.sum(1).int() - 1)
    bits = torch.zeros((s.rows, W * 32), dtype=torch.int64, device="cuda")
    bits[:, :T] = seen.long()
    s.mask.copy_((bits.view(s.rows, W, 32) << torch.arange(32, device="cuda")).sum(2))   # (the low 32 bits)
    cos, sin = s.cos[s.position.long()][:, None], s.sin[s.position.long()][:, None]
    s.q_out.copy_(_rotated(s.q, cos, sin))
    out = {"mask": s.mask, "position": s.position, "q": s.q_out, "k": s.k, "v": s.v}
    new_k = _rotated(s.new_k, cos, sin)
    if s.k_scale is None:
        s.k[0, page, :, slot] = new_k
        s.v[0, page, :, slot] = s.new_v
        return out
    for new, codes, scales, back in ((new_k, s.k[0], s.k_scale[0], s.k_out), (s.new_v, s.v[0], s.v_scale[0], s.v_out)):
        q, h = _quantise(new, c["fmt"])
        _bytes(codes)[page, :, slot] = q.view(torch.uint8)
        scales[page, :, slot] = h
        back.copy_(_cells(codes, scales, page, slot))
    return {**out, "k": s.k_out, "v": s.v_out}


def _plain_tree(s):
    c = s.case
    D, hk, P = c["dim"], c["kv_heads"], c["page"]
    G, S = c["q_heads"] // hk, c["seqs"]
    key = torch.arange(s.len, device="cuda")
    inside = key[None] < s.kv_len[:, None]                                          # [S, L]
    page = torch.where(inside, s.table[:, key // P], 0).long()
    slot = (key % P)[None].expand_as(page)
    k = _cells(s.k[0], None if s.k_scale is None else s.k_scale[0], page, slot).permute(0, 2, 3, 1)     # [S, hk, D, L]
    v = torch.where(inside[..., None, None], _cells(s.v[0], None if s.v_scale is None else s.v_scale[0], page, slot), 0.0).permute(0, 2, 1, 3)
    t = torch.arange(s.new, device="cuda")
    count = s.row_start[1:] - s.row_start[:-1]
    row = torch.minimum(s.row_start[:-1, None] + t, s.row_start[1:, None] - 1).long()   # [S, T], the last row again where there are fewer
    q = s.q[row].float().view(S, s.new, hk, G, D).permute(0, 2, 3, 1, 4).reshape(S, hk, G * s.new, D)
    j = key[None] - (s.kv_len - count)[:, None]                                     # [S, L]: the key's index among the new ones
    at = j.clamp(0, s.words * 32 - 1).long()
    bit = s.mask[row].gather(2, (at // 32)[:, None].expand(S, s.new, s.len)) >> (at % 32)[:, None] & 1
    seen = inside[:, None] & ((j < 0)[:, None] | (bit == 1))                        # [S, T, L]
    x = (q @ k).view(S, hk, G, s.new, s.len).mul_(D ** -0.5)
    x = x.masked_fill_(~seen[:, None, None], -math.inf)
    x = x.sub_(x.amax(dim=-1, keepdim=True)).exp_()
    x = x.div_(x.sum(dim=-1, keepdim=True)).view(S, hk, G * s.new, s.len)
    o = (x @ v).view(S, hk, G, s.new, D).permute(0, 3, 1, 2, 4).reshape(S, s.new, c["q_heads"], D)
    seq, index, _, _, _ = _places(s)
    s.out.copy_(o[seq, index])
    return {"out": s.out}


def _held(s):
    """What the caches of all layers hold, codes as the numbers they are."""
    out = {"k": _bytes(s.k), "v": _bytes(s.v)}
    if s.k_scale is not None:
        out.update(k_scale=s.k_scale, v_scale=s.v_scale)
    return out


def _plain_move(s):
    seq, _, _, page, slot = _places(s)
    from_page, from_slot = s.table[seq, (s.source // s.case["page"]).long()].long(), (s.source % s.case["page"]).long()
    for t in _held(s).values():
        t[:, page, :, slot] = t[:, from_page, :, from_slot]
    return _held(s)


def _plain_reorder(s):
    c = s.case
    P, B = c["page"], c["beams"]
    first = torch.arange(c["groups"] * B, device="cuda") // B * B
    parent = first + s.parent.long()
    full = (s.kv_len // P).long()
    mine, theirs = s.table.gather(1, full[:, None])[:, 0].long(), s.table[parent].gather(1, full[:, None])[:, 0].long()
    new = torch.arange(P, device="cuda") < (s.kv_len % P)[:, None]                  # [beams, slots]
    for t in _held(s).values():
        keep = new.view(1, -1, 1, P, *([1] * (t.dim() - 4)))
        t[:, mine] = torch.where(keep, t[:, theirs], t[:, mine])
    entry = torch.arange(s.table.shape[1], device="cuda")
    s.table.copy_(torch.where(entry < full[:, None], s.table[parent], s.table))
    return {"table": s.table, **_held(s)}


def _plain_select(s):
    c = s.case
    G, B, V, n = c["groups"], c["beams"], c["vocab"], c["picks"]
    x = s.logits[:, :V]
    # The best of each beam: fp16 numbers in order as whole ones, and of equal ones the lowest token.
    code = (x + 0.0).view(torch.int16).int()
    key = (torch.where(code < 0, -32768 - code, code).long() << 32) + (V - 1 - torch.arange(V, device="cuda"))
    best = key.topk(min(n, V), dim=1).values
    token = V - 1 - (best & 0xFFFFFFFF)
    token = token.sort(dim=1).values
    # log-softmax and scores in 64 bits: the order goes by them
    y = x.double()
    top = y.amax(dim=1, keepdim=True)
    total = (s.score.double().view(-1, 1) + ((x.gather(1, token).double() - top) - (y - top).exp().sum(dim=1, keepdim=True).log()))
    if s.done is not None:   # a beam that has ended goes on as it is, with one candidate
        ended = s.done.view(-1, 1) != 0
        one = torch.arange(token.shape[1], device="cuda") == 0
        total = torch.where(ended, torch.where(one, s.score.double().view(-1, 1), -math.inf), total)
        token = torch.where(ended, s.eos, token)
    total, token = total.view(G, -1), token.view(G, -1)
    order = total.sort(dim=1, descending=True, stable=True)
    count = min(n, token.shape[1])
    value, at = order.values[:, :count], order.indices[:, :count]
    there = value > -math.inf
    s.out_score.fill_(-math.inf)
    s.token.fill_(-1)
    s.parent.fill_(-1)
    s.out_score[:, :count] = value.float()
    s.token[:, :count] = torch.where(there, token.gather(1, at), -1).int()
    s.parent[:, :count] = torch.where(there, at // (token.shape[1] // B), -1).int()
    out = {"score": s.out_score, "token": s.token, "parent": s.parent}
    if s.done is None:
        return out
    s.out_done.copy_((s.token >= 0) & (s.token == s.eos))
    return {**out, "done": s.out_done}


def run(state):
    s, c = state, state.case
    if not own:
        return {"draft": _plain_draft, "tree": _plain_tree, "move": _plain_move, "select": _plain_select, "reorder": _plain_reorder}[c["op"]](s)
    ctx = _ctx()
    if c["op"] == "draft":
        ctx.tree_layout(s.batch, _p(s.parent), s.words, _p(s.mask), _p(s.position))
        ctx.rope_kv_write_at(s.handles[0], s.batch, _p(s.position), _p(s.cos), _p(s.sin), s.len, c["dim"], c["q_heads"], _p(s.q), 0, _p(s.q_out), 0,
                             _p(s.new_k), 0, _p(s.new_v), 0)
        out = {"mask": s.mask, "position": s.position, "q": s.q_out, "k": s.k, "v": s.v}
        if c["fmt"] == "fp16":
            return out
        ctx.kv_read(s.handles[0], s.batch, _p(s.k_out), 0, _p(s.v_out), 0)
        return {**out, "k": s.k_out, "v": s.v_out}
    if c["op"] == "tree":
        ctx.attention_tree(s.handles[0], s.batch, c["q_heads"], _p(s.q), 0, _p(s.out), 0, c["dim"] ** -0.5, s.words, _p(s.mask))
        return {"out": s.out}
    if c["op"] == "move":
        ctx.kv_move(s.handles, s.batch, _p(s.source))
        return _held(s)
    if c["op"] == "reorder":
        ctx.kv_reorder(s.handles, s.batch, c["beams"], _p(s.parent))
        return {"table": s.table, **_held(s)}
    ctx.beam_select(c["groups"], c["beams"], c["vocab"], _p(s.logits), s.logits.shape[1], _p(s.score), _p(s.done), s.eos, c["picks"], _p(s.out_score), _p(s.token),
                    _p(s.parent), _p(s.out_done))
    out = {"score": s.out_score, "token": s.token, "parent": s.parent}
    return out if s.done is None else {**out, "done": s.out_done}


# ---- in 64 bits, from the definition ---------------------------------------------------------------
def _exact_rotation(x, positions):
    half = x.shape[-1] // 2
    rate = ROPE_BASE ** (-2.0 * torch.arange(half, dtype=torch.float64, device="cuda") / x.shape[-1])
    angle = torch.as_tensor(positions, dtype=torch.float64, device="cuda").view(-1, 1, 1) * rate
    x = x.double()
    c, s = angle.cos().float().double(), angle.sin().float().double()   # (the tables hold 32 bits)
    y = torch.empty_like(x)
    y[..., :half] = x[..., :half] * c - x[..., half:] * s
    y[..., half:] = x[..., half:] * c + x[..., :half] * s
    return y.half()                                                     # (the cache takes fp16 rows)


def _exact_stored(x, fmt):
    """What the cells of these fp16 rows stand for."""
    x = x.double()
    if fmt == "fp16":
        return x
    want = x.abs().max(dim=-1, keepdim=True).values / CODES[fmt]
    step = torch.exp2(torch.clamp(torch.floor(torch.log2(want.clamp(min=2.0 ** -40))) - 10, min=-24.0))      # between neighbours in fp16
    scale = torch.where(want == 0, 1.0, torch.ceil(want / step) * step)
    y = x / scale
    if fmt == "int8":
        return torch.round(y) * scale
    step = torch.exp2(torch.clamp(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -30))), min=-6.0) - 3.0)   # 3 bits behind the first, from 2^-6 on
    return torch.clamp(torch.round(y / step) * step, -448.0, 448.0) * scale


def _exact_draft(s):
    c, P = s.case, s.case["page"]
    parent, table = s.parent.tolist(), s.table.tolist()
    mask, pos, cells, row = [], [], [], 0
    for i, (n, length) in enumerate(_lengths(c)):
        for j in range(n):
            seen, up = 0, j
            depth = -1
            while up >= 0:
                seen, up, depth = seen | 1 << up, parent[row + up], depth + 1
            mask.append([(seen >> 32 * w & 0xFFFFFFFF) - (1 << 32 if seen >> (32 * w + 31) & 1 else 0) for w in range(s.words)])
            pos.append(length - n + depth)
            cells.append((table[i][(length - n + j) // P], (length - n + j) % P))
        row += n
    whole = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    out = {"mask": whole(mask), "position": whole(pos), "q": _exact_rotation(s.q, pos).double()}
    k, v = _exact_stored(_exact_rotation(s.new_k, pos), c["fmt"]), _exact_stored(s.new_v, c["fmt"])
    if c["fmt"] != "fp16":
        return {**out, "k": k, "v": v}
    out["k"], out["v"] = s.k.double(), s.v.double()
    for r, (page, slot) in enumerate(cells):
        out["k"][0, page, :, slot], out["v"][0, page, :, slot] = k[r], v[r]
    return out


def _exact_tree(s):
    c, D, P = s.case, s.case["dim"], s.case["page"]
    table, parent, G, parts, at = s.table.cpu(), s.parent.tolist(), c["q_heads"] // c["kv_heads"], [], 0

    def sequence(i, length, codes, scales):
        """[position, kv head, dim] of one sequence."""
        pages = table[i, : -(-length // P)].long().cuda()
        value = codes[0, pages].double() if scales is None else _bytes(codes)[0, pages].view(codes.dtype).double() * scales[0, pages].double()[..., None]
        return value.transpose(1, 2).reshape(-1, c["kv_heads"], D)[:length]

    for i, (n, length) in enumerate(_lengths(c)):
        k, v = sequence(i, length, s.k, s.k_scale), sequence(i, length, s.v, s.v_scale)
        hidden = torch.zeros((n, length), dtype=torch.bool)
        hidden[:, length - n:] = True
        for j in range(n):
            up = j
            while up >= 0:
                hidden[j, length - n + up] = False
                up = parent[at + up]
        hidden = hidden.cuda()
        got = torch.empty((n, c["q_heads"], D), dtype=torch.float64, device="cuda")
        for h in range(c["q_heads"]):
            score = s.q[at:at + n, h].double() @ k[:, h // G].T / math.sqrt(D)
            got[:, h] = torch.softmax(score.masked_fill(hidden, -math.inf), dim=-1) @ v[:, h // G]
        parts.append(got)
        at += n
    return {"out": torch.cat(parts)}


def _exact_move(s):
    c, P = s.case, s.case["page"]
    table, source, ends = s.table.tolist(), s.source.tolist(), s.kv_len.tolist()
    to, of, row = [], [], 0
    for i, (n, _) in enumerate(_lengths(c)):
        for j in range(n):
            a, b = ends[i] - n + j, source[row + j]
            to.append(table[i][a // P] * P + a % P)
            of.append(table[i][b // P] * P + b % P)
        row += n
    out = {}
    for name, t in _held(s).items():
        flat = t.transpose(2, 3).flatten(1, 2)            # [layer][page and slot][kv head] ..
        new = flat.clone()
        new[:, to] = flat[:, of]
        new = new.unflatten(1, (-1, P)).transpose(2, 3)
        out[name] = new.double() if new.is_floating_point() else new
    return out


def _exact_reorder(s):
    c, P, B = s.case, s.case["page"], s.case["beams"]
    table, parent, held = s.table.tolist(), s.parent.tolist(), _held(s)
    new_table = [list(r) for r in table]
    new = {name: t.double() if t.is_floating_point() else t.clone() for name, t in held.items()}
    for g, n in enumerate(_beam_lengths(c)):
        for b in range(B):
            me, it = g * B + b, g * B + parent[g * B + b]
            new_table[me][:n // P] = table[it][:n // P]
            a, z = table[me][n // P], table[it][n // P]
            for name, t in new.items():
                t[:, a, :, :n % P] = held[name][:, z, :, :n % P].to(t.dtype)
    return {"table": torch.tensor(new_table, dtype=torch.int32, device="cuda"), **new}


def _exact_select(s):
    c = s.case
    B, V, n, rows = c["beams"], c["vocab"], c["picks"], []
    for g in range(c["groups"]):
        total = torch.log_softmax(s.logits[g * B:(g + 1) * B, :V].double(), dim=1) + s.score[g].double()[:, None]
        if s.done is not None:
            for b in range(B):
                if s.done[g, b]:
                    total[b] = -math.inf
                    total[b, s.eos] = s.score[g, b].double()
        flat = total.flatten()
        most = torch.topk(flat, min(n, flat.numel())).values[-1]
        at = torch.nonzero(flat >= most)[:, 0]                                   # (ascending)
        at = at[torch.sort(flat[at], descending=True, stable=True).indices][:n]
        ok = flat[at] > -math.inf
        fill = n - len(at)
        pad = lambda x, v: torch.cat((x, torch.full((fill,), v, dtype=x.dtype, device="cuda")))  # noqa: E731
        rows.append((pad(flat[at], -math.inf), pad(torch.where(ok, at % V, -1), -1).int(), pad(torch.where(ok, at // V, -1), -1).int()))
    score, token, parent = (torch.stack(x) for x in zip(*rows))
    out = {"score": score, "token": token, "parent": parent}
    return out if s.done is None else {**out, "done": ((token >= 0) & (token == s.eos)).int()}


def exact(case, seed):
    s = prepare(case, seed)
    return {"draft": _exact_draft, "tree": _exact_tree, "move": _exact_move, "select": _exact_select, "reorder": _exact_reorder}[case["op"]](s)
