"""Calls of the beam selection in which a thread has several rounds of logits: their rows and, in 64 bits, their picks."""
import numpy as np

# groups, beams, vocab, picks, and what 148 SMs make of it: segments of a row, rounds of a segment (1024 vectors of 8 logits each)
SHAPES = [(64, 8, 151936, 16, 4, 5), (16, 8, 1 << 20, 9, 19, 7), (300, 8, 70001, 8, 1, 9), (512, 8, 32769, 4, 1, 5), (40, 32, 300007, 32, 2, 20), (1, 19, 1 << 26, 32, 128, 64)]
KINDS = ["random", "up", "down", "late", "few", "equal", "masked"]


def rows_of(kind, beams, vocab, seed):
    rng = np.random.default_rng(seed)
    if kind == "equal":
        return np.full((beams, vocab), 0.25, np.float16)
    if kind == "few":
        return (rng.integers(0, 2, (beams, vocab), np.int8) * 3).astype(np.float16)
    x = rng.standard_normal((beams, vocab), np.float32) * np.float32(2.5)
    if kind in ("up", "down"):
        x = np.sort(x, axis=-1)
        x = x[:, ::-1] if kind == "down" else x
    elif kind == "late":
        x[:, -40:] += 14
    elif kind == "masked":      # all but a few, in one place, and the lowest values in others
        x[:, : vocab - vocab // 3] = -np.inf
        x[:, ::7] = -65504
    return np.ascontiguousarray(x).astype(np.float16)


def best_of(logits, score, picks):
    """One group's totals, tokens, parents, and the smallest distance between totals of different beams among the picks and the first one left out."""
    tokens, parents, totals = [], [], []
    for b, row in enumerate(logits):
        sum_, most = 0.0, np.float64(row.max())
        for i in range(0, len(row), 1 << 22):
            sum_ += np.exp(row[i:i + (1 << 22)].astype(np.float64) - most).sum()
        least = np.partition(row, -picks - 1)[-picks - 1] if len(row) > picks else -np.inf
        t = np.flatnonzero((row >= least) & (row > -np.inf))
        t = t[np.lexsort((t, -row[t].astype(np.float32)))][:picks + 1]
        tokens.append(t)
        parents.append(np.full(len(t), b))
        totals.append(np.float64(score[b]) + ((row[t].astype(np.float64) - most) - np.log(sum_)))
    t, p, total = (np.concatenate(x) for x in (tokens, parents, totals))
    order = np.lexsort((t, p, -total))[:picks + 1]
    near = min((abs(total[a] - total[c]) for a, c in zip(order, order[1:]) if p[a] != p[c]), default=np.inf)
    order = order[:picks]
    return total[order], t[order].astype(np.int32), p[order].astype(np.int32), near
