"""Drafted trees, beams and cells that move, in plain 64-bit arithmetic and host loops."""
import numpy as np


def random_tree(n, rng):
    """Parents: each goes on from one of the eight before it, or begins at the sequence's end."""
    return [-1 if i == 0 or rng.random() < 0.15 else int(rng.integers(max(0, i - 8), i)) for i in range(n)]


def masks_of(parents):
    """What each row sees, as whole numbers, and its depth."""
    seen, depth = [], []
    for i, p in enumerate(parents):
        seen.append((seen[p] if p >= 0 else 0) | 1 << i)
        depth.append(depth[p] + 1 if p >= 0 else 0)
    return seen, depth


def words_of(masks, words):
    return np.array([[m >> 32 * w & 0xFFFFFFFF for w in range(words)] for m in masks], np.uint32).reshape(-1, words)


def attend_keys(q, k, v, scale, keys):
    """Row i of q over the keys keys[i]: the result and what an error bound needs (attention_bound)."""
    n, D = q.shape
    out, spread, most, steep = np.zeros((n, D)), np.zeros((n, D)), np.zeros(n), np.zeros(n)
    for i, key in enumerate(keys):
        if not len(key):
            continue
        with np.errstate(invalid="ignore", over="ignore"):
            s = scale * (k[key] @ q[i])
            w = np.exp(s - s.max())
            w /= w.sum()
            out[i] = w @ v[key]
            spread[i] = w @ np.abs(v[key])
            most[i] = np.abs(v[key], where=np.isfinite(v[key]), out=np.zeros_like(v[key])).max()
            far = np.abs(k[key]) @ np.abs(q[i])
            steep[i] = scale * np.where(np.isfinite(far), far, 0).max()
    return out, spread, most, steep


def tree_keys(mask, n, length):
    """The keys that a row with this mask sees, in a sequence of `length` positions whose last n are the tree."""
    base = length - n
    return np.array([key for key in range(length) if key < base or mask >> (key - base) & 1], int)


def best_continuations(logits, score, done, eos, picks):
    """One group: logits [beams, vocab] fp16, score [beams] fp32, done [beams] or None -> totals in 64 bits, tokens, parents, and the smallest distance
    between totals of different beams among the picks and the first one left out."""
    B, V = logits.shape
    x = logits.astype(np.float64)
    total = np.full((B, V), -np.inf)
    for b in range(B):
        if done is not None and done[b]:
            total[b, eos] = score[b]
            continue
        m = x[b].max() if not np.isnan(x[b]).any() else np.nan
        if not np.isfinite(m):
            continue
        with np.errstate(divide="ignore"):
            total[b] = np.float64(score[b]) + ((x[b] - m) - np.log(np.exp(x[b] - m).sum()))
    flat = np.where(np.isnan(total), -np.inf, total).ravel()
    order = np.lexsort((np.arange(flat.size), -flat))[:picks + 1]
    order = order[flat[order] > -np.inf]
    near = min((abs(flat[a] - flat[c]) for a, c in zip(order, order[1:]) if a // V != c // V), default=np.inf)
    order = order[:picks]
    fill = picks - len(order)
    pad = lambda a, v: np.concatenate([a, np.full(fill, v)])  # noqa: E731
    return pad(flat[order], -np.inf), pad(order % V, -1).astype(np.int32), pad(order // V, -1).astype(np.int32), near
