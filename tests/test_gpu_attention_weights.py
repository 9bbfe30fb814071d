"""The softmax's weights as fp16: what their rounding must not do to a result."""
import math

import numpy as np
import pytest

import kv_reference as ref
from test_gpu_attention import check_attention, run_attention

pytestmark = pytest.mark.gpu

# (the parts of the last one's items are joined by the blocks that have them, those of the chunk by a kernel of their own)
SHAPES = {"token": [(1, 600)], "drafts": [(5, 600)], "chunk": [(140, 600)], "chunks": [(140, 600)] * 40}


def _set(c, name, rows):
    """rows [pages, heads, page, D] as the cache's contents, on both sides."""
    if c.fmt == "fp16":
        c.host[name] = rows.view(np.uint16)
    else:
        c.host[name], c.host[name + "_scale"] = ref.quantised(rows, c.fmt)
        c.ctx.upload(c.host[name + "_scale"].view(np.uint16), c.dev[name + "_scale"])
    c.ctx.upload(c.host[name], c.dev[name])


def _by_position(c, length, rows):
    """rows [length, D] to every head's cells of the first sequence; zeros elsewhere."""
    x = np.zeros((c.pages, c.kv_heads, c.page, c.D), np.float16)
    p = np.arange(length)
    x[c.table[0, p // c.page], :, p % c.page] = rows[:, None]
    return x


@pytest.mark.parametrize("shape", list(SHAPES))
@pytest.mark.parametrize("fmt,D", [("fp16", 64), ("fp16", 128), ("int8", 64), ("fp8", 128)])
def test_largest_values_do_not_become_infinite(nnb, ctx, fmt, D, shape):
    """Values of 65504 under weights that are all rounded up: 1 to one key of 16 and 1/2 (1 + 0.6 2^-10) to the others.  Their sum is larger by 3.4e-4 than that
    of the weights before rounding, and 65504 (1 + 2.5e-4) would be stored as an infinity."""
    seqs, page = SHAPES[shape], 16
    new, length = seqs[0]
    c = ref.Cache(nnb, ctx, fmt, [n for _, n in seqs], 1, D, page, seed=61)
    c.table[:] = c.table[0]
    k = np.zeros((length, D), np.float16)
    k[np.arange(length) % 16 != 0, 0] = -1
    k[np.arange(length) % 16 != 0, 1] = math.log2(1 + 0.6 * 2.0 ** -10)
    if fmt != "fp16":                            # (8 bits: as two dims that codes can hold; the scale is 1/127 or 1/448, rounded up)
        k[:, 1] = 0
    _set(c, "k", _by_position(c, length, k))
    _set(c, "v", _by_position(c, length, np.full((length, D), 65504, np.float16)))
    q = np.zeros((new * len(seqs), 2, D), np.float16)
    q[..., :2] = 1
    scale = math.log(2.0)
    got = run_attention(nnb, ctx, c, q, [n for n, _ in seqs], scale=scale)
    ctx.sync()
    assert np.isfinite(got).all()
    check_attention(c, got, q, seqs, scale, 0, 0, f"largest values {fmt} D{D} {shape}")
    c.close()


@pytest.mark.parametrize("shape", ["token", "drafts", "chunk"])
@pytest.mark.parametrize("gap,size", [(0.0, 2.0 ** -16), (0.0, 2.0 ** -6), (10.0, 2.0 ** -6), (4.0, 2.0 ** -10)])
@pytest.mark.parametrize("fmt,D", [("fp16", 64), ("int8", 64), ("int8", 128), ("fp8", 64), ("fp8", 128)])
def test_a_value_row_of_zeros_leaves_the_others_their_weights(nnb, ctx, fmt, D, shape, gap, size):
    """The first key has a value row of zeros (its scale is 1), 2^gap times the others' weight, and the others' values are small (scales of size / 40).

    The weights of codes carry the values' scales.  The largest of them, W, is kept between 2^7 and 2^15 as an fp16 number, so that another one is off by 2^-11 of
    itself or by 2^-25 2^-7 W, whichever is more: a summand of the result, with codes up to Q, by 2^-32 W Q."""
    new, length = SHAPES[shape][0]
    length = 12 + new if size == 2.0 ** -16 else length
    seqs = [(new, length)]
    c = ref.Cache(nnb, ctx, fmt, [length], 1, D, 16, seed=62)
    rng = np.random.default_rng(63)
    k, v = (0.3 * rng.standard_normal((length, D))).astype(np.float16), (size * rng.standard_normal((length, D))).astype(np.float16)
    k[:, 0] = 0
    k[0], v[0] = 0, 0
    k[0, 0] = 1
    _set(c, "k", _by_position(c, length, k))
    _set(c, "v", _by_position(c, length, v))
    q = rng.standard_normal((new, 2, D)).astype(np.float16)
    scale = D ** -0.5
    q[..., 0] = gap * math.log(2.0) / scale
    got = run_attention(nnb, ctx, c, q, [new], scale=scale).astype(np.float64)
    ctx.sync()
    ks, vs = c.sequence("k", 0, length), c.sequence("v", 0, length)
    codes = {"fp16": 0.0, "int8": 127.0, "fp8": 448.0}[fmt]
    for h in range(2):
        want, spread, most, steep = ref.attend(q[:, h].astype(np.float64), ks[:, 0], vs[:, 0], np.arange(length - new, length), scale, 0, 0)
        bound = ref.attention_bound(want, spread, most, steep, length, D)
        for i, p in enumerate(range(length - new, length)):
            s = scale * (ks[:p + 1, 0] @ q[i, h].astype(np.float64))
            w = np.exp(s - s.max())
            w /= w.sum()
            top = 0.0 if fmt == "fp16" else (w * c.host["v_scale"][c.table[0, np.arange(p + 1) // 16], 0, np.arange(p + 1) % 16].astype(np.float64)).max()
            off = np.abs(got[i, h] - want[i]) / (bound[i] + (p + 1) * 2.0 ** -32 * top * codes)
            assert off.max() <= 1, (i, h, off.max())
    c.close()
