"""Many short items to a block of the kernel for many rows: each of its warps goes from segment to segment of its own, told by one of its lanes."""
import numpy as np
import pytest

import kv_reference as ref
from test_gpu_attention import check_attention, run_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt,D,page,hq,hk", [("fp16", 64, 16, 8, 2), ("fp16", 128, 32, 4, 2), ("int8", 64, 16, 6, 2), ("int8", 128, 16, 8, 2), ("fp8", 64, 64, 2, 2), ("fp8", 128, 16, 40, 2)])
def test_many_segments_to_a_block(nnb, ctx, fmt, D, page, hq, hk):
    """Sequences of 0 to 70 new tokens and 1 to 4 key tiles in no order, so that a block's segments differ in rows, tiles and in whether two
    query tiles hold the same rows; every repetition gives the same bits."""
    rng = np.random.default_rng(41)
    seqs = [(int(n), int(n + rng.integers(0, 600))) for n in rng.integers(0, 71, 400)]
    c = ref.Cache(nnb, ctx, fmt, [n for _, n in seqs], hk, D, page, seed=42)
    new = [n for n, _ in seqs]
    q = rng.standard_normal((sum(new), hq, D)).astype(np.float16)
    window = dict(window=300, sinks=5)
    first = run_attention(nnb, ctx, c, q, new, max_new=128, **window)
    ctx.sync()
    for _ in range(20):
        again = run_attention(nnb, ctx, c, q, new, max_new=128, **window)
        assert np.array_equal(first.view(np.uint16), again.view(np.uint16))
    ctx.sync()
    keep, row, rows = list(range(0, 400, 7)), 0, []       # (the host's formula on every seventh)
    for i, n in enumerate(new):
        if i in keep:
            rows.append(np.arange(row, row + n))
        row += n
    pick = np.concatenate(rows)

    class Some:
        kv_heads = hk

        def sequence(self, name, i, n):
            return c.sequence(name, keep[i], n)

    check_attention(Some(), first[pick], q[pick], [seqs[i] for i in keep], D ** -0.5, 300, 5, f"segments {fmt} D{D}")
    c.close()
