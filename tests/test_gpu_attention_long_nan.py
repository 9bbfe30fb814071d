"""A row of very many keys that is computed once more from its formula takes longer than the limit of the next launch's waits: that launch must not be begun meanwhile."""
import numpy as np
import pytest

from helpers import make_weight, make_x
from oracle import cpu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("length", [1 << 19, 1 << 24])
def test_the_next_launch_waits_for_rows_that_are_computed_once_more(nnb, ctx, length):
    """Some 160 ns a key for twelve rows: 2.7 s at 2^24 keys, against a limit of about 2 s.  (All positions lie in one page, which holds an infinity.)"""
    D, G, page = 64, 12, 256
    cells = np.zeros((page, D), np.float16)
    k = ctx.upload(cells)
    cells[7, 3] = np.inf
    v = ctx.upload(cells)
    cache = ctx.kv_cache("fp16", 1, page, 1, D, k, v)
    up = [ctx.upload(a) for a in (np.array([0, 1], np.int32), np.array([length], np.int32), np.zeros(length // page, np.int32))]
    q, out = ctx.upload(np.zeros((G, D), np.float16)), ctx.alloc(G * D * 2)
    N, K = 4096, 4864
    W, s = make_weight("int8", N, K, 81)
    qw, x = nnb.QuantWeight(ctx, "int8", W, s), make_x(1, K, 82)
    dx, y = ctx.upload(x.view(np.uint16)), ctx.alloc(N * 2)
    ctx.attention(cache, nnb.KVBatch(1, 1, 1, length, length // page, *up), G, q, 0, out, 0, 1.0)
    ctx.linear(1, N, K, dx, qw.buf, y)
    ctx.sync()                                                    # (raised NN_ERR_TIMEOUT where the launch had begun too early)
    got = ctx.download(out, (G, D), np.float16)
    assert (got[:, 3] == np.inf).all() and not np.delete(got, 3, axis=1).any()
    assert cpu.rel_l2(ctx.download(y, (1, N), np.float16).astype(np.float32), cpu.linear("int8", x, W, s).astype(np.float32)) < 1e-3
    qw.release()
    cache.close()
    for b in (k, v, *up, q, out, dx, y):
        ctx.free(b)
