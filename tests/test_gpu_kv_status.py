"""A wait that ran out and a bad page between two synchronisations: nn_sync reports the one that makes results invalid."""
import numpy as np
import pytest

import kv_reference as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("order", ["wait first", "page first", "page alone"])
@pytest.mark.parametrize("kind", ["write", "read", "few rows", "many rows"])
def test_a_bad_page_does_not_hide_a_wait_that_ran_out(nnb, ctx, kind, order):
    c = ref.Cache(nnb, ctx, "fp16", [10], 2, 64, 16, seed=51)
    k, v, q, out = (ctx.upload(np.zeros((2, n, 64), np.float16)) for n in (2, 2, 4, 4))
    table = c.table.copy()
    table[0, 0] = c.pages
    good, bad = c.batch([2]), c.batch([2], table=table, max_new=200 if kind == "many rows" else 2)
    comm = nnb.Comm(ctx, None, 0, 1)

    def bad_page():
        if kind == "write":
            ctx.kv_write(c.handle, bad, k, 0, v, 0)
        elif kind == "read":
            ctx.kv_read(c.handle, bad, k, 0, v, 0)
        else:
            ctx.attention(c.handle, bad, 4, q, 0, out, 0, 0.125)

    try:
        comm.symm_alloc(256)
        ctx.sync()
        calls = [bad_page] if order == "page alone" else [lambda: comm.wait(timeout_ms=50), bad_page]     # (nothing signals)
        for call in calls[::-1] if order == "page first" else calls:
            call()
        with pytest.raises(nnb.NNError) as e:
            ctx.sync()
        assert e.value.code == (nnb.NN_ERR_ARG if order == "page alone" else nnb.NN_ERR_TIMEOUT)
        assert "out of range" in str(e.value)           # (the page is mentioned in either case)
        ctx.sync()                                      # both have been reported
        ctx.attention(c.handle, good, 4, q, 0, out, 0, 0.125)
        ctx.sync()
    finally:
        comm.close()
        c.close()
        for b in (k, v, q, out):
            ctx.free(b)
