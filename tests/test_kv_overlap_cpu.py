"""A write whose cache lies over what tells it where to write, or how far to turn: refused (addresses alone; nothing is read)."""
import ctypes

import pytest

BUF = 1 << 20
CELLS, SCALES = 4 * 16 * 2 * 64, 4 * 16 * 2 * 2     # bytes of 4 pages of 16 positions and 2 heads of 64 dims in 8 bits, and of their scales
K, V, KS, VS = BUF, 2 * BUF, 3 * BUF, 4 * BUF
NO_CONTEXT = b"null context"


def _call(nnb, L, name, rot=64, cos=32 * BUF, sin=33 * BUF, **where):
    h = ctypes.c_void_p()
    assert L.nn_kv_cache_create(None, 1, 4, 16, 2, 64, K, V, KS, VS, ctypes.byref(h)) == 0
    b = nnb.KVBatch(**{**dict(num_seqs=2, num_rows=6, max_new=3, max_len=100, table_stride=8, row_start=16 * BUF, kv_len=17 * BUF, page_table=18 * BUF), **where})
    q, k, v, out = (n * BUF for n in (64, 65, 66, 67))
    rc = {"nn_kv_write": lambda: L.nn_kv_write(None, h, b, k, 0, v, 0),
          "nn_rope_kv_write": lambda: L.nn_rope_kv_write(None, h, b, cos, sin, 100, rot, 4, q, 0, q, 0, k, 0, v, 0),
          "nn_kv_read": lambda: L.nn_kv_read(None, h, b, k, 0, v, 0),
          "nn_attention": lambda: L.nn_attention(None, h, b, 4, q, 0, out, 0, 0.125, 0, 0)}[name]()
    L.nn_kv_cache_free(h)
    return rc, L.nn_last_error()


@pytest.mark.parametrize("name", ["nn_kv_write", "nn_rope_kv_write"])
@pytest.mark.parametrize("where", [dict(row_start=K), dict(row_start=V + CELLS - 4), dict(kv_len=KS + SCALES - 4), dict(kv_len=K - 4), dict(page_table=VS + 8), dict(page_table=V - 60)])
def test_cache_over_the_batch(nnb, built_lib, name, where):
    rc, text = _call(nnb, built_lib, name, **where)
    assert rc == nnb.NN_ERR_ARG and name.encode() in text and b"the cache overlaps the batch" in text, text


@pytest.mark.parametrize("where", [dict(cos=K), dict(sin=V + CELLS - 16), dict(cos=KS - 100 * 32 * 4 + 16), dict(sin=VS)])
def test_cache_over_the_rotation(nnb, built_lib, where):
    rc, text = _call(nnb, built_lib, "nn_rope_kv_write", **where)
    assert rc == nnb.NN_ERR_ARG and b"the cache overlaps" in text and b"cos" in text, text


@pytest.mark.parametrize("where", [{}, dict(row_start=K + CELLS), dict(kv_len=KS - 8), dict(page_table=VS + SCALES), dict(cos=K - 100 * 32 * 4), dict(sin=V + CELLS)])
def test_next_to_the_cache(nnb, built_lib, where):
    rc, text = _call(nnb, built_lib, "nn_rope_kv_write", **where)
    assert NO_CONTEXT in text, text


@pytest.mark.parametrize("name", ["nn_kv_read", "nn_attention"])
def test_reading_calls_do_not_mind(nnb, built_lib, name):
    assert NO_CONTEXT in _call(nnb, built_lib, name, row_start=K)[1]
