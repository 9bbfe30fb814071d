"""The key/value cache and the attention without a GPU: index arithmetic on bad pages and lengths, and what the entry points refuse."""
import ctypes
import os
import subprocess

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include "kv_index.h"
#include <cstdio>
#include <climits>
#include <vector>
using namespace nnb;
#define CHECK(c) do { if (!(c)) { printf("line %d: %s\n", __LINE__, #c); return 1; } } while (0)
int main() {
    const int odd[] = {INT_MIN, -1000, -1, 0, 1, 5, 16, 39, 40, 41, 1000, INT_MAX};
    for (int s : odd) for (int e : odd) for (int n : odd) {
        const SeqExtent x = seq_extent(s, e, n, 40, 64);
        CHECK(0 <= x.row0 && x.row0 <= x.row1 && x.row1 <= 40 && 0 <= x.len && x.len <= 64);
        CHECK(x.bad == (n < 0 || n > 64 || s < 0 || e < s || e > 40));
        if (s >= 0 && s <= e && e <= 40) CHECK(x.row0 == s && x.row1 == e);
    }
    for (int p : odd) CHECK(page_ok(p, 40) == (p >= 0 && p < 40));
    // cells beyond 2^31 rows and 2^32 bytes
    CHECK(cell_row(1 << 20, 7, 255, 8, 8) == ((((int64_t)1 << 20) * 8 + 7) << 8) + 255);
    CHECK(cell_row(0x7FFFFF, 0, 0, 8, 5) * 128 * 2 == (int64_t)0x7FFFFF * 8 * 32 * 256);
    // the tiles of a range of queries: every visible key lies in one, none comes twice, none is without a visible key
    const int windows[] = {0, 1, 2, 15, 16, 17, 64, 1000, INT_MAX}, sinks[] = {0, 1, 4, 16, 17, 100, INT_MAX};
    for (int tile : {16, 32, 128}) for (int p0 = -3; p0 < 150; p0 += 7) for (int n : {1, 3, 20}) for (int w : windows) for (int k : sinks) {
        const int p1 = p0 + n - 1;
        const TileRange r = visible_tiles(p0, p1, w, k, tile);
        std::vector<int> hit(200 / tile + 2, 0), want(hit);
        for (int i = 0; i < r.tiles(); ++i) { const int t = r.tile_at(i); CHECK(t >= 0 && t < (int)hit.size()); hit[t]++; CHECK(i == 0 || t > r.tile_at(i - 1)); }
        for (int p = p0; p <= p1; ++p) for (int key = 0; key <= p; ++key) if (key_visible(key, p, w, w ? k : 0)) want[key / tile] = 1;
        for (size_t t = 0; t < hit.size(); ++t) CHECK(hit[t] <= 1 && hit[t] >= want[t]);
        if (p0 >= 0) for (size_t t = 0; t < hit.size(); ++t) CHECK(hit[t] == want[t]);
    }
    CHECK(visible_tiles(-5, -1, 0, 0, 16).tiles() == 0);
    CHECK(visible_tiles(INT_MAX - 1, INT_MAX - 1, 0, 0, 128).end == 1 << 24);
    return 0;
}
"""


def test_index_arithmetic(tmp_path):
    src, exe = tmp_path / "kv_index.cpp", tmp_path / "kv_index"
    src.write_text(PROGRAM)
    subprocess.check_call(["g++", "-std=c++17", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover", "-I",
                           os.path.join(REPO, "adreno-llms_b200", "csrc"), str(src), "-o", str(exe)])
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr


BUF = 1 << 20     # (an address: nothing is read)


def _create(nnb, L, fmt=0, pages=4, page=16, heads=2, dim=64, k=BUF, v=2 * BUF, ks=None, vs=None):
    h = ctypes.c_void_p()
    rc = L.nn_kv_cache_create(None, fmt, pages, page, heads, dim, k, v, ks, vs, ctypes.byref(h))
    assert (rc == 0) == bool(h.value)
    return rc, h


@pytest.mark.parametrize("change,code,text", [
    (dict(fmt=3), "ARG", b"format"), (dict(pages=0), "ARG", b"num_pages"), (dict(heads=-1), "ARG", b"kv_heads"),
    (dict(page=8), "UNSUPPORTED", b"page_size"), (dict(page=48), "UNSUPPORTED", b"page_size"), (dict(page=512), "UNSUPPORTED", b"page_size"),
    (dict(dim=80), "UNSUPPORTED", b"head_dim"), (dict(dim=256), "UNSUPPORTED", b"head_dim"), (dict(pages=1 << 27, heads=8), "UNSUPPORTED", b"cells"),
    (dict(k=None), "ARG", b"null pages"), (dict(v=None), "ARG", b"null pages"), (dict(k=BUF + 8), "ARG", b"aligned"),
    (dict(fmt=1), "ARG", b"scale"), (dict(fmt=2, ks=BUF), "ARG", b"scale"), (dict(vs=BUF), "ARG", b"no scale"), (dict(fmt=1, ks=BUF, vs=BUF + 2), "ARG", b"aligned"),
    (dict(v=BUF + 4 * 16 * 2 * 64 * 2 - 16), "ARG", b"overlap"), (dict(v=BUF - 16), "ARG", b"overlap"), (dict(fmt=1, ks=3 * BUF, vs=3 * BUF + 240), "ARG", b"overlap"),
    (dict(fmt=2, ks=BUF + 16, vs=3 * BUF), "ARG", b"overlap"), (dict(fmt=2, ks=3 * BUF, vs=2 * BUF), "ARG", b"overlap"),
])
def test_cache_refusals(nnb, built_lib, change, code, text):
    rc, _ = _create(nnb, built_lib, **change)
    assert rc == getattr(nnb, "NN_ERR_" + code) and text in built_lib.nn_last_error()


def _batch(nnb, **change):
    d = dict(num_seqs=2, num_rows=6, max_new=3, max_len=100, table_stride=8, row_start=3 * BUF, kv_len=4 * BUF, page_table=5 * BUF)
    d.update(change)
    return nnb.KVBatch(**d)


Q, K, V, OUT = 64 * BUF, 65 * BUF, 66 * BUF, 67 * BUF


def _attention(L, h, b, q_heads=4, q=Q, qs=0, out=OUT, os_=0, scale=0.125, window=0, sinks=0):
    return L.nn_attention(None, h, b, q_heads, q, qs, out, os_, scale, window, sinks)


def _rope(L, h, b, cos=8 * BUF, sin=9 * BUF, n=100, rot=64, q_heads=4, q=Q, qs=0, qo=Q, qos=0, k=K, ks=0, v=V, vs=0):
    return L.nn_rope_kv_write(None, h, b, cos, sin, n, rot, q_heads, q, qs, qo, qos, k, ks, v, vs)


def _read(L, h, b, k=K, ks=0, v=V, vs=0):
    return L.nn_kv_read(None, h, b, k, ks, v, vs)


def _write(L, h, b, k=K, ks=0, v=V, vs=0):
    return L.nn_kv_write(None, h, b, k, ks, v, vs)


NO_CONTEXT = b"null context"


@pytest.mark.parametrize("call", [_attention, _rope, _read, _write])
@pytest.mark.parametrize("change,text", [
    ({}, NO_CONTEXT), (dict(num_seqs=0), NO_CONTEXT), (dict(num_rows=0, row_start=None), NO_CONTEXT), (dict(num_seqs=-1), b"num_seqs"), (dict(num_rows=-1), b"num_rows"),
    (dict(max_new=0), b"max_new"), (dict(max_len=0), b"max_len"), (dict(table_stride=0), b"table_stride"), (dict(max_len=129), b"page table row"),
    (dict(max_len=128), NO_CONTEXT), (dict(table_stride=1 << 30, max_len=1 << 30, page_table=1 << 40), NO_CONTEXT),
    (dict(row_start=None), b"null row_start"), (dict(kv_len=None), b"null row_start"), (dict(page_table=None), b"null row_start"), (dict(kv_len=4 * BUF + 2), b"4-byte"),
])
def test_batch_refusals(nnb, built_lib, call, change, text):
    rc, h = _create(nnb, built_lib)
    assert rc == 0
    assert call(built_lib, h, _batch(nnb, **change)) == nnb.NN_ERR_ARG and text in built_lib.nn_last_error()
    assert call(built_lib, None, _batch(nnb)) == nnb.NN_ERR_ARG and call(built_lib, h, None) == nnb.NN_ERR_ARG
    assert built_lib.nn_kv_cache_free(h) == 0 and built_lib.nn_kv_cache_free(None) == 0


# dense rows: q 4 x 64 values, k and v 2 x 64; 6 rows
@pytest.mark.parametrize("call,change,text", [
    (_attention, dict(q_heads=3), b"multiple"), (_attention, dict(q_heads=0), b"multiple"), (_attention, dict(q=None), b"q is null"), (_attention, dict(out=None), b"out is null"),
    (_attention, dict(q=Q + 8), b"aligned"), (_attention, dict(qs=255), b"stride"), (_attention, dict(qs=260), b"stride"), (_attention, dict(os_=-256), b"stride"),
    (_attention, dict(scale=0.0), b"scale"), (_attention, dict(scale=-1.0), b"scale"), (_attention, dict(scale=float("inf")), b"scale"), (_attention, dict(scale=float("nan")), b"scale"),
    (_attention, dict(window=-1), b"window"), (_attention, dict(sinks=-1), b"sinks"), (_attention, dict(out=Q), b"overlaps"), (_attention, dict(out=Q + 16), b"overlaps"),
    (_attention, dict(out=Q + 6 * 512), NO_CONTEXT), (_attention, dict(out=Q + 512, qs=512, os_=512), NO_CONTEXT), (_attention, dict(out=Q + 496, qs=512, os_=512), b"overlaps"),
    (_attention, dict(out=BUF), b"overlaps"), (_attention, dict(out=3 * BUF), b"overlaps"), (_attention, dict(out=4 * BUF), b"overlaps"),
    (_attention, dict(out=5 * BUF + 48), b"overlaps"), (_attention, dict(out=5 * BUF + 64), NO_CONTEXT), (_rope, dict(qo=5 * BUF), b"overlaps"), (_read, dict(k=4 * BUF), b"overlap"),
    (_rope, dict(qo=8 * BUF), b"q_out overlaps cos"), (_rope, dict(qo=9 * BUF + 12784), b"q_out overlaps cos"), (_rope, dict(qo=9 * BUF + 12800), NO_CONTEXT),
    (_rope, dict(rot=0), b"rotary_dim"), (_rope, dict(rot=8), b"rotary_dim"), (_rope, dict(rot=80), b"rotary_dim"), (_rope, dict(cos=None), b"cos"), (_rope, dict(sin=9 * BUF + 4), b"cos"),
    (_rope, dict(n=0), b"table_len"), (_rope, dict(q=None), b"q_heads"), (_rope, dict(q_heads=0), b"q_heads"), (_rope, dict(qo=None), b"q_heads"),
    (_rope, dict(q_heads=0, q=None, qo=None), NO_CONTEXT), (_rope, dict(qo=Q + 16), b"q_out overlaps"), (_rope, dict(qo=K), b"q_out overlaps"), (_rope, dict(qo=2 * BUF), b"q_out overlaps"),
    (_rope, dict(qs=512, qos=512, ks=512, vs=512, k=Q + 512, v=Q + 768), NO_CONTEXT), (_rope, dict(qs=512, qos=512, ks=512, vs=512, k=Q + 496, v=Q + 768), b"q_out overlaps"),
    (_rope, dict(k=BUF), b"lies in the cache"), (_write, dict(v=2 * BUF + 1024), b"lies in the cache"), (_write, dict(k=None), b"k is null"), (_write, dict(vs=120), b"stride"),
    (_read, dict(v=K), b"overlap"), (_read, dict(k=2 * BUF), b"overlap"), (_read, dict(v=K + 256, ks=256, vs=256), NO_CONTEXT), (_read, dict(v=V + 2), b"aligned"),
])
def test_operand_refusals(nnb, built_lib, call, change, text):
    rc, h = _create(nnb, built_lib)
    assert call(built_lib, h, _batch(nnb), **change) == nnb.NN_ERR_ARG and text in built_lib.nn_last_error(), built_lib.nn_last_error()
    built_lib.nn_kv_cache_free(h)


MIRROR = r"""
#include "nnopt_linear.hpp"
int main() {
    nn_kv_cache* cache = nullptr;
    if (nn_kv_cache_create(nullptr, NN_KV_FP16, 4, 16, 2, 64, (nn_buf)0x100000, (nn_buf)0x200000, nullptr, nullptr, &cache) != NN_OK) return 1;
    nn_kv_batch b = {1, 1, 1, 64, 4, (nn_buf)0x300000, (nn_buf)0x400000, (nn_buf)0x500000};
    nn_buf q = (nn_buf)0x4000000, k = (nn_buf)0x5000000, v = (nn_buf)0x6000000, out = (nn_buf)0x7000000, cos = (nn_buf)0x8000000, sin = (nn_buf)0x9000000;
    // (without a context every call is refused)
    if (nnopt::fused_rope_kvwrite_m1(nullptr, cache, &b, cos, sin, 64, 64, 4, q, k, v)) return 2;
    if (nnopt::fused_decode_attn_m1(nullptr, cache, &b, 4, q, out, 0.125f)) return 3;
    return nn_kv_cache_free(cache) == NN_OK ? 0 : 4;
}
"""


def test_cpp_mirror_of_rotation_and_attention(built_lib, tmp_path):
    src, exe = tmp_path / "mirror.cpp", tmp_path / "mirror"
    src.write_text(MIRROR)
    base = os.path.join(REPO, "adreno-llms_b200")
    subprocess.check_call(["g++", "-std=c++17", "-Wall", "-Werror", "-I", os.path.join(base, "host"), str(src), "-o", str(exe), "-L" + os.path.join(base, "lib"),
                           "-lnnopt_b200", "-Wl,-rpath," + os.path.join(base, "lib")])
    assert subprocess.run([str(exe)]).returncode == 0
