"""Drafted trees, moves and beams without a GPU: the masks' bits, and what the entry points refuse."""
import ctypes
import os
import subprocess

import pytest

from test_kv_cpu import BUF, K, NO_CONTEXT, OUT, Q, V, _batch, _create

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include "kv_index.h"
#include <cstdio>
#include <climits>
#include <vector>
using namespace nnb;
#define CHECK(c) do { if (!(c)) { printf("line %d: %s\n", __LINE__, #c); return 1; } } while (0)
int main() {
    for (int n = -3; n < 40; ++n) CHECK(low_bits32(n) == (n <= 0 ? 0u : n >= 32 ? ~0u : ~0u >> (32 - n)));
    unsigned x = 12345;
    for (int words : {1, 2, 3, 32}) {
        std::vector<uint32_t> mask(words);   // (exactly as long as it may be read: run with the address sanitizer)
        for (int turn = 0; turn < 3; ++turn) {
            for (uint32_t& w : mask) w = turn == 0 ? ~0u : turn == 1 ? 0u : (x = x * 1664525u + 1013904223u);
            for (int n : {0, 1, 31, 32, 33, 32 * words - 1, 32 * words}) for (int len : {n, n + 1, n + 31, n + 32, n + 500, n / 2}) {
                if (n > 32 * words) continue;
                const int base = len - n;   // (below 0 where the sequence is shorter than its rows)
                for (int at = 0; at < len + 200; at += 7) {
                    uint32_t want = 0;
                    for (int i = 0; i < 32; ++i) {
                        const int key = at + i;
                        if (key < len && (key < base || (mask[(key - base) / 32] >> ((key - base) % 32) & 1))) want |= 1u << i;
                    }
                    CHECK(tree_bits(mask.data(), words, at, base, len) == want);
                }
            }
        }
    }
    uint32_t one = 1;
    CHECK(tree_bits(&one, 1, 1 << 30, (1 << 30) - 1, 1 << 30) == 0);
    CHECK(tree_bits(&one, 1, 0, (1 << 30) - 1, 1 << 30) == ~0u);
    CHECK(tree_bits(&one, 1, (1 << 30) - 2, (1 << 30) - 1, 1 << 30) == 3u);
    return 0;
}
"""


def test_bits_of_a_mask(tmp_path):
    src, exe = tmp_path / "tree.cpp", tmp_path / "tree"
    src.write_text(PROGRAM)
    subprocess.check_call(["g++", "-std=c++17", "-Wall", "-Werror", "-fsanitize=undefined,address", "-fno-sanitize-recover", "-I",
                           os.path.join(REPO, "adreno-llms_b200", "csrc"), str(src), "-o", str(exe)])
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr


PARENT, MASK, POS, COS, SIN = 32 * BUF, 33 * BUF, 34 * BUF, 35 * BUF, 36 * BUF


def _layout(L, h, b, parent=PARENT, words=1, mask=MASK, position=POS):
    return L.nn_tree_layout(None, b, parent, words, mask, position)


def _tree(L, h, b, q_heads=4, q=Q, qs=0, out=OUT, os_=0, scale=0.125, words=1, mask=MASK):
    return L.nn_attention_tree(None, h, b, q_heads, q, qs, out, os_, scale, words, mask)


def _rope_at(L, h, b, position=POS, cos=COS, sin=SIN, n=100, rot=64, q_heads=4, q=Q, qs=0, qo=Q, qos=0, k=K, ks=0, v=V, vs=0):
    return L.nn_rope_kv_write_at(None, h, b, position, cos, sin, n, rot, q_heads, q, qs, qo, qos, k, ks, v, vs)


def _handles(*caches):
    return (ctypes.c_void_p * len(caches))(*(getattr(c, "value", c) for c in caches))


def _move(L, h, b, source=PARENT):
    return L.nn_kv_move(None, _handles(h), 1, b, source)


def _reorder(L, h, b, beams=2, parent=PARENT):
    return L.nn_kv_reorder(None, _handles(h), 1, b, beams, parent)


@pytest.mark.parametrize("call", [_layout, _tree, _rope_at, _move, _reorder])
@pytest.mark.parametrize("change,text", [
    ({}, NO_CONTEXT), (dict(num_seqs=0), NO_CONTEXT), (dict(num_seqs=-2), b"num_seqs"), (dict(max_len=0), b"max_len"), (dict(kv_len=None), b"null row_start"),
    (dict(kv_len=4 * BUF + 2), b"4-byte"),
])
def test_batches(nnb, built_lib, call, change, text):
    rc, h = _create(nnb, built_lib)
    assert rc == 0
    assert call(built_lib, h, _batch(nnb, **change)) == nnb.NN_ERR_ARG and text in built_lib.nn_last_error(), built_lib.nn_last_error()
    assert call(built_lib, h, None) == nnb.NN_ERR_ARG
    built_lib.nn_kv_cache_free(h)


@pytest.mark.parametrize("call", [_layout, _tree, _rope_at, _move])
@pytest.mark.parametrize("change,text", [
    (dict(num_rows=0, row_start=None), NO_CONTEXT), (dict(num_rows=-1), b"num_rows"), (dict(max_new=0), b"max_new"), (dict(row_start=None), b"null row_start"),
])
def test_batches_with_rows(nnb, built_lib, call, change, text):
    rc, h = _create(nnb, built_lib)
    assert call(built_lib, h, _batch(nnb, **change)) == nnb.NN_ERR_ARG and text in built_lib.nn_last_error(), built_lib.nn_last_error()
    built_lib.nn_kv_cache_free(h)


@pytest.mark.parametrize("call", [_tree, _rope_at, _move, _reorder])
@pytest.mark.parametrize("change,text", [
    (dict(table_stride=0), b"table_stride"), (dict(max_len=129), b"page table row"), (dict(max_len=128), NO_CONTEXT), (dict(page_table=None), b"null row_start"),
    (dict(page_table=5 * BUF + 2), b"4-byte"),
])
def test_batches_with_pages(nnb, built_lib, call, change, text):
    rc, h = _create(nnb, built_lib)
    assert call(built_lib, h, _batch(nnb, **change)) == nnb.NN_ERR_ARG and text in built_lib.nn_last_error(), built_lib.nn_last_error()
    built_lib.nn_kv_cache_free(h)


# cache: keys at BUF and values at 2 BUF of 16384 bytes; 6 rows of 2 sequences, row_start at 3 BUF, kv_len at 4 BUF, the table of 2 x 8 entries at 5 BUF
@pytest.mark.parametrize("call,change,code,text", [
    (_layout, dict(words=0), "UNSUPPORTED", b"mask_words"), (_layout, dict(words=33), "UNSUPPORTED", b"mask_words"), (_layout, dict(words=32), "ARG", NO_CONTEXT),
    (_layout, dict(parent=None), "ARG", b"null parent"), (_layout, dict(mask=None), "ARG", b"null parent"), (_layout, dict(position=None), "ARG", b"null parent"),
    (_layout, dict(mask=MASK + 2), "ARG", b"aligned"), (_layout, dict(mask=PARENT), "ARG", b"overlap"), (_layout, dict(position=PARENT + 20), "ARG", b"overlap"),
    (_layout, dict(position=PARENT + 24), "ARG", NO_CONTEXT), (_layout, dict(mask=POS - 20), "ARG", b"overlap"), (_layout, dict(mask=3 * BUF + 8), "ARG", b"overlap"),
    (_layout, dict(position=4 * BUF), "ARG", b"overlap"), (_layout, dict(mask=PARENT - 24), "ARG", NO_CONTEXT), (_layout, dict(mask=PARENT - 24, words=2), "ARG", b"overlap"),
    (_tree, dict(words=0), "UNSUPPORTED", b"mask_words"), (_tree, dict(mask=None), "ARG", b"mask"), (_tree, dict(mask=MASK + 1), "ARG", b"mask"),
    (_tree, dict(mask=OUT + 6 * 512 - 4), "ARG", b"overlaps the mask"), (_tree, dict(mask=OUT + 6 * 512), "ARG", NO_CONTEXT), (_tree, dict(q_heads=3), "ARG", b"multiple"),
    (_tree, dict(scale=0.0), "ARG", b"scale"), (_tree, dict(out=Q), "ARG", b"overlaps"), (_tree, dict(q=None), "ARG", b"q is null"), (_tree, dict(qs=255), "ARG", b"stride"),
    (_rope_at, dict(position=None), "ARG", b"position is null"), (_rope_at, dict(position=POS + 1), "ARG", b"aligned"), (_rope_at, dict(position=BUF + 64), "ARG", b"position"),
    (_rope_at, dict(position=Q + 512), "ARG", b"position"), (_rope_at, dict(rot=0), "ARG", b"rotary_dim"), (_rope_at, dict(cos=None), "ARG", b"cos"),
    (_move, dict(source=None), "ARG", b"source"), (_move, dict(source=PARENT + 2), "ARG", b"source"), (_move, dict(source=2 * BUF + 16380), "ARG", b"overlaps source"),
    (_move, dict(source=2 * BUF + 16384), "ARG", NO_CONTEXT),
    (_reorder, dict(beams=0), "UNSUPPORTED", b"beams"), (_reorder, dict(beams=33), "UNSUPPORTED", b"beams"), (_reorder, dict(beams=3), "ARG", b"multiple"), (_reorder, dict(beams=1), "ARG", NO_CONTEXT),
    (_reorder, dict(parent=None), "ARG", b"parent"), (_reorder, dict(parent=5 * BUF + 60), "ARG", b"page table"), (_reorder, dict(parent=5 * BUF + 64), "ARG", NO_CONTEXT),
    (_reorder, dict(parent=BUF), "ARG", b"overlaps parent"),
])
def test_operands(nnb, built_lib, call, change, code, text):
    rc, h = _create(nnb, built_lib)
    assert call(built_lib, h, _batch(nnb), **change) == getattr(nnb, "NN_ERR_" + code) and text in built_lib.nn_last_error(), built_lib.nn_last_error()
    built_lib.nn_kv_cache_free(h)


def test_more_rows_than_a_mask_has_bits(nnb, built_lib):
    rc, h = _create(nnb, built_lib)
    for call in (_layout, _tree):
        assert call(built_lib, h, _batch(nnb, max_new=33)) == nnb.NN_ERR_ARG and b"bits of a mask" in built_lib.nn_last_error()
        assert call(built_lib, h, _batch(nnb, max_new=33), words=2) == nnb.NN_ERR_ARG and NO_CONTEXT in built_lib.nn_last_error()
    built_lib.nn_kv_cache_free(h)


def test_caches_of_layers(nnb, built_lib):
    L, b = built_lib, _batch(nnb)
    _, one = _create(nnb, L)
    _, two = _create(nnb, L, k=10 * BUF, v=11 * BUF)
    _, other_page = _create(nnb, L, page=32, k=10 * BUF, v=11 * BUF)
    _, over = _create(nnb, L, k=12 * BUF, v=2 * BUF + 16368)
    _, more_heads = _create(nnb, L, heads=3, dim=128, k=14 * BUF, v=15 * BUF)
    _, fewer_pages = _create(nnb, L, fmt=1, pages=2, k=16 * BUF, v=17 * BUF, ks=18 * BUF, vs=19 * BUF)
    calls = [lambda *c: L.nn_kv_move(None, _handles(*c), len(c), b, PARENT), lambda *c: L.nn_kv_reorder(None, _handles(*c), len(c), b, 2, PARENT)]
    for call in calls:
        for caches, text in (((one, two), NO_CONTEXT), ((one, more_heads, fewer_pages, two), NO_CONTEXT), ((one, one), b"overlap"), ((two, one, over), b"overlap"),
                             ((one, other_page), b"pages of 32"), ((one, None), b"cache 1 is null")):
            assert call(*caches) == nnb.NN_ERR_ARG and text in L.nn_last_error(), (caches, L.nn_last_error())
    assert L.nn_kv_move(None, None, 1, b, PARENT) == nnb.NN_ERR_ARG and b"num_caches" in L.nn_last_error()
    assert L.nn_kv_move(None, None, -1, b, PARENT) == nnb.NN_ERR_ARG and b"num_caches" in L.nn_last_error()
    assert L.nn_kv_move(None, None, 0, b, PARENT) == nnb.NN_ERR_ARG and NO_CONTEXT in L.nn_last_error()      # nothing to do
    assert L.nn_kv_reorder(None, None, 0, b, 2, PARENT) == nnb.NN_ERR_ARG and b"no caches" in L.nn_last_error()
    # what a call writes must not be what tells it where to: the batch inside the second cache
    for bad in (dict(kv_len=10 * BUF + 64), dict(page_table=11 * BUF)):
        for call in (L.nn_kv_move, ):
            assert call(None, _handles(one, two), 2, _batch(nnb, **bad), PARENT) == nnb.NN_ERR_ARG and b"cache 1 overlaps" in L.nn_last_error()
        assert L.nn_kv_reorder(None, _handles(one, two), 2, _batch(nnb, **bad), 2, PARENT) == nnb.NN_ERR_ARG and b"cache 1 overlaps" in L.nn_last_error()
    assert L.nn_kv_reorder(None, _handles(one), 1, _batch(nnb, kv_len=5 * BUF + 32), 2, PARENT) == nnb.NN_ERR_ARG and b"overlaps kv_len" in L.nn_last_error()
    # of the batch only lengths and page table count
    assert L.nn_kv_reorder(None, _handles(one), 1, _batch(nnb, row_start=None, num_rows=0, max_new=0), 2, PARENT) == nnb.NN_ERR_ARG and NO_CONTEXT in L.nn_last_error()
    for c in (one, two, other_page, over, more_heads, fewer_pages):
        L.nn_kv_cache_free(c)


SCORE, DONE, O1, O2, O3, O4 = (BUF * i for i in range(40, 46))


# 3 groups of 4 beams of 1000 tokens, 8 picks
def _select(L, groups=3, beams=4, vocab=1000, logits=BUF, stride=0, score=SCORE, done=DONE, eos=2, picks=8, o1=O1, o2=O2, o3=O3, o4=O4):
    return L.nn_beam_select(None, groups, beams, vocab, logits, stride, score, done, eos, picks, o1, o2, o3, o4)


@pytest.mark.parametrize("change,code,text", [
    ({}, "ARG", NO_CONTEXT), (dict(groups=0), "ARG", NO_CONTEXT), (dict(groups=-1), "ARG", b"groups"), (dict(vocab=0), "ARG", b"vocab"),
    (dict(beams=0), "UNSUPPORTED", b"beams"), (dict(beams=33), "UNSUPPORTED", b"beams"), (dict(picks=0), "UNSUPPORTED", b"picks"), (dict(picks=33), "UNSUPPORTED", b"picks"),
    (dict(groups=2049, logits=1 << 30), "UNSUPPORTED", b"rows"), (dict(groups=2048, logits=1 << 30), "ARG", NO_CONTEXT), (dict(logits=None), "ARG", b"null logits"), (dict(score=None), "ARG", b"null logits"),
    (dict(o1=None), "ARG", b"null logits"), (dict(o2=None), "ARG", b"null logits"), (dict(o3=None), "ARG", b"null logits"), (dict(o4=None, done=None, eos=-1), "ARG", NO_CONTEXT),
    (dict(eos=-1), "ARG", b"eos"), (dict(eos=1000), "ARG", b"eos"), (dict(done=None, eos=-1), "ARG", b"eos"), (dict(o4=None, eos=-1), "ARG", b"eos"),
    (dict(logits=BUF + 1), "ARG", b"aligned"), (dict(logits=BUF + 2), "ARG", NO_CONTEXT), (dict(score=SCORE + 2), "ARG", b"aligned"), (dict(o3=O3 + 1), "ARG", b"aligned"),
    (dict(stride=999), "ARG", b"stride"), (dict(stride=-5), "ARG", b"stride"), (dict(stride=1001), "ARG", NO_CONTEXT),
    (dict(o2=O1 + 92), "ARG", b"outputs overlap"), (dict(o2=O1 + 96), "ARG", NO_CONTEXT), (dict(o4=O3), "ARG", b"outputs overlap"),
    (dict(o1=BUF + 23996), "ARG", b"overlaps logits"), (dict(o1=BUF + 24000), "ARG", NO_CONTEXT), (dict(o1=SCORE), "ARG", b"overlaps"), (dict(o1=SCORE, picks=4), "ARG", NO_CONTEXT),
    (dict(o2=SCORE, picks=4), "ARG", b"overlaps"), (dict(o4=DONE, picks=4), "ARG", NO_CONTEXT), (dict(o4=DONE), "ARG", b"overlaps"), (dict(o1=DONE, picks=4), "ARG", b"overlaps"),
    (dict(o1=SCORE + 4, picks=4), "ARG", b"overlaps"),
])
def test_beam_select_refusals(nnb, built_lib, change, code, text):
    assert _select(built_lib, **change) == getattr(nnb, "NN_ERR_" + code) and text in built_lib.nn_last_error(), built_lib.nn_last_error()
