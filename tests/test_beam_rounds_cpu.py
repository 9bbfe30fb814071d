"""That the calls of the GPU test on many rounds have as many as they are meant to have."""
import ctypes

import numpy as np
import pytest

import branch_reference as br
from beam_rounds import KINDS, SHAPES, best_of, rows_of


@pytest.mark.parametrize("groups,beams,vocab,picks,segments,rounds", SHAPES)
def test_segments_and_rounds(built_lib, groups, beams, vocab, picks, segments, rounds):
    segs, per = ctypes.c_int(), ctypes.c_int()
    built_lib._ZN3nnb13beam_segmentsEiiiPiS0_(groups * beams, vocab, 148, ctypes.byref(segs), ctypes.byref(per))
    assert segs.value == segments
    vectors = -(-vocab // 8)
    assert -(-min(per.value, vectors) // 1024) == rounds
    assert groups * beams * segs.value <= 8192
    # rows are joined one by one, not by segments (four blocks for each SM, lists of 128 segments and 1024 candidates at most)
    assert groups * beams * segments > 4 * 148 or beams * segments > 128


@pytest.mark.parametrize("kind", KINDS)
def test_picks_of_rows_and_of_a_sort_agree(kind):
    logits, score = rows_of(kind, 3, 400, 151), np.array([-0.25, -0.5, -1.75], np.float32)
    for picks in (1, 7, 32):
        total, token, parent, near = best_of(logits, score, picks)
        want = br.best_continuations(logits, score, None, -1, picks)
        assert np.allclose(total, want[0], rtol=0, atol=1e-12) and np.array_equal(token, want[1]) and np.array_equal(parent, want[2]) and near == pytest.approx(want[3], abs=1e-12)
