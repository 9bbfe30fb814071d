"""The host side of a decode step's attention, on a context that only keeps account of its buffers."""
import importlib

import numpy as np
import pytest


class Account:
    """Sizes of what is allocated; an upload that passes its buffer's end is an error."""

    def __init__(self):
        self.next, self.size, self.caches = 1 << 12, {}, 0

    def alloc(self, n):
        self.next += 1 << 32
        self.size[self.next] = n
        return self.next

    def free(self, p):
        del self.size[p]

    def upload(self, a, buf=None):
        a = np.ascontiguousarray(a)
        buf = self.alloc(max(a.nbytes, 16)) if buf is None else buf
        assert a.nbytes <= self.size[buf], f"{a.nbytes} bytes into a buffer of {self.size[buf]}"
        return buf

    def kv_cache(self, *a):
        self.caches += 1
        return self

    def close(self):
        self.caches -= 1

    def kv_write(self, *a):
        pass

    sync = rope_kv_write = attention = lambda self, *a: None


def _modules():
    return (importlib.import_module("adreno_llms_b200." + m) for m in ("synth", "decode_step"))


@pytest.mark.parametrize("lengths", [[], [3], [3, 4, 5], [3, 4, 5, 6, 7, 8]])
def test_one_length_for_each_row(nnb, lengths):
    synth, dstep = _modules()
    shape = synth.ModelShape("tiny", 128, 2, 128, 64, 256, 64)
    c = Account()
    with pytest.raises(ValueError, match="lengths"):
        dstep.Attention(c, shape, 2, lengths)
    assert not c.size and not c.caches          # (refused before anything is made)
    at = dstep.Attention(c, shape, 2, [3, 4])
    with pytest.raises(ValueError, match="lengths"):
        at.set_lengths(lengths)
    assert list(at.lengths) == [3, 4]
    at.set_lengths([5, 0])
    at.advance()
    assert list(at.lengths) == [6, 1]


@pytest.mark.parametrize("cache,lengths", [("fp16", [3, 40]), ("int8", [0, 0]), ("fp8", [17, 0])])
def test_a_closed_attention_gives_its_buffers_back(nnb, cache, lengths):
    synth, dstep = _modules()
    c = Account()
    mine = c.alloc(64)
    at = dstep.Attention(c, synth.ModelShape("tiny", 128, 3, 128, 64, 256, 64), 2, lengths, cache=cache)
    assert c.caches == 3
    per_layer = 2 if cache == "fp16" else 4
    assert len(c.size) == 1 + 3 * per_layer + 6     # cells and scales; cos, sin, row starts, lengths, pages, output: not what filled the cache
    at.close()
    assert list(c.size) == [mine] and c.caches == 0
    at.close()                                      # (once more: nothing left to do)
    assert list(c.size) == [mine] and c.caches == 0
