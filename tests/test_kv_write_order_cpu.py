"""What a write to the key/value cache reads of its operands, stated over the kernel's source (reads of rows that count for nothing change no result)."""
import re

from test_kernel_order_cpu import block_after, source


def test_rows_of_no_sequence_are_not_read():
    """Rows behind the last sequence and before the first one are neither read nor written: loads of queries, keys and values stand behind the end of the threads of such rows."""
    body = block_after(source("kv_cache.cu"), "kv_write_kernel(const KvWriteArgs a)")
    end = body.index("if (at.none) return;")
    reading = body.index("auto load = [&]")
    inside = body[reading:reading + len(block_after(body, "auto load = [&]")) + body[reading:].index("{")]
    assert all(re.search(r"a\.%s\b" % x, inside) for x in "qkv")      # (the loads are in there)
    calls = [m.start() for m in re.finditer(r"\bload\(", body)]
    assert calls and min(calls) > end
    rest = body.replace(inside, "")
    assert not re.search(r"a\.[qkv] \+", rest)
