"""Orderings inside the beam selection that no run can show to be missing, stated over the kernel's source."""
import re

from test_kernel_order_cpu import block_after, source


def test_the_flag_of_the_last_block_is_written_behind_barriers_alone():
    """last_of ends with every thread's read of the flag and no barrier, and it may be called twice: what writes the flag otherwise would be seen by a warp
    that is late (its block would leave as if others were still to come).  Its own write stands behind its first barrier."""
    s = source("beam.cu")
    body = block_after(s, "bool last_of(unsigned* counter, unsigned n, volatile int* flag)")
    assert body.lstrip("{").lstrip().startswith("__syncthreads();")
    assert body.index("__syncthreads();") < body.index("*flag =") < body.rindex("__syncthreads();") < body.index("return *flag")
    kernel = block_after(s, "beam_select_kernel(const BeamSelectArgs a)")
    uses = re.findall(r"[^;{}]*\bflag\b[^;{}]*", kernel)
    assert len(uses) >= 3
    for use in uses:
        assert re.search(r"__shared__ int flag\b", use) or re.search(r"last_of\([^()]*(\([^()]*\)[^()]*)*&flag\)", use), use


def test_the_bar_is_set_before_and_read_behind_barriers():
    """The bar of the shares' largest values: set to none by one thread, raised by one, read by all, with a barrier between each two."""
    kernel = block_after(source("beam.cu"), "beam_select_kernel(const BeamSelectArgs a)")
    uses = [m.start() for m in re.finditer(r"\bbar\b", kernel)][1:]      # (the first is its declaration)
    assert len(uses) == 3
    for a, b in zip(uses, uses[1:]):
        assert "__syncthreads();" in kernel[a:b]
