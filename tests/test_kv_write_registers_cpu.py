"""How many blocks of the cache writes an SM holds: where that is one fewer, whole ranges of row counts need another round of blocks (1200 to 2700 rows of 48 heads took 4 to 12 % longer)."""
import os
import re
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "adreno-llms_b200", "csrc")


def test_registers_of_rows_in_four_warps(nnb, tmp_path):
    r = subprocess.run(["nvcc", "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17", "-Xcompiler", "-fPIC", "-Xptxas", "-v", "-x", "cu", "-c",
                        os.path.join(CSRC, "kv_cache.cu"), "-o", str(tmp_path / "kv_cache.o")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    found = re.findall(r"Compiling entry function '\w*kv_write_kernelILi(\d)ELi(\d+)ELb(\d)E.*?(\d+) bytes spill stores.*?Used (\d+) registers", r.stderr, re.S)
    assert len(found) == 12
    for fmt, dim, spread, spilled, registers in found:
        assert spilled == "0", (fmt, dim, spread)
        if spread == "1":      # 128 threads: nine blocks of fp16 rows, eight of rows that are quantised
            assert int(registers) <= (56 if fmt == "0" else 64), (fmt, dim, registers)
