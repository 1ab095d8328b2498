"""The batched token mixers' index arithmetic (csrc/q38_paged.hpp: rows of ragged batches, pages,
the split of attention's steps into shares) through the CPU test program tests/cpp/paged_test.cpp."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BIN = os.path.join(ROOT, "qwen38-flash.cpp_amd", "_build", "paged_test")


def test_index_arithmetic():
    assert os.path.exists(BIN), "paged_test is not built (make -C qwen38-flash.cpp_amd)"
    p = subprocess.run([BIN], capture_output=True, text=True, timeout=300)
    assert p.returncode == 0 and "checks passed" in p.stdout, p.stdout + p.stderr
