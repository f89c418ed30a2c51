"""What the K/V history's compiled parts assume of each other and of the memory they are given (no GPU)."""
import os
import re


CSRC = os.path.join(os.path.dirname(__file__), "..", "otter_amd", "csrc")


def test_shared_rows_that_vectors_read_are_aligned():
    """LDS arrays of floats whose rows are read and written 16 bytes at a time say so: a plain float array has 4-byte alignment."""
    src = open(os.path.join(CSRC, "attn_cache.hpp")).read()
    declared = re.findall(r"__shared__([^;]*?)\bfloat (\w+)\[", src)
    assert [n for _, n in declared].count("merge") == 2
    for attributes, name in declared:
        if name in ("red", "ls"):                                               # (one number at a time)
            continue
        assert "aligned(16)" in attributes, name
