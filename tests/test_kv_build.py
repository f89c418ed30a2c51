"""What the K/V history's compiled parts assume of each other and of the memory they are given (no GPU)."""
import os
import re
import types

import pytest

import otter_amd
from otter_amd import _lib

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


@pytest.mark.parametrize("version", [None, _lib.ABI_VERSION - 1, _lib.ABI_VERSION + 1])
def test_a_binding_of_another_version_is_refused(monkeypatch, version):
    """The binding has the C structs' layouts compiled in: one that was built for another version of them is not given the library's addresses."""
    bound = []
    other = types.SimpleNamespace(bind=lambda *a: bound.append(a), **({} if version is None else {"ABI_VERSION": version}))
    monkeypatch.setattr(_lib, "_binding", None)
    monkeypatch.setattr(otter_amd, "_kv_binding", other, raising=False)
    with pytest.raises(_lib.OtterHipError, match="make -C otter_amd/csrc"):
        _lib.kv_binding()
    assert not bound and _lib._binding is None
    monkeypatch.undo()
    assert _lib.kv_binding().ABI_VERSION == _lib.ABI_VERSION


def test_build_compiles_what_is_already_there(monkeypatch):
    """build() is the check that the sources compile: objects that exist do not count as built."""
    import __graft_entry__ as entry
    ran = []
    monkeypatch.setattr(entry.subprocess, "run", lambda cmd, **kw: ran.append((cmd, kw)))
    entry.build()
    (cmd, kw), = ran
    assert cmd[0] == "make" and "-B" in cmd and kw.get("check") is True
