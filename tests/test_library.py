"""The C-ABI library builds, loads and exports every symbol the header declares (no GPU)."""
import os
import re
import subprocess

import pytest

from miniserve_b200 import _lib, build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def declared_functions():
    text = open(os.path.join(ROOT, "include", "mssample.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    return sorted(set(re.findall(r"\b(ms_[a-z0-9_]+)\s*\(", text)))


def test_builds_and_exports_declared_symbols():
    build.build()
    L = _lib.lib()
    names = declared_functions()
    assert "ms_sample" in names
    for n in names:
        assert hasattr(L, n), n
        assert n in _lib.SIGNATURES, n
    assert L.ms_version() >= 100
    assert L.ms_error_string(-1).decode().startswith("invalid")


def test_binding_that_does_not_load_says_what_to_do(tmp_path, monkeypatch):
    """An extension of another torch fails in the loader, on a missing symbol:
    here one that needs a symbol that no library has."""
    source, made = tmp_path / "binding.c", tmp_path / "_binding.so"
    source.write_text("void *of_another_torch(void); void *PyInit__binding(void) { return of_another_torch(); }")
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", made, source], check=True)
    monkeypatch.setattr(_lib, "BINDING_PATH", str(made))
    monkeypatch.setattr(_lib, "_binding", None)
    with pytest.raises(_lib.SamplerLibraryError, match="build it again"):
        _lib.binding()
    made.unlink()
    with pytest.raises(_lib.SamplerLibraryError, match="is missing"):
        _lib.binding()


def test_dependent_grids_read_coherently():
    """The decode-step kernels are launched while the grid before them may
    still write what they read: none of them uses the read-only path."""
    csrc = os.path.join(ROOT, "miniserve_b200", "csrc")
    for name in ("ms_kv.cu", "ms_attn.cu", "ms_attn.cuh", "ms_int8.cu", "ms_tc.cuh"):
        text = re.sub(r"//.*", "", open(os.path.join(csrc, name)).read())
        assert not re.search(r"__ldg|ld\.global\.nc|__restrict__", text), name
