"""How the 4-bit cache's and the verification's kernels read (no GPU)."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "miniserve_b200", "csrc")


@pytest.mark.parametrize("name", ["ms_kv.cuh", "ms_kv4.cu", "ms_kv4.cuh", "ms_attn4.cu", "ms_attn4.cuh", "ms_verify.cu"])
def test_dependent_grids_read_coherently(name):
    """They are launched while the grid before them may still write what they
    read: none uses the read-only path, by itself or by what the compiler may
    make of a pointer that promises it."""
    text = re.sub(r"//.*", "", open(os.path.join(CSRC, name)).read())
    assert not re.search(r"__ldg|ld\.global\.nc|__restrict__", text)
