"""Rules of the dense operators' kernels that no run can show: read in their sources (no GPU needed)."""
import os
import re

import pytest

import apoe

CSRC = os.path.join(os.path.dirname(os.path.abspath(apoe.__file__)), "csrc")


def code(name):
    """A source without its comments."""
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*|/\*.*?\*/", "", f.read(), flags=re.S)


@pytest.mark.parametrize("name", ["apoe_dense.cu", "apoe_tile.cuh"])
def test_kernels_that_start_early_load_coherently(name):
    """A kernel started by a programmatic launch runs while its predecessor still writes: a non-coherent load (of memory that
    nothing writes while the kernel runs) of that data is wrong even after the wait."""
    text = code(name)
    assert "griddepcontrol" in text or "pdl_wait" in text
    for word in ("__ldg", "ld.global.nc", "__restrict__", "__restrict"):
        assert not re.search(r"(?<![\w.])" + re.escape(word) + r"(?!\w)", text), word
