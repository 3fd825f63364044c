"""Kernels that start while the one before them still runs (programmatic dependent launch) read memory by ordinary
loads, which their wait orders, and not by the non-coherent path, which wants memory that nothing writes meanwhile."""
import re

import pytest

from npu_b200 import build

FILES = sorted(p.name for p in build.CSRC.glob("*.cu")) + sorted(p.name for p in build.CSRC.glob("*.cuh"))


@pytest.mark.parametrize("name", FILES)
def test_no_load_takes_the_non_coherent_path(name):
    code = re.sub(r"//[^\n]*|/\*.*?\*/", "", (build.CSRC / name).read_text(), flags=re.S)
    # __restrict__ with const lets the compiler choose that path by itself.
    assert not re.findall(r"__ldg\b|ld\.global\.nc|__restrict__", code)
