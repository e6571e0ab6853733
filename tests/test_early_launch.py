"""Kernels that begin before the stream's previous kernel has ended read what it
wrote. Non-coherent loads are defined only for memory that nothing writes during
the kernel's life, which here began before the writer's end, so none is used
(read from the sources: no input shows a stale line on demand)."""

from __future__ import annotations

import re

import pytest

from moe_serving_profile_b200.build import CSRC

EARLY = sorted(p.name for p in CSRC.glob("*.cu") if re.search(r"grid_dep_(wait|begin)\(", p.read_text()))


def test_the_early_kernels_are_found():
    assert {"int8.cu", "norm.cu", "route.cu"} <= set(EARLY)


@pytest.mark.parametrize("name", EARLY)
def test_no_non_coherent_loads(name):
    code = re.sub(r"//[^\n]*|/\*.*?\*/", "", (CSRC / name).read_text(), flags=re.S)
    # __restrict__ lets the compiler choose such loads by itself
    assert not re.findall(r"__ldg|ld\.global(?:\.\w+)*\.nc|__restrict__", code)
