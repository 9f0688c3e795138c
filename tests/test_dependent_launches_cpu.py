"""Kernels that are always launched as dependents let the next launch in behind their own wait: a caller may put one of them between a
kernel that prepares weights and a launch that reads weights ahead of its wait."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "turbopi_b200" / "csrc"


@pytest.mark.parametrize("source,kernels", [("paged_cache.cu", 2), ("paged_attention.cu", 2), ("packed_attention.cu", 1)])
def test_the_wait_comes_first(source, kernels):
    text = re.sub(r"//[^\n]*", "", (CSRC / source).read_text())
    bodies = re.findall(r"__global__[^{;]*\{\n(.*?)^\}", text, re.S | re.M)
    assert len(bodies) == kernels
    for body in bodies:
        wait = body.index("pdl_wait_prior_grids()")
        assert wait < body.index("pdl_launch_dependents()")
        assert not re.search(r"P\.(cu|cache\.(table|lengths|k_pages|v_pages)|joins|part_\w+|q|k|v)\b\[", body[:wait])
