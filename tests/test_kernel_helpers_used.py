"""Nothing stays in the headers of the kernels that no kernel calls."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flat-attention_b200", "csrc")
SOURCES = {os.path.basename(f): re.sub(r"//[^\n]*", "", open(f).read()) for f in glob.glob(os.path.join(CSRC, "*.cu*"))}


@pytest.mark.parametrize("header", sorted(f for f in SOURCES if f.startswith(("tree", "turns")) and f.endswith(".cuh")))
def test_every_helper_of_the_serving_kernels_is_called(header):
    names = re.findall(r"(?:__forceinline__|inline)\s+[\w:]+\s+(\w+)\s*\(", SOURCES[header])
    assert names
    everything = "".join(SOURCES.values())
    for name in names:
        defined = len(re.findall(r"(?:__forceinline__|inline)\s+[\w:]+\s+%s\s*\(" % name, everything))
        assert len(re.findall(r"\b%s\s*(?:<[^;(){}]*>)?\s*\(" % name, everything)) > defined, name
