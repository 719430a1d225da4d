"""4-bit pages, weights per position, cut caches and verified drafts where they went wrong once, as far as that goes without a GPU."""
import os
import re

import pytest

from test_pages import Fake, Recorder

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "orangu_b200", "csrc")


def test_registers_change_hands_once_a_warpgroup():
    """All warps of a warpgroup have to execute the same setmaxnreg: a kernel has one that gives and one that takes, each ahead of any role's branch."""
    found = 0
    for name in sorted(os.listdir(CSRC)):
        if not name.endswith((".cu", ".cuh")):
            continue
        for kernel in re.split(r"\b__global__\b", open(os.path.join(CSRC, name)).read())[1:]:
            sites = re.findall(r"setmaxnreg\.(inc|dec)", kernel)
            assert sorted(sites) in ([], ["dec", "inc"]), (name, sites)
            found += len(sites)
    assert found == 2
