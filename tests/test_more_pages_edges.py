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


@pytest.fixture()
def cache():
    from orangu_b200 import PagedCache

    be = type("B", (), {})()
    be._h, be._lib = 1, Recorder()
    pool = On((2, 9, 2, 9 * 64), "torch.uint8")
    return PagedCache(be, pool, pool, On((3, 4), "torch.int32"))


class On(Fake):
    def __init__(self, shape, dtype, device="cuda:0"):
        super().__init__(shape, dtype)
        self.device = device


def test_weights_are_checked_before_anything_moves(cache):
    """keep() moves keys and values by one call and weights by another: weights that the second would refuse are refused before the first."""
    i32 = lambda *s: On(s, "torch.int32")  # noqa: E731
    calls = cache._lib.calls
    n = len(calls)
    for bad in (On((2, 2, 2, 63), "torch.float32"), On((2, 2, 2, 64), "torch.float32", "cpu"), On((2, 2, 2, 64), "torch.float32", "cuda:1")):
        for call in (lambda: cache.keep(i32(2), i32(2, 5), i32(2), mass=bad), lambda: cache.evict(i32(2), bad, i32(2, 2, 2, 4), i32(2), 9)):
            with pytest.raises(ValueError):
                call()
    q = On((5, 4, 64), "torch.bfloat16")
    with pytest.raises(ValueError):
        cache.attention_tokens(q, i32(3), i32(2), 0.1, q, 3, 10, mass=On((2, 2, 63), "torch.float32"))
    assert len(calls) == n
    cache.keep(i32(2), i32(2, 5), i32(2), mass=On((2, 2, 2, 64), "torch.float32"))
    assert [name for name, _ in calls[n:]] == ["ob_pages_keep", "ob_pages_keep_mass"]
