"""4-bit pages, attention of new tokens, cut caches and verified drafts, as far as they go without a GPU: the plain statements, refusals that come before any
device call, and what the Python class checks itself."""
import ctypes as C
import itertools
import os

import numpy as np
import pytest

import more_pages_plain as more
from test_pages import Fake, Recorder

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    from orangu_b200 import build, capi

    build.build_all()
    return capi.load()


def test_constants_and_null_handles(lib):
    from orangu_b200 import capi

    text = open(os.path.join(ROOT, "include", "orangu_b200.h")).read()
    assert f"#define OB_TYPE_Q4_PAGES {capi.TYPE_Q4_PAGES}u" in text
    for name in ("ob_pages_store", "ob_pages_load", "ob_pages_attention_tokens", "ob_pages_evict", "ob_pages_keep_mass", "ob_drafts_verify"):
        zeros = [None if a is C.c_void_p else 0 if a is not C.c_float else 0.5 for a in capi.SIGNATURES[name][1]]
        assert getattr(lib, name)(*zeros) == -1, name


def test_python_checks():
    from orangu_b200 import PagedCache, verify_drafts

    be = type("B", (), {})()
    be._h, be._lib = 1, Recorder()
    pool, tables = (2, 9, 2, 9 * 64), Fake((3, 4), "torch.int32")
    for bad in (dict(k=Fake((2, 9, 2, 100), "torch.uint8")), dict(k=Fake(pool, "torch.int8")), dict(v=Fake((2, 9, 2, 9 * 128), "torch.uint8")), dict(v=Fake(pool, "torch.float16"))):
        with pytest.raises(ValueError):
            PagedCache(be, **{**dict(k=Fake(pool, "torch.uint8"), v=Fake(pool, "torch.uint8"), tables=tables), **bad})
    c = PagedCache(be, Fake(pool, "torch.uint8"), Fake(pool, "torch.uint8"), tables)
    assert (c.n_layer, c.n_pages, c.n_head_kv, c.head_dim) == (2, 9, 2, 64)
    i32 = lambda *s: Fake(s, "torch.int32")  # noqa: E731
    q, out, kv = Fake((5, 4, 64), "torch.bfloat16"), Fake((5, 4, 64), "torch.bfloat16", False), Fake((5, 2, 64), "torch.bfloat16")
    c.attention_tokens(q, i32(3), i32(2), 0.1, out, 3, 10, mass=Fake((2, 2, 70), "torch.float32"), stream=0)
    name, args = be._lib.calls[-1]
    assert name == "ob_pages_attention_tokens" and args[2] == 2 and args[4] == 30 and args[5] == 256 and args[9] is None and args[15] == 264 and args[17] == 70 and args[-1] == 1
    c.store(kv, kv, i32(3), i32(2), 4)
    assert be._lib.calls[-1][0] == "ob_pages_store" and be._lib.calls[-1][1][5:8] == (30, 128, 128) and be._lib.calls[-1][1][-1] is None
    c.keep(i32(2), i32(2, 5), i32(2), mass=Fake((2, 2, 2, 64), "torch.float32"))
    assert [n for n, _ in be._lib.calls[-2:]] == ["ob_pages_keep", "ob_pages_keep_mass"]
    n = len(be._lib.calls)
    good = dict(q=q, first_token=i32(3), n_ctx=i32(2), scale=0.1, out=out, max_tokens=3, max_context=10)
    for bad in (dict(q=Fake((5, 4, 64), "torch.float32")), dict(q=Fake((5, 4, 128), "torch.bfloat16")), dict(out=Fake((5, 4, 64), "torch.float16")), dict(first_token=i32(2)), dict(n_ctx=Fake((2,), "torch.int64")),
                dict(visible=Fake((4,), "torch.int64")), dict(mass=Fake((3, 2, 64), "torch.float32")), dict(mass=Fake((2, 2, 64), "torch.float16"))):
        with pytest.raises(ValueError):
            c.attention_tokens(**{**good, **bad})
    m = Fake((2, 2, 2, 64), "torch.float32")
    for call in (lambda: c.store(kv, Fake((4, 2, 64), "torch.bfloat16"), i32(3), i32(2), 4), lambda: c.store(q, q, i32(3), i32(2), 4), lambda: c.load(kv, Fake((5, 2, 64), "torch.float16"), i32(3), i32(2), 4),
                 lambda: c.load(Fake((5, 2, 64), "torch.float32"), Fake((5, 2, 64), "torch.float32"), i32(3), i32(2), 4), lambda: c.evict(i32(2), m, i32(2, 2, 2), i32(2), 9), lambda: c.evict(i32(2), m, i32(1, 2, 2, 4), i32(2), 9),
                 lambda: c.evict(i32(2), m, i32(2, 2, 2, 4), i32(3), 9), lambda: c.keep(i32(2), i32(2, 5), i32(2), mass=Fake((1, 2, 2, 64), "torch.float32")), lambda: c.attention_tree(q, i32(3), i32(2), i32(5), 0.1, q, 3, 3)):
        with pytest.raises(ValueError):
            call()

    class Rows(Fake):
        def stride(self):
            return (self.shape[1] + 3, 1)

    p, f = Rows((6, 10), "torch.float32"), Fake((6,), "torch.float32")
    verify_drafts(be, p, None, i32(6), i32(6), i32(3), f, i32(2, 64), i32(2), i32(2), stream=7)
    name, args = be._lib.calls[-1]
    assert name == "ob_drafts_verify" and args[1:5] == (2, 6, 10, 0) and args[6] == 13 and args[7] is None and args[-1] == 7
    n += 1
    for bad in (dict(target=Rows((6, 10), "torch.float64")), dict(draft=Rows((6, 9), "torch.float32")), dict(draft=Rows((6, 10), "torch.float16")), dict(tokens=i32(5)), dict(parent=Fake((6,), "torch.int64")),
                dict(uniform=Fake((6,), "torch.float64")), dict(kept=i32(3, 64)), dict(kept=i32(64)), dict(n_kept=i32(3)), dict(next_token=i32(1))):
        with pytest.raises(ValueError):
            verify_drafts(be, **{**dict(target=p, draft=p, tokens=i32(6), parent=i32(6), first_token=i32(3), uniform=f, kept=i32(2, 64), n_kept=i32(2), next_token=i32(2)), **bad})
    assert len(be._lib.calls) == n  # nothing reached the library


# ---------------------------------------------------------------------------------------- the plain statements themselves
def test_plain_codes():
    """Entries are whole numbers from -8 to 7 of a unit that is an f16 number of 7 significant bits; kept again they are the same."""
    r = np.random.default_rng(0)
    for scale in (1e-7, 1e-4, 1.0, 300.0, 1e5):
        x = r.standard_normal((50, 64)) * scale
        y = more.in_four_bits(x)
        assert np.array_equal(y.astype(np.float16).astype(np.float64), y) and np.array_equal(more.in_four_bits(y), y) or scale < 1e-4
        unit = np.clip(np.abs(x), 0, 7168).reshape(50, 2, 32).max(-1) / 8 * (1 + 2.0 ** -6) + 2.0 ** -24
        assert (np.abs(y - np.clip(x, -7168, 7168)).reshape(50, 2, 32) <= unit[..., None]).all()


@pytest.mark.parametrize("drafted", [True, False])
def test_plain_verification_keeps_the_targets_distribution(drafted):
    """All drafts of a root with two children, their numbers on a grid: the token after the root comes out as often as the target says."""
    p, q, steps = np.array([0.5, 0.25, 0.125, 0.125]), np.array([0.125, 0.25, 0.375, 0.25]), 128
    grid = (np.arange(steps) + 0.5) / steps
    freq = np.zeros(4)
    for a, b in itertools.product(range(4), repeat=2):
        if not drafted and (a, b) != (1, 2):
            continue
        weight = q[a] * q[b] if drafted else 1.0
        for u1 in grid:
            for u2 in grid[::8]:
                target, draft = np.tile(p, (3, 1)), np.tile(q, (3, 1))
                # (the last number is shared with u1's: only its marginal counts where a child was accepted, and a grid of its own where none was)
                kept, count, _ = more.verify(target, draft if drafted else None, [0, a, b], [-1, 0, 0], [0, 3], [0.5, u1, u2])
                if count[0] > 1:
                    freq[[0, a, b][kept[0, 1]]] += weight / steps / (steps // 8)
                else:
                    for u0 in grid[::16]:
                        token = more.verify(target, draft if drafted else None, [0, a, b], [-1, 0, 0], [0, 3], [u0, u1, u2])[2]
                        freq[token[0]] += weight / steps / (steps // 8) / (steps // 16)
    assert np.abs(freq - p).max() < 0.05 and abs(freq.sum() - 1) < 1e-9  # the grid's steps: 1/128, 1/16 and 1/8 of what is left


def test_plain_eviction():
    mass = np.array([5, 1, 1, 9, np.nan, 1, 2, 0], np.float32).reshape(1, 1, 1, 8)
    kept, left = more.evict(mass, [8], 4, 1, 1)
    assert kept[0, 0, 0].tolist() == [0, 3, 6, 7] and left.tolist() == [4]
    assert more.evict(mass, [8], 5, 1, 1)[0][0, 0, 0].tolist() == [0, 1, 3, 6, 7]
    assert more.evict(mass, [3], 5, 1, 1)[0][0, 0, 0].tolist() == [0, 1, 2, -1, -1]


def test_plain_attention_adds_weights_up():
    r = np.random.default_rng(1)
    k, v, q = r.standard_normal((5, 1, 4)), r.standard_normal((5, 1, 4)), r.standard_normal((2, 3, 4))
    out, mass = np.zeros((2, 3, 4)), np.full((1, 1, 8), 2.0)
    more.attend_tokens(q, [k], [v], [np.ones(5, bool)], [0, 2], [3], None, 0.5, out, mass, lambda a, b: 0.0)
    assert abs(mass[0, 0, :3].sum() - 6 + mass[0, 0, 3:5].sum() - 6) < 1e-12 and (mass[0, 0, 5:] == 2.0).all()
    e = np.exp(k[:4, 0] @ q[0, 1] * 0.5)
    assert np.allclose(out[0, 1], e @ v[:4, 0] / e.sum())
