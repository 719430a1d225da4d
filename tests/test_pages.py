"""Operators over the pages of a caller's cache, as far as they go without a GPU: the plain statements the GPU tests compare with, the C struct, refusals
that come before any device call, and what the Python class checks itself."""
import ctypes as C
import itertools
import os
import subprocess
import tempfile

import numpy as np
import pytest

import pages_plain as plain

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    from orangu_b200 import build, capi

    build.build_all()
    return capi.load()


def test_struct_layout():
    from orangu_b200 import capi

    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "t.cpp"), os.path.join(d, "t")
        open(src, "w").write('#include <cstdio>\n#include <cstddef>\n#include "orangu_b200.h"\nint main(){ std::printf("%zu %zu %zu %zu %u %u", sizeof(ob_pages_desc), offsetof(ob_pages_desc, type),'
                             ' offsetof(ob_pages_desc, head_dim), offsetof(ob_pages_desc, tables), OB_TYPE_F16, OB_TYPE_BF16); }\n')
        subprocess.run(["/usr/bin/g++", "-std=c++17", "-I", os.path.join(ROOT, "include"), src, "-o", exe], check=True)
        out = [int(v) for v in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()]
    D = capi.PagesDesc
    assert out == [C.sizeof(D), D.type.offset, D.head_dim.offset, D.tables.offset, capi.TYPE_F16, capi.TYPE_BF16]
    notes = open(os.path.join(ROOT, "INTEGRATION.md")).read()
    rust = notes[notes.index("pub struct ob_pages_desc"):]
    rust = rust[:rust.index("\n}")]
    for name, _ in D._fields_:
        assert f"pub {name}:" in rust or f"pub r#{name}:" in rust


def test_a_null_handle_is_a_status(lib):
    from orangu_b200 import capi

    h, d = C.c_void_p(), capi.PagesDesc()
    assert lib.ob_pages_create(None, C.byref(d), C.byref(h)) == -1 and not h.value
    lib.ob_pages_destroy(None)
    for name, (_, args) in capi.SIGNATURES.items():
        if name.startswith("ob_pages_") and name not in ("ob_pages_create", "ob_pages_destroy"):
            zeros = [None if a in (C.c_void_p,) else 0 if a is not C.c_float else 0.5 for a in args]
            assert getattr(lib, name)(*zeros) == -1, name


class Fake:
    """An array as the Python class sees one."""

    def __init__(self, shape, dtype, contiguous=True):
        self.shape, self.dtype, self._contiguous = shape, dtype, contiguous

    def data_ptr(self):
        return 4096

    def is_contiguous(self):
        return self._contiguous

    def stride(self):
        return (self.shape[1] * self.shape[2] + 8, self.shape[2], 1)


class Recorder:
    """The library's place: takes every call."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *a: self.calls.append((name, a)) or 0


def test_python_checks():
    from orangu_b200 import PagedCache

    be = type("B", (), {})()
    be._h, be._lib = 1, Recorder()
    pool, tables = (2, 9, 2, 16, 64), Fake((3, 4), "torch.int32")
    for bad in (dict(k=Fake(pool[:4], "torch.float16")), dict(k=Fake((2, 9, 2, 8, 64), "torch.float16")), dict(k=Fake(pool, "torch.float32")), dict(v=Fake(pool, "torch.bfloat16")),
                dict(v=Fake((2, 8, 2, 16, 64), "torch.float16")), dict(k=Fake(pool, "torch.float16", False)), dict(tables=Fake((3, 4), "torch.int64")), dict(tables=Fake((12,), "torch.int32"))):
        with pytest.raises(ValueError):
            PagedCache(be, **{**dict(k=Fake(pool, "torch.float16"), v=Fake(pool, "torch.float16"), tables=tables), **bad})
    c = PagedCache(be, Fake(pool, "torch.float16"), Fake(pool, "torch.float16"), tables)
    i32 = lambda *s: Fake(s, "torch.int32")  # noqa: E731
    q, out, bits = Fake((5, 4, 64), "torch.float16"), Fake((5, 4, 64), "torch.float16", False), Fake((5,), "torch.int64")
    c.attention_tree(q, i32(3), i32(2), bits, 0.1, out, 3, 10, stream=0)
    name, args = be._lib.calls[-1]
    assert name == "ob_pages_attention_tree" and args[2] == 2 and args[4] == 256 and args[5] == 5 and args[9] == 4 and args[14] == 264
    assert args[-1] == 1  # torch's default stream is the runtime's legacy stream, not the context's own
    c.attention_tree(q, i32(3), i32(2), bits, 0.1, out, 3, 10)
    assert be._lib.calls[-1][1][-1] is None
    n = len(be._lib.calls)
    for bad in (dict(q=Fake((5, 4, 128), "torch.float16")), dict(q=Fake((5, 4, 64), "torch.bfloat16")), dict(first_token=i32(2)), dict(n_ctx=Fake((2,), "torch.int64")), dict(visible=Fake((4,), "torch.int64")),
                dict(visible=Fake((5,), "torch.int32")), dict(out=Fake((5, 8, 64), "torch.float16"))):
        with pytest.raises(ValueError):
            c.attention_tree(**{**dict(q=q, first_token=i32(3), n_ctx=i32(2), visible=bits, scale=0.1, out=out, max_drafts=3, max_context=10), **bad})
    codes, scales = Fake((9, 2, 2, 64), "torch.int8"), Fake((9, 2), "torch.float32")
    for bad in (dict(codes=Fake((9, 2, 2, 64), "torch.uint8")), dict(scales=Fake((9, 3), "torch.float32")), dict(selected=i32(5, 1, 4)), dict(n_pos=i32(4)), dict(row_seq=i32(4))):
        with pytest.raises(ValueError):
            c.select(**{**dict(q=q, codes=codes, scales=scales, n_pos=i32(5), selected=i32(5, 2, 4), max_pos=9), **bad})
    for call in (lambda: c.copy(i32(3), i32(4)), lambda: c.fork(i32(3), i32(3), i32(3), i32(2)), lambda: c.keep(i32(2), i32(3, 5), i32(3)), lambda: c.bounds(i32(2), i32(3), codes, scales, 4),
                 lambda: c.attention(q, i32(4, 2, 4), i32(5), 0.1, out)):
        with pytest.raises(ValueError):
            call()
    assert len(be._lib.calls) == n  # nothing reached the library


# ---------------------------------------------------------------------------------------- the plain statements themselves
def test_plain_choice_against_all_choices():
    """The chosen pages are those whose scores no other choice beats, page by page, with the smallest numbers among equals."""
    r = np.random.default_rng(2)
    for _ in range(40):
        pages, n = int(r.integers(1, 8)), int(r.integers(1, 6))
        codes = r.integers(-3, 4, (pages, 1, 2, 4)).astype(np.int8)
        codes[:, :, 0] = np.maximum(codes[:, :, 0], codes[:, :, 1])
        scales = np.full((pages, 1), 0.5, np.float32)
        q = r.integers(-2, 3, (1, 2, 4)).astype(np.float32) * 127  # units of whole numbers: exact scores
        got = plain.select(q, codes, scales, [list(range(pages))], [pages * 16], n, 0, 0, [0], 1)[0, 0]
        score = []
        for p in range(pages):
            best = -np.inf
            for h in range(2):
                d = np.abs(q[0, h]).max() / np.float32(127)
                c = np.rint(q[0, h] / (d if d else np.float32(1)))
                best = max(best, float(d * np.float32(0.5) * np.float32(sum(max(a * float(hi), a * float(lo)) for a, hi, lo in zip(c, codes[p, 0, 0], codes[p, 0, 1])))))
            score.append(best)
        want = max(itertools.combinations(range(pages), min(n, pages)), key=lambda s: (sorted((score[p] for p in s), reverse=True), [-p for p in s]))
        assert [p for p in got if p >= 0] == list(want) and (got[len(want):] == -1).all()


def test_plain_bounds_hold():
    r = np.random.default_rng(1)
    k, _ = plain.bits16((3, 2, 16, 64), r, "bf16")
    codes, scales = np.zeros((3, 2, 2, 64), np.int8), np.zeros((3, 2), np.float32)
    plain.bounds(k, [[2, 0]], [0], [21], codes, scales)
    for page, rows in ((2, 16), (0, 5)):
        part = k[page, :, :rows]
        up, down = codes[page, :, 0] * scales[page][:, None].astype(np.float64), codes[page, :, 1] * scales[page][:, None].astype(np.float64)
        slack = np.abs(part).max() * 2.0 ** -22
        assert (part.max(1) <= up + slack).all() and (part.min(1) >= down - slack).all()
        assert (up - part.max(1) < scales[page][:, None] * 1.001).all()
    assert (scales[1] == 0).all()


def test_plain_tree_is_attention_of_each_path():
    """A token of a tree sees what it would at the end of its own path."""
    r = np.random.default_rng(3)
    k, _ = plain.bits16((4, 1, 16, 64), r, "f16")
    v, _ = plain.bits16((4, 1, 16, 64), r, "f16")
    q, _ = plain.bits16((4, 2, 64), r, "f16")
    bits = [0b0001, 0b0011, 0b0101, 0b1011]
    out = np.zeros(q.shape)
    plain.tree(q, k, v, [[3, 1, 0]], [0, 4], [20], bits, 0.1, out, lambda *a: 0.0)
    flat = lambda x: np.concatenate([x[3, 0], x[1, 0], x[0, 0]])  # noqa: E731
    for t, b in enumerate(bits):
        at = list(range(20)) + [20 + j for j in range(4) if b >> j & 1]
        for h in range(2):
            s = flat(k)[at] @ q[t, h] * 0.1
            w = np.exp(s - s.max())
            assert np.allclose(out[t, h], w / w.sum() @ flat(v)[at], rtol=1e-12)
