"""The picking half of the choice of pages (csrc/pages_pick.cuh), its threads as threads of the host: right lists whichever warp is held up behind a
barrier, and nothing that two threads touch without a barrier between them."""
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


def build(tmp_path, *flags):
    exe = str(tmp_path / "pick")
    r = subprocess.run(["/usr/bin/g++", "-std=c++17", "-O1", "-g", "-Wno-unknown-pragmas", *flags, "-I", HERE, os.path.join(HERE, "pages_pick_host.cpp"), "-o", exe, "-lpthread"],
                       capture_output=True, text=True)
    return r, exe


def test_lists_with_a_warp_held_up(tmp_path):
    r, exe = build(tmp_path)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True)  # (ends itself after four minutes)
    assert r.returncode == 0, f"{r.returncode}: {r.stdout}"


def test_no_two_threads_touch_a_word_without_a_barrier_between(tmp_path):
    r, exe = build(tmp_path, "-fsanitize=thread")
    if r.returncode:
        pytest.skip("no thread sanitizer here")
    r = subprocess.run([exe], capture_output=True, text=True, env={**os.environ, "TSAN_OPTIONS": "halt_on_error=1"})
    if "unexpected memory mapping" in r.stderr:
        pytest.skip("the thread sanitizer does not run here")
    assert r.returncode == 0, f"{r.returncode}: {r.stdout}{r.stderr[:2000]}"
