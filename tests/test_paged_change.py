"""The index arithmetic of the paged operators (csrc/paged_index.h) on the host, for starts and lengths that change under the
kernels: what has no place is told apart before anything is read or written for it."""
import os
import shutil
import subprocess

import pytest

from moss_tts import _build

HOST = os.path.join(os.path.dirname(os.path.abspath(__file__)), "host")


def test_items_of_a_batch_that_changes(tmp_path):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no host compiler")
    exe = str(tmp_path / "check")
    subprocess.run([cxx, "-std=c++17", "-O1", "-I", _build.CSRC, os.path.join(HOST, "paged_change_check.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr
