"""The rows that a run's prefix is read for (csrc/paged_index.h), on the host."""
import os
import shutil
import subprocess

import pytest

from moss_tts import _build


def test_what_a_run_reads(tmp_path):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no host compiler")
    exe = str(tmp_path / "check")
    source = os.path.join(os.path.dirname(os.path.abspath(__file__)), "host", "paged_taken_check.cpp")
    subprocess.run([cxx, "-std=c++17", "-O1", "-I", _build.CSRC, source, "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr
