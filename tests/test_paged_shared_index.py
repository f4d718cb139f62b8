"""The index arithmetic of the shared prefixes (csrc/paged_index.h) on the host, and what the C entries refuse without a GPU."""
import ctypes
import os
import shutil
import subprocess

import pytest

from moss_tts import _build
from test_abi_paged import BAD_CACHE, BATCH, CACHE, NULL, ODD, Call, F, P, lib  # noqa: F401
from test_abi_paged8 import BAD_CACHE8, CACHE8

HOST = os.path.join(os.path.dirname(os.path.abspath(__file__)), "host")


def test_runs_and_parts_on_the_host(tmp_path):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no host compiler")
    exe = str(tmp_path / "check")
    subprocess.run([cxx, "-std=c++17", "-O1", "-I", _build.CSRC, os.path.join(HOST, "paged_shared_check.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr


@pytest.mark.parametrize("bits", [16, 8])
def test_refusals(lib, bits):  # noqa: F811
    need = lib.moss_paged_shared_workspace_bytes(3, 4, 16, 32, 8, 128)
    assert need > 0
    fn, cache = (lib.moss_paged_shared_decode_attention, CACHE) if bits == 16 else (lib.moss_paged_shared_decode_attention_fp8, CACHE8)
    call = Call(fn, q=P, q_stride=4096, **cache, **BATCH, groups=P, shared=P, B=3, W=4, qh=32, kh=8, d=128, scale=F(0.1), out=P,
                workspace=P, workspace_bytes=need, dtype=0, stream=NULL)
    for bad in (BAD_CACHE if bits == 16 else BAD_CACHE8) + [
            dict(q=NULL), dict(q=ODD), dict(q_stride=4088), dict(q_stride=4100), dict(scale=F(float("nan"))), dict(out=NULL),
            dict(out=ODD), dict(workspace=NULL), dict(workspace=ODD), dict(workspace_bytes=need - 1), dict(groups=NULL),
            dict(shared=NULL), dict(groups=ctypes.c_void_p(4098)), dict(shared=ctypes.c_void_p(4098))]:
        assert call(**bad) == 1, bad


def test_workspace(lib):  # noqa: F811
    size = lib.moss_paged_shared_workspace_bytes
    own = lib.moss_paged_decode_workspace_bytes
    assert size(64, 100, 16, 32, 8, 128) > own(64, 100, 16, 32, 8, 128)
    for bad in ((0, 4, 16, 32, 8, 128), (65536, 4, 16, 32, 8, 128), (3, 0, 16, 32, 8, 128), (3, 4, 17, 32, 8, 128), (3, 4, 16, 31, 8, 128),
                (3, 4, 16, 32, 8, 80), (3, 4, 16, 2048, 8, 128)):
        assert size(*bad) == 0
