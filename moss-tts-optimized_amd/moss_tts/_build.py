"""Build ``libmoss_hip.so`` (gfx950) from ``csrc/*.hip`` with hipcc, in-tree.

``python -m moss_tts._build`` (with ``moss-tts-optimized_amd`` on ``sys.path``) or
``__graft_entry__.build()``.  Each translation unit compiles to its own object in
parallel; the shared library is linked atomically into ``moss_tts/_lib/``, and beside it the
Python module ``_moss_calls.so`` of the batch operators' calls (``csrc/host/calls.cpp``, the host compiler).
"""
from __future__ import annotations

import concurrent.futures as cf
import glob
import os
import shutil
import subprocess
import sys

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)                      # moss-tts-optimized_amd/
CSRC = os.path.join(ROOT, "csrc")
OBJ = os.path.join(ROOT, "_build")
LIBDIR = os.path.join(PKG, "_lib")
LIB = os.path.join(LIBDIR, "libmoss_hip.so")
CALLS = os.path.join(LIBDIR, "_moss_calls.so")   # csrc/host/calls.cpp: the Python module beside it
INCLUDE = os.path.join(os.path.dirname(ROOT), "include")
ARCH = "gfx950"

CFLAGS = [
    f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC", "-fvisibility=hidden",
    "-mcode-object-version=5",
    # packed fp32 VALU forms are kept out of the generated code
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wno-unused-command-line-argument",
]


def hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found; the gfx950 library cannot be built")


def _compile(src: str, verbose: bool) -> str:
    obj = os.path.join(OBJ, os.path.basename(src)[:-4] + ".o")
    cmd = [hipcc(), *CFLAGS, "-I", CSRC, "-c", src, "-o", obj]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src}:\n{r.stdout}\n{r.stderr}")
    return obj


def _compile_calls(verbose: bool) -> None:
    """The compiled Python calls, against the torch that is installed."""
    import sysconfig

    import torch

    from ._runtime import native

    top = os.path.dirname(torch.__file__)
    cxx = shutil.which("g++") or shutil.which("c++")
    # hipcc, which the library needs anyway, is a host compiler too
    compiler = [cxx] if cxx else [hipcc(), "-x", "c++", "-Wno-unused-command-line-argument"]
    tmp = CALLS + ".tmp"
    cmd = [*compiler, "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", f'-DMOSS_BUILT_FOR="{native.calls_tag()}"',
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", "-D__HIP_PLATFORM_AMD__", "-I", INCLUDE,
           "-I", os.path.join(top, "include"), "-I", sysconfig.get_paths()["include"],
           "-I", os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "include"), os.path.join(CSRC, "host", "calls.cpp"),
           "-o", tmp, "-L", os.path.join(top, "lib"),
           "-ltorch", "-ltorch_cpu", "-ltorch_python", "-lc10", "-lc10_hip", "-ldl"]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"the compiled calls failed to build:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, CALLS)


def build(verbose: bool = False, jobs: int | None = None) -> str:
    os.makedirs(OBJ, exist_ok=True)
    os.makedirs(LIBDIR, exist_ok=True)
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.hip")))
    if not srcs:
        raise RuntimeError(f"no HIP sources under {CSRC}")
    jobs = jobs or min(len(srcs), max(1, min(8, os.cpu_count() or 1)))
    with cf.ThreadPoolExecutor(jobs) as ex:
        calls = ex.submit(_compile_calls, verbose)
        objs = list(ex.map(lambda s: _compile(s, verbose), srcs))
        calls.result()
    tmp = LIB + ".tmp"
    cmd = [hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", *objs, "-o", tmp]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
