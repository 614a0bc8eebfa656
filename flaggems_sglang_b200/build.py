"""Builds csrc/*.cu into libfmoe_b200.so (sm_100a only) with nvcc, in-tree.

    python -m flaggems_sglang_b200.build [--force] [--verbose]

The library is a plain C-ABI shared object (see include/fmoe_b200.h); it links
only the CUDA runtime.  Objects are rebuilt when a source or header is newer.
Behind it _host.so is built from csrc/host.cpp, the short way from Python into some
of the operators; it calls the library through the same C entry points, and where it
cannot be built (no C++ compiler, other torch headers) they are called through ctypes.
"""
from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(os.path.dirname(HERE), "include")
OBJ_DIR = os.path.join(HERE, "build")
LIB_PATH = os.path.join(HERE, "libfmoe_b200.so")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-std=c++17", "-lineinfo",
    "-Xcompiler", "-fPIC",
    "--expt-relaxed-constexpr",
    "-Xptxas", "-v",
    "-I", INCLUDE,
]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found; set NVCC or install the CUDA toolkit")


def _sources():
    return sorted(f for f in os.listdir(CSRC) if f.endswith(".cu"))


def _deps_mtime() -> float:
    hdrs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    hdrs += [os.path.join(INCLUDE, f) for f in os.listdir(INCLUDE)]
    return max(os.path.getmtime(h) for h in hdrs)


HOST_SRC = os.path.join(CSRC, "host.cpp")
HOST_PATH = os.path.join(HERE, "_host.so")


def _host_command() -> list[str]:
    """The module with the short way into some of the operators: C++ against the torch and Python of this interpreter."""
    import torch

    base = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(_nvcc())))
    return [os.environ.get("CXX") or shutil.which("g++") or "c++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-w",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f'-DBUILT_FOR_TORCH="{torch.__version__}"',
            "-I", sysconfig.get_paths()["include"], "-I", os.path.join(base, "include"),
            "-I", os.path.join(base, "include", "torch", "csrc", "api", "include"), "-I", os.path.join(cuda, "include"),
            HOST_SRC, "-o", HOST_PATH, "-L", os.path.join(base, "lib"), "-ltorch_python", "-ltorch_cpu", "-ltorch_cuda", "-ltorch", "-lc10", "-lc10_cuda"]


def _build_host(force: bool, verbose: bool) -> None:
    """_host.so, where the sources or the command (and with it torch or Python) are other than those it was built by."""
    try:
        cmd = _host_command()
    except ImportError:
        sys.stderr.write("no torch: csrc/host.cpp is not built\n")
        return
    words = " ".join(w for w in cmd if w not in (HOST_SRC, HOST_PATH))  # the tree may be elsewhere now
    record = os.path.join(OBJ_DIR, "host.command")
    built_by = open(record).read() if os.path.exists(record) else None
    newest = max(os.path.getmtime(HOST_SRC), os.path.getmtime(os.path.join(INCLUDE, "fmoe_b200.h")))
    if not force and built_by == words and os.path.exists(HOST_PATH) and os.path.getmtime(HOST_PATH) >= newest:
        return
    if os.path.exists(HOST_PATH):
        os.remove(HOST_PATH)
    if not os.path.exists(os.path.join(sysconfig.get_paths()["include"], "Python.h")):
        why = "no Python.h"
    else:
        try:
            r = subprocess.run(cmd, capture_output=True, text=True)
            why = None if r.returncode == 0 else " ".join(cmd) + "\n" + r.stdout + r.stderr
        except OSError as e:
            why = str(e)
    if why is not None:
        if os.path.exists(HOST_PATH):
            os.remove(HOST_PATH)
        sys.stderr.write(f"{why}\ncsrc/host.cpp is not built: its operators are called through ctypes\n")
        return
    if verbose:
        sys.stderr.write(" ".join(cmd) + "\n" + r.stdout + r.stderr)
    with open(record, "w") as f:
        f.write(words)


def ptxas_report(src: str) -> str:
    """Where the registers and spills of a source file's kernels are kept, as the compiler printed them."""
    return os.path.join(OBJ_DIR, src[:-3] + ".ptxas")


def build(force: bool = False, verbose: bool = False) -> str:
    os.makedirs(OBJ_DIR, exist_ok=True)
    nvcc = _nvcc()
    hdr_m = _deps_mtime()
    jobs = []
    objs = []
    for src in _sources():
        s = os.path.join(CSRC, src)
        o = os.path.join(OBJ_DIR, src[:-3] + ".o")
        objs.append(o)
        if force or not os.path.exists(o) or not os.path.exists(ptxas_report(src)) or os.path.getmtime(o) < max(os.path.getmtime(s), hdr_m):
            jobs.append([nvcc, *NVCC_FLAGS, "-c", s, "-o", o])

    def run(cmd):
        r = subprocess.run(cmd, capture_output=True, text=True)
        return cmd, r

    if jobs:
        with ThreadPoolExecutor(max_workers=min(8, len(jobs))) as ex:
            for cmd, r in ex.map(run, jobs):
                if verbose or r.returncode != 0:
                    sys.stderr.write(" ".join(cmd) + "\n" + r.stdout + r.stderr)
                if r.returncode != 0:
                    raise RuntimeError(f"nvcc failed for {cmd[-3]}")
                with open(ptxas_report(os.path.basename(cmd[-3])), "w") as f:
                    f.write(r.stderr)
    if jobs or force or not os.path.exists(LIB_PATH):
        cmd = [nvcc, "-shared", "-o", LIB_PATH, *objs, "-gencode", "arch=compute_100a,code=sm_100a", "--cudart", "shared"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            sys.stderr.write(r.stdout + r.stderr)
            raise RuntimeError("link failed")
    _build_host(force, verbose)
    return LIB_PATH


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    a = ap.parse_args()
    print(build(force=a.force, verbose=a.verbose))
