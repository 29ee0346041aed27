"""Builds ``libaimet_b200.so`` (the C-ABI kernel library) in-tree with nvcc for sm_100a, and the extension
module ``_calls.so`` (host code of the per-token operators) with the host compiler.

Usage: ``python -m aimet_b200.build [--force] [--verbose]``.  Both are written next to
this file; nothing is cached outside the source tree.
"""

from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
SRC_DIR = os.path.join(PKG_DIR, "csrc")
OBJ_DIR = os.path.join(PKG_DIR, "build")
LIB_PATH = os.path.join(PKG_DIR, "libaimet_b200.so")
CALLS_SRC = os.path.join(SRC_DIR, "calls.cpp")
CALLS_PATH = os.path.join(PKG_DIR, "_calls.so")  # the Python extension module aimet_b200._calls
STAMP_PATH = LIB_PATH + ".stamp"

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC",
    "--expt-relaxed-constexpr",
]


def _nvcc() -> str:
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        raise RuntimeError("nvcc not found; aimet_b200 needs the CUDA toolkit to build its kernels")
    return nvcc


def _sources() -> list[str]:
    return sorted(os.path.join(SRC_DIR, f) for f in os.listdir(SRC_DIR) if f.endswith(".cu"))


def _source_digest() -> str:
    """Hash of everything the library is made from: the sources, the public header, the flags."""
    import hashlib

    from importlib.metadata import version

    h = hashlib.sha256(" ".join(NVCC_FLAGS).encode())
    h.update((version("torch") + sys.version).encode())  # what the extension module is compiled against
    paths = sorted(os.path.join(SRC_DIR, f) for f in os.listdir(SRC_DIR))
    paths.append(os.path.join(PKG_DIR, os.pardir, "include", "aimet_b200.h"))
    for p in paths:
        h.update(os.path.basename(p).encode())
        with open(p, "rb") as f:
            h.update(f.read())
    return h.hexdigest()


def is_up_to_date() -> bool:
    """True when the library on disk was built from exactly the present sources (by content, not by
    file times: a checkout or a copy to another machine changes times but not contents)."""
    if not (os.path.exists(LIB_PATH) and os.path.exists(CALLS_PATH) and os.path.exists(STAMP_PATH)):
        return False
    with open(STAMP_PATH) as f:
        return f.read().strip() == _source_digest()


def _build_calls() -> None:
    """The extension module: host code over torch's C++ interface and the C ABI header."""
    import sysconfig

    import torch

    torch_dir = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(_nvcc()))
    tmp = CALLS_PATH + ".tmp"
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",  # pylint: disable=protected-access
           "-I" + os.path.join(torch_dir, "include"), "-I" + os.path.join(torch_dir, "include", "torch", "csrc", "api", "include"),
           "-I" + sysconfig.get_paths()["include"], "-I" + os.path.join(cuda, "include"), CALLS_SRC, "-o", tmp,
           "-L" + os.path.join(torch_dir, "lib"), "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"g++ failed for {CALLS_SRC}:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, CALLS_PATH)


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile every ``csrc/*.cu`` and link the shared library. Returns its path."""
    if not force and is_up_to_date():
        return LIB_PATH
    nvcc = _nvcc()
    os.makedirs(OBJ_DIR, exist_ok=True)
    extra = ["-Xptxas", "-v"] if verbose else []

    def compile_one(src: str) -> str:
        obj = os.path.join(OBJ_DIR, os.path.basename(src)[:-3] + ".o")
        cmd = [nvcc, *NVCC_FLAGS, *extra, "-c", src, "-o", obj]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if verbose and res.stderr:
            sys.stderr.write(res.stderr)
        if res.returncode != 0:
            raise RuntimeError(f"nvcc failed for {src}:\n{res.stdout}\n{res.stderr}")
        return obj

    with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as pool:
        calls = pool.submit(_build_calls)
        objs = list(pool.map(compile_one, _sources()))
        calls.result()

    tmp = LIB_PATH + ".tmp"
    cmd = [nvcc, "-shared", "-o", tmp, *objs, "-gencode", "arch=compute_100a,code=sm_100a", "-cudart", "static"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, LIB_PATH)
    with open(STAMP_PATH, "w") as f:
        f.write(_source_digest() + "\n")
    return LIB_PATH


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    ns = ap.parse_args()
    print(build(force=ns.force, verbose=ns.verbose))
