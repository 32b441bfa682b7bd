"""Build recipe for the in-tree sm_100a shared library ``libqmv_b200.so``.

Run ``python my-inference-engine_b200/build.py`` or call ``build_library()``.
nvcc cross-compiles for sm_100a without a GPU.  The CUDA runtime is linked
statically and its symbols are kept private (``--exclude-libs``), so the
library can be loaded next to torch's own runtime.
"""
from __future__ import annotations

import concurrent.futures
import contextlib
import fcntl
import os
import subprocess
import sys
import time

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
REPO_DIR = os.path.dirname(PKG_DIR)
CSRC = os.path.join(PKG_DIR, "csrc")
LIB_PATH = os.path.join(PKG_DIR, "libqmv_b200.so")

OBJ_DIR = os.path.join(PKG_DIR, "build")

SOURCES = ["qmv_kernels.cu", "qmv_capi.cpp", "qmv_qwen2.cpp", "qmv_gguf.cpp", "quantized_matvec.cpp",
           "qmv_attention.cu", "qmv_attention_tc.cu", "qmv_attention_capi.cpp"]
HEADERS = ["qmv_internal.h", "qmv_attention.h", "qmv_attention.cuh"]
PUBLIC_HEADERS = ["qmv_b200.h", "quantized_matvec.h", "gguf_quantized_view.h"]

NVCC_FLAGS = [
    "-std=c++17",
    "-O3",
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo",
    "-Xcompiler", "-fPIC,-fvisibility=hidden,-Wall",
    "-Xptxas", "-v",
]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", "nvcc"):
        if cand and (os.path.isabs(cand) and os.path.exists(cand) or not os.path.isabs(cand)):
            return cand
    return "nvcc"


def _inputs():
    files = [os.path.join(CSRC, s) for s in SOURCES + HEADERS]
    files += [os.path.join(REPO_DIR, "include", h) for h in PUBLIC_HEADERS]
    return files


def up_to_date() -> bool:
    if not os.path.exists(LIB_PATH):
        return False
    t = os.path.getmtime(LIB_PATH)
    return all(os.path.getmtime(f) <= t for f in _inputs())


def _run(cmd, out: str, began: int) -> str:
    """nvcc into a file of this process, which takes its place once it is whole,
    as old as ``began``, when its sources were last looked at (what changes
    meanwhile is newer); an object's messages are in out + ".log" before it."""
    part = f"{out}.tmp{os.getpid()}"
    try:
        proc = subprocess.run([*cmd, "-o", part], capture_output=True, text=True)
        if proc.returncode != 0:
            raise RuntimeError("nvcc failed:\n" + proc.stdout + proc.stderr)
        if out.endswith(".o"):
            with open(out + ".log", "w") as fh:
                fh.write(proc.stderr)
        os.utime(part, ns=(began, began))
        os.replace(part, out)
    finally:
        if os.path.exists(part):
            os.remove(part)
    return proc.stderr


@contextlib.contextmanager
def _alone():
    """One build at a time in this tree."""
    os.makedirs(OBJ_DIR, exist_ok=True)
    with open(os.path.join(OBJ_DIR, "lock"), "w") as fh:
        fcntl.flock(fh, fcntl.LOCK_EX)
        yield


def _compile(source: str, force: bool):
    """One source to its object (skipped when newer than the source and every
    header); (object, nvcc's messages)."""
    src, obj = os.path.join(CSRC, source), os.path.join(OBJ_DIR, source + ".o")
    log = obj + ".log"
    began = time.time_ns()
    deps = [src] + [f for f in _inputs() if f.endswith((".h", ".cuh"))] + [os.path.abspath(__file__)]
    if not force and os.path.exists(obj) and os.path.exists(log) and \
            all(os.path.getmtime(f) <= os.path.getmtime(obj) for f in deps):
        with open(log) as fh:
            return obj, fh.read()
    cmd = [_nvcc(), *NVCC_FLAGS, "-I", os.path.join(REPO_DIR, "include"), "-I", CSRC, "-c", src]
    return obj, _run(cmd, obj, began)


def build_library(force: bool = False, verbose: bool = False) -> str:
    """Compile libqmv_b200.so in place (skipped when up to date), the sources
    side by side."""
    with _alone():
        if not force and up_to_date():
            return LIB_PATH
        began = time.time_ns()
        with concurrent.futures.ThreadPoolExecutor(len(SOURCES)) as pool:
            built = list(pool.map(lambda s: _compile(s, force), SOURCES))
        messages = "".join(m for _, m in built)
        _run([_nvcc(), *NVCC_FLAGS, "-shared", *[obj for obj, _ in built], "-Xlinker", "--exclude-libs,ALL"], LIB_PATH, began)
        with open(os.path.join(PKG_DIR, "ptxas_report.txt"), "w") as fh:
            fh.write(messages)
    if verbose:
        sys.stderr.write(messages)
    return LIB_PATH


if __name__ == "__main__":
    print(build_library(force="--force" in sys.argv, verbose="-v" in sys.argv))
