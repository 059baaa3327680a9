"""In-tree build of libpto_b200.so (nvcc, sm_100a only).

Run as ``python -m pto_isa_mirror_b200.build``. The library lands in ``pto_isa_mirror_b200/lib/`` next to the
sources so that it travels with the source tree; nothing is written outside the package directory. Each source is
compiled to an object of its own, those that changed at the same time, and the objects are linked.
"""
from __future__ import annotations

import os
import subprocess
import sys

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG_DIR, "csrc")
LIB_DIR = os.path.join(PKG_DIR, "lib")
OBJ_DIR = os.path.join(LIB_DIR, "obj")
LIB = os.path.join(LIB_DIR, "libpto_b200.so")
_ABI = os.path.join("..", "..", "include", "pto_b200.h")
# source -> the headers it includes
SOURCES = {
    "pto_b200_capi.cu": ["capi_shared.cuh", "gemm_tile_loop.cuh", "gemm_tile_loop_2cta.cuh", "gemv.cuh", "gemv_mx.cuh",
                         "ksplit_reduce.cuh", "mx_quantize.cuh", "row_elements.cuh", "sm100_ptx.cuh", _ABI],
    "nvfp4_capi.cu": ["capi_shared.cuh", "gemm_tile_loop.cuh", "gemm_nvfp4.cuh", "nvfp4_quantize.cuh", "row_elements.cuh", "sm100_ptx.cuh",
                       _ABI],
    "checkpoint_capi.cu": ["capi_shared.cuh", "gemm_tile_loop.cuh", "gemm_wgrad_mx.cuh", "mx_quantize.cuh",
                           "row_elements.cuh", "sm100_ptx.cuh", _ABI],
}

NVCC_FLAGS = [
    "-std=c++17",
    "-O3",
    "-gencode",
    "arch=compute_100a,code=sm_100a",
    "-lineinfo",
    "-Xcompiler",
    "-fPIC",
]


def _deps(source):
    return [os.path.normpath(os.path.join(CSRC, f)) for f in [source, *SOURCES[source]]]


def _object(source):
    return os.path.join(OBJ_DIR, source[: -len(".cu")] + ".o")


def _newest(paths):
    return max(os.path.getmtime(p) for p in paths)


def _stale(target, deps) -> bool:
    return not os.path.exists(target) or _newest(deps) > os.path.getmtime(target)


def needs_build() -> bool:
    return _stale(LIB, [d for s in SOURCES for d in _deps(s)])


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile the CUDA sources into lib/libpto_b200.so and return its path."""
    if not force and not needs_build():
        return LIB
    os.makedirs(OBJ_DIR, exist_ok=True)
    nvcc = os.environ.get("NVCC", "nvcc")
    flags = NVCC_FLAGS + (["-Xptxas", "-v"] if verbose else [])
    running = []
    for source in SOURCES:
        if force or _stale(_object(source), _deps(source)):
            cmd = [nvcc, *flags, "-c", "-o", _object(source), os.path.join(CSRC, source)]
            running.append((cmd, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True)))
    failed = ""
    for cmd, proc in running:
        out, err = proc.communicate()
        if verbose:
            sys.stderr.write(err)
        if proc.returncode != 0:
            failed += " ".join(cmd) + "\n" + out + err
    if failed:
        raise RuntimeError("nvcc failed:\n" + failed)
    cmd = [nvcc, "-shared", *flags, "-o", LIB, *(_object(s) for s in SOURCES)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError("nvcc failed:\n" + " ".join(cmd) + "\n" + proc.stdout + proc.stderr)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
