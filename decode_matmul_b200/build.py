"""Builds libdmm.so (the CUDA library behind the C ABI in include/dmm.h) with nvcc for sm_100a.

The library has two translation units, csrc/dmm_api.cu (the products) and csrc/dmm_attn_api.cu (attention), which
include the kernel headers and are compiled side by side; the result is written next to this file so that it travels
with the source tree.  The object files stay there too, and one is taken as it is when its sources have not changed and
the same compiler would make it with the same command (an ``.o.cmd`` beside it says which did).
"""
from __future__ import annotations

import os
import re
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libdmm.so")
UNITS = ("dmm_api.cu", "dmm_attn_api.cu")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC",
]


def sources():
    out = []
    for root, _, files in os.walk(CSRC):
        out += [os.path.join(root, f) for f in files if f.endswith((".cu", ".cuh", ".h"))]
    out.append(os.path.join(HERE, "..", "include", "dmm.h"))
    return out


def _depends(path, seen=None):
    """A source file and everything of this library that it includes."""
    seen = set() if seen is None else seen
    path = os.path.normpath(path)
    if path not in seen:
        seen.add(path)
        with open(path) as f:
            for name in re.findall(r'^#include "([^"]+)"', f.read(), re.M):
                _depends(os.path.join(os.path.dirname(path), name), seen)
    return seen


def _made_by(obj) -> str | None:
    """What an object file was made with, None when nothing says so."""
    try:
        with open(obj + ".cmd") as f:
            return f.read()
    except OSError:
        return None


def needs_build() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    return any(os.path.getmtime(s) > t for s in sources())


def build(force: bool = False, verbose: bool = False) -> str:
    """Compiles the library when it is missing or older than its sources; returns its path.

    Safe when several processes (one rank per GPU) import the package at once: the build runs
    under a file lock, into a temporary name that is renamed over the library only when nvcc
    succeeded, and a process that waited for the lock looks again before building."""
    if not force and not needs_build():
        return LIB
    import fcntl

    with open(LIB + ".lock", "w") as lock:
        fcntl.flock(lock, fcntl.LOCK_EX)
        try:
            if not force and not needs_build():
                return LIB
            nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
            version = subprocess.run([nvcc, "--version"], capture_output=True, text=True).stdout
            objects, running, log = [], [], ""
            for unit in UNITS:
                source = os.path.join(CSRC, unit)
                obj = source[:-3] + ".o"
                objects.append(obj)
                made_by = "\n".join([nvcc, *NVCC_FLAGS, unit, version])
                if (not force and os.path.exists(obj) and _made_by(obj) == made_by
                        and all(os.path.getmtime(s) <= os.path.getmtime(obj) for s in _depends(source))):
                    continue
                if os.path.exists(obj + ".cmd"):
                    os.remove(obj + ".cmd")
                tmp = f"{obj}.{os.getpid()}.tmp"
                cmd = [nvcc, *(["-Xptxas", "-v"] if verbose else []), *NVCC_FLAGS, "-c", "-o", tmp, source]
                running.append((obj, tmp, made_by, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
            failed = False
            for obj, tmp, made_by, proc in running:
                log += proc.communicate()[0]
                if proc.returncode == 0:
                    os.replace(tmp, obj)
                    with open(obj + ".cmd", "w") as f:
                        f.write(made_by)
                    continue
                failed = True
                if os.path.exists(tmp):
                    os.remove(tmp)
            if failed:
                raise RuntimeError("nvcc failed:\n" + log)
            tmp = f"{LIB}.{os.getpid()}.tmp"
            res = subprocess.run([nvcc, *NVCC_FLAGS, "-shared", "-o", tmp, *objects], capture_output=True, text=True)
            if res.returncode != 0:
                if os.path.exists(tmp):
                    os.remove(tmp)
                raise RuntimeError("nvcc failed:\n" + res.stdout + res.stderr)
            os.replace(tmp, LIB)
            if verbose:
                sys.stderr.write(log)
        finally:
            fcntl.flock(lock, fcntl.LOCK_UN)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
