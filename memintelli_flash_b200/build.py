"""Build recipe for the native library (nvcc, sm_100a, in-tree).

    python -m memintelli_flash_b200.build

compiles ``csrc/memintelli_b200.cu`` and ``csrc/lm_ops.cu`` (which include the kernel
sources), side by side, into ``_lib/libmemintelli_b200.so``.  A unit is recompiled only
when one of its sources is newer than its object file.
"""
from __future__ import annotations

import glob
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB_DIR = os.path.join(HERE, "_lib")
LIB = os.path.join(LIB_DIR, "libmemintelli_b200.so")
INCLUDE = os.path.join(os.path.dirname(HERE), "include")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-std=c++17", "-O3", "-lineinfo",
    "-Xcompiler", "-fPIC",
    "-Xptxas", "-v",
]

# sources that only the tuning operators' unit includes; every other source belongs to memintelli_b200.cu
LM_SOURCES = ("lm_ops.cu", "lm_abi.cu", "lm_common.cuh", "embedding.cu", "token_loss.cu", "grad_clip.cu")
SHARED_SOURCES = ("common.cuh", "kernels.cuh")


def _nvcc():
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cuh"))
                  + glob.glob(os.path.join(INCLUDE, "*.h")))


def _units():
    """(main source, object file, sources it depends on) of each translation unit."""
    lm, core = [], []
    for p in sources():
        name = os.path.basename(p)
        if name in LM_SOURCES or name in SHARED_SOURCES or name.endswith(".h"):
            lm.append(p)
        if name not in LM_SOURCES:
            core.append(p)
    return [(os.path.join(CSRC, f"{n}.cu"), os.path.join(LIB_DIR, f"{n}.o"), deps)
            for n, deps in (("memintelli_b200", core), ("lm_ops", lm))]


def _newer(target: str, deps) -> bool:
    return os.path.exists(target) and all(os.path.getmtime(s) <= os.path.getmtime(target) for s in deps)


def up_to_date() -> bool:
    return _newer(LIB, sources())


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and up_to_date():
        return LIB
    os.makedirs(LIB_DIR, exist_ok=True)
    nvcc, units = _nvcc(), _units()
    running = []
    for main, obj, deps in units:
        if not force and _newer(obj, deps):
            continue
        cmd = [nvcc, *NVCC_FLAGS, "-I", INCLUDE, "-c", "-o", obj + ".tmp", main]
        running.append((obj, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
    done = [(obj, p.communicate()[0], p.returncode) for obj, p in running]
    for obj, text, rc in done:
        if rc != 0:
            raise RuntimeError("nvcc failed:\n" + text)
        if verbose:
            print(text)
        os.replace(obj + ".tmp", obj)
    tmp = LIB + ".tmp"
    res = subprocess.run([nvcc, *NVCC_FLAGS[:2], "-shared", "-o", tmp, *(obj for _, obj, _ in units)],
                         capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError("nvcc failed:\n" + res.stdout + res.stderr)
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
