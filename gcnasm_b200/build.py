"""Build the in-tree CUDA library ``gcnasm_b200/_lib/libb2g.so`` for sm_100a.

nvcc cross-compiles without a GPU; the resulting shared object travels with the
source tree.  ``python -m gcnasm_b200.build`` or ``__graft_entry__.build()``.
"""
from __future__ import annotations

import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
LIB = os.path.join(HERE, "_lib", "libb2g.so")
SOURCES = [os.path.join(HERE, "csrc", f) for f in ("b2g_api.cu", "b2g_kv4_api.cu")]
# every source and header under csrc/ plus the public headers: editing any of them rebuilds
DEPS = sorted(os.path.join(HERE, "csrc", f) for f in os.listdir(os.path.join(HERE, "csrc"))
              if f.endswith((".cu", ".cuh", ".h"))) + [os.path.join(ROOT, "include", "b2g", f)
                                                       for f in ("gemm.h", "kv4.h")]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", "nvcc"):
        if cand and (os.path.sep not in cand or os.path.exists(cand)):
            return cand
    return "nvcc"


def up_to_date() -> bool:
    if not os.path.exists(LIB):
        return False
    t = os.path.getmtime(LIB)
    return all(os.path.getmtime(d) <= t for d in DEPS if os.path.exists(d))


def _object(src: str) -> str:
    return os.path.join(HERE, "_lib", os.path.basename(src) + ".o")


def _object_up_to_date(src: str) -> bool:
    """The object is newer than everything its last compilation read (nvcc's dependency file)."""
    obj = _object(src)
    if not (os.path.exists(obj) and os.path.exists(obj + ".d")):
        return False
    with open(obj + ".d") as f:
        deps = f.read().replace("\\\n", " ").split(":", 1)[-1].split()
    t = os.path.getmtime(obj)
    return src in deps and all(os.path.exists(d) and os.path.getmtime(d) <= t for d in deps)


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and up_to_date():
        return LIB
    os.makedirs(os.path.dirname(LIB), exist_ok=True)
    todo = []
    for src in SOURCES:
        if not force and _object_up_to_date(src):
            continue
        obj = _object(src)
        cmd = [nvcc(), *NVCC_FLAGS, *(["-Xptxas=-v"] if verbose else []), "-I", os.path.join(ROOT, "include"),
               "-I", os.path.join(HERE, "csrc"), "-MD", "-MF", obj + ".d", "-c", src, "-o", obj]
        todo.append((cmd, subprocess.Popen(cmd)))
    for cmd, p in [(c, p) for c, p in todo if p.wait()]:
        raise subprocess.CalledProcessError(p.returncode, cmd)
    subprocess.run([nvcc(), *NVCC_FLAGS, "-shared", *map(_object, SOURCES), "-o", LIB + ".tmp"], check=True)
    os.replace(LIB + ".tmp", LIB)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
