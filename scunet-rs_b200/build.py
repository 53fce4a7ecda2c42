"""Build `libscunet_b200.so` in-tree with nvcc for sm_100a.

    python scunet-rs_b200/build.py [--force]

Two translation units, compiled side by side: `csrc/scunet_b200.cu` holds the network's
kernels and its C ABI, `csrc/scunet_ops.cu` the block operators'. cudart is linked
statically and the driver API is reached through `cudaGetDriverEntryPoint`, so the
library loads on a machine without a GPU driver (the CPU test suite checks its exported
symbols there).
"""
from __future__ import annotations

import os
import subprocess
import sys
from pathlib import Path

HERE = Path(__file__).resolve().parent
CSRC = HERE / "csrc"
LIB = HERE / "libscunet_b200.so"
OBJ = HERE / "_build"
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC",
]
LINK = ["-shared", "-cudart", "static", "-ldl"]


def sources():
    return [*sorted(CSRC.glob("*.cu*")), *sorted(CSRC.glob("*.h")), HERE.parent / "include" / "scunet_b200.h"]


def up_to_date():
    if not LIB.exists():
        return False
    t = LIB.stat().st_mtime
    return all(s.stat().st_mtime <= t for s in sources())


def build(force=False, verbose=False):
    if not force and up_to_date():
        return LIB
    objects = [(src, OBJ / f"{src.stem}.o") for src in sorted(CSRC.glob("*.cu"))]
    OBJ.mkdir(exist_ok=True)
    _run([[NVCC, *FLAGS, "-c", "-o", str(o), str(src)] for src, o in objects], verbose)
    _run([[NVCC, *FLAGS, *LINK, "-o", str(LIB), *[str(o) for _, o in objects]]], verbose)
    return LIB


def _run(cmds, verbose):
    """Run the commands side by side; raise with the output of the first that failed."""
    if verbose:
        for cmd in cmds:
            print(" ".join(cmd), flush=True)
    running = [subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True) for cmd in cmds]
    for p, out in [(p, p.communicate()[0]) for p in running]:
        if p.returncode != 0:
            raise RuntimeError(f"nvcc failed ({p.returncode}):\n{out}")


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
