"""Build libone_b200.so (the sm_100a engine) in-tree with nvcc.

    python medit-one_b200/build.py [--force]

The library is a plain C-ABI shared object (include/one_b200.h): no torch headers,
compiled for sm_100a only. It lands in medit-one_b200/one/libone_b200.so, where the
`one` package loads it.
"""
from __future__ import annotations

import hashlib
import os
import subprocess
import sys
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT = os.path.join(HERE, "one", "libone_b200.so")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-std=c++17", "-lineinfo",
         "-Xcompiler", "-fPIC", "-diag-suppress=177"]
UNITS = ["engine", "linear_moe_noalloc", "serving", "serving_quant"]  # compiled side by side, one library


def _sources():
    files = sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh")))
    files.append(os.path.join(os.path.dirname(HERE), "include", "one_b200.h"))
    return files


def _digest():
    h = hashlib.sha256()
    for f in _sources():
        with open(f, "rb") as fh:
            h.update(fh.read())
    h.update(" ".join(FLAGS).encode())
    return h.hexdigest()


def _run_all(cmds, verbose):
    """Runs the commands side by side; raises for the first that fails."""
    if verbose:
        print("\n".join(" ".join(c) for c in cmds), flush=True)
    running = [subprocess.Popen(c) for c in cmds]
    codes = [p.wait() for p in running]
    for c, rc in zip(cmds, codes):
        if rc:
            raise subprocess.CalledProcessError(rc, c)


def build(force: bool = False, verbose: bool = True) -> str:
    stamp = OUT + ".sha256"
    dig = _digest()
    if not force and os.path.exists(OUT) and os.path.exists(stamp) and open(stamp).read().strip() == dig:
        return OUT
    with tempfile.TemporaryDirectory() as tmp:
        objects = {os.path.join(tmp, name + ".o"): os.path.join(CSRC, name + ".cu") for name in UNITS}
        _run_all([[NVCC, *FLAGS, "-c", "-o", obj, src] for obj, src in objects.items()], verbose)
        _run_all([[NVCC, *FLAGS, "-shared", "-o", OUT, *objects]], verbose)
    with open(stamp, "w") as fh:
        fh.write(dig)
    return OUT


if __name__ == "__main__":
    build(force="--force" in sys.argv)
