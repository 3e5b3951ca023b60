"""Build the sm_100a C-ABI library ``liboc_b200.so`` in-tree.

    python onecompression-runtime_b200/build.py [--verbose] [--changed]

The library's translation units (``csrc/*.cu``) are compiled by nvcc for ``sm_100a``
only, side by side, and linked next to the Python package
(``onecomp_runtime/liboc_b200.so``), where ``onecomp_runtime._lib`` loads it. Objects
stay in ``_build/``; without ``force`` only units older than a source they include
are compiled again.
No torch headers are involved: the Python layer binds the plain C ABI.
"""
from __future__ import annotations

import os
import re
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

HERE = Path(__file__).resolve().parent
CSRC = HERE / "csrc"
OBJ = HERE / "_build"
OUT = HERE / "onecomp_runtime" / "liboc_b200.so"
INCLUDE = HERE.parent / "include"

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC,-O3",
    "--expt-relaxed-constexpr",
]


def nvcc_path() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found")


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu")) + sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.h")) + [INCLUDE / "oc_b200.h"]


def included(unit: Path) -> set[Path]:
    """The unit and every source it includes, directly or not."""
    found, todo = set(), [unit]
    while todo:
        path = todo.pop()
        if path in found:
            continue
        found.add(path)
        for name in re.findall(r'^#include "([^"]+)"', path.read_text(), flags=re.M):
            dep = (path.parent / name).resolve()
            if dep.exists():
                todo.append(dep)
    return found


def needs_build() -> bool:
    if not OUT.exists():
        return True
    t = OUT.stat().st_mtime
    return any(p.stat().st_mtime > t for p in sources())


def _run(cmd: list[str], verbose: bool) -> None:
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError(f"nvcc failed with exit code {res.returncode}")
    if verbose:
        sys.stderr.write(res.stderr)


def build(force: bool = False, verbose: bool = False) -> Path:
    if not force and not needs_build():
        return OUT
    OBJ.mkdir(exist_ok=True)
    units = sorted(CSRC.glob("*.cu"))
    objects = [OBJ / (u.stem + ".o") for u in units]
    stale = [(u, o) for u, o in zip(units, objects)
             if force or not o.exists() or any(p.stat().st_mtime > o.stat().st_mtime for p in included(u))]

    def compile_unit(pair: tuple[Path, Path]) -> None:
        unit, obj = pair
        flags = ["-Xptxas=-v"] if verbose else []
        _run([nvcc_path(), *flags, *NVCC_FLAGS, f"-I{INCLUDE}", "-c", str(unit), "-o", str(obj)], verbose)

    with ThreadPoolExecutor(max(1, len(stale))) as pool:
        list(pool.map(compile_unit, stale))
    _run([nvcc_path(), *NVCC_FLAGS, "-shared", *map(str, objects), "-o", str(OUT) + ".tmp"], verbose)
    os.replace(str(OUT) + ".tmp", OUT)
    return OUT


if __name__ == "__main__":
    build(force="--changed" not in sys.argv, verbose="--verbose" in sys.argv)
    print(OUT)
