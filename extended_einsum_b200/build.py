"""Builds the sm_100a shared library libxe_b200.so in-tree with nvcc.

The library is the C ABI declared in include/xe_b200.h; the Python package
loads it with ctypes (extended_einsum_b200/_lib.py).
"""

from __future__ import annotations

import os
import re
import shutil
import subprocess
import sys
from pathlib import Path

PACKAGE_DIR = Path(__file__).resolve().parent
REPO_ROOT = PACKAGE_DIR.parent
CSRC = PACKAGE_DIR / "csrc"
LIBRARY = PACKAGE_DIR / "libxe_b200.so"
SOURCES = [CSRC / "xe_b200.cu", CSRC / "xe_sequence.cu"]
DEPENDENCIES = sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.h")) + [REPO_ROOT / "include" / "xe_b200.h"]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC",
    "--expt-relaxed-constexpr",
]


def find_nvcc() -> str:
    for candidate in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if candidate and Path(candidate).exists():
            return candidate
    raise RuntimeError("nvcc not found: the sm_100a library cannot be built")


def is_stale() -> bool:
    if not LIBRARY.exists():
        return True
    built = LIBRARY.stat().st_mtime
    return any(p.stat().st_mtime > built for p in SOURCES + DEPENDENCIES)


def _includes(source: Path) -> list[Path]:
    """The source and the headers of the repository that it includes, directly or not."""
    found, todo = [], [source]
    while todo:
        path = todo.pop()
        if path in found or not path.exists():
            continue
        found.append(path)
        for name in re.findall(r'^#include "([^"]+)"', path.read_text(), flags=re.M):
            todo.append((path.parent / name).resolve())
    return found


def build(force: bool = False, verbose: bool = False, extra_flags: list[str] | None = None) -> Path:
    """Compiles libxe_b200.so for sm_100a if a source is newer than the library.

    Each source becomes an object of its own, compiled side by side; one whose includes are all
    older than its object is kept (with the default flags)."""
    if not force and not is_stale():
        return LIBRARY
    nvcc, running, objects = find_nvcc(), [], []
    for source in SOURCES:
        obj = source.with_suffix(".o")
        objects.append(obj)
        newest = max(p.stat().st_mtime for p in [*_includes(source), Path(__file__)])
        if not force and not extra_flags and obj.exists() and obj.stat().st_mtime > newest:
            continue
        cmd = [nvcc, *NVCC_FLAGS, *(extra_flags or []), "-c", "-o", str(obj) + ".tmp", str(source)]
        if verbose:
            print(" ".join(cmd), file=sys.stderr)
        running.append((obj, cmd, subprocess.Popen(cmd, cwd=str(REPO_ROOT))))
    failed = [cmd for _, cmd, process in running if process.wait() != 0]
    if failed:
        raise subprocess.CalledProcessError(1, failed[0])
    for obj, _, _ in running:
        os.replace(str(obj) + ".tmp", obj)
    tmp = LIBRARY.with_suffix(".so.tmp")
    link = [nvcc, *NVCC_FLAGS[:2], "-shared", "-o", str(tmp), *map(str, objects)]
    subprocess.run(link, check=True, cwd=str(REPO_ROOT))
    os.replace(tmp, LIBRARY)
    if extra_flags:  # objects of other flags are not kept for a later build
        for obj in objects:
            obj.unlink()
    return LIBRARY


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True, extra_flags=[a for a in sys.argv[1:] if a != "--force"])
