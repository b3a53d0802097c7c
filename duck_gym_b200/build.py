"""Builds the CUDA library ``duck_gym_b200/_lib/libduck_b200.so`` for sm_100a.

The library exports only the C ABI of ``include/duck_b200.h``; it does not
link against torch.  ``python -m duck_gym_b200.build`` rebuilds it.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import time
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PACKAGE = Path(__file__).resolve().parent
ROOT = PACKAGE.parent
SOURCES = sorted((PACKAGE / "csrc").glob("*.cu")) + sorted((PACKAGE / "csrc").glob("*.cuh")) + sorted(
    (PACKAGE / "csrc").glob("*.hpp")) + [ROOT / "include" / "duck_b200.h"]
UNITS = sorted((PACKAGE / "csrc").glob("*.cu"))   # one object each; they share no device code
LIB_DIR = PACKAGE / "_lib"
LIB_PATH = LIB_DIR / "libduck_b200.so"
OBJ_DIR = LIB_DIR / "obj"


def nvcc():
    home = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    path = Path(home) / "bin" / "nvcc"
    return str(path) if path.exists() else shutil.which("nvcc") or "nvcc"


def flags(verbose=False):
    f = [
        "-gencode", "arch=compute_100a,code=sm_100a",
        "-lineinfo", "-O3", "-std=c++17",
        "--expt-relaxed-constexpr",
        # Host code parses the model in double; keep its rounding identical to
        # the reference loader (no contraction).
        "-Xcompiler", "-fPIC,-ffp-contract=off",
        "-ccbin", "/usr/bin/g++",
    ]
    if verbose:
        f += ["-Xptxas", "-v"]
    return f


def up_to_date():
    if not LIB_PATH.exists():
        return False
    built = LIB_PATH.stat().st_mtime
    return all(p.stat().st_mtime <= built for p in SOURCES + [Path(__file__)])


def object_up_to_date(unit):
    """Whether a unit's object is newer than the files of this repository that
    its compilation read (listed by nvcc beside it) and than this file."""
    obj = OBJ_DIR / (unit.stem + ".o")
    deps = obj.with_suffix(".d")
    if not obj.exists() or not deps.exists():
        return False
    listed = [Path(w) for w in deps.read_text().replace("\\\n", " ").split(":", 1)[-1].split()]
    ours = [p for p in listed if not p.is_absolute() or ROOT in p.resolve().parents]
    if not ours or not all(p.exists() for p in ours):
        return False
    built = obj.stat().st_mtime
    return all(p.stat().st_mtime <= built for p in ours + [unit, Path(__file__)])


def run(cmd, verbose):
    result = subprocess.run(cmd, capture_output=True, text=True)
    if result.returncode != 0:
        raise RuntimeError("nvcc failed:\n" + " ".join(cmd) + "\n" + result.stdout + result.stderr)
    if verbose:
        sys.stderr.write(result.stdout + result.stderr)


def compile_unit(unit, verbose):
    obj = OBJ_DIR / (unit.stem + ".o")
    tmp = obj.with_suffix(".o.tmp")
    began = time.time()
    run([nvcc(), *flags(verbose), "-MD", "-MF", str(obj.with_suffix(".d")), "-c", str(unit), "-o", str(tmp)], verbose)
    os.utime(tmp, (began, began))   # a source changed while it was compiled is newer than its object
    tmp.replace(obj)


def build_library(force=False, verbose=False):
    """Compile the units with a newer source, at the same time, and link the
    library; return its path."""
    if not force and up_to_date():
        return LIB_PATH
    OBJ_DIR.mkdir(parents=True, exist_ok=True)
    stale = [u for u in UNITS if force or not object_up_to_date(u)]
    with ThreadPoolExecutor(max(1, len(stale))) as pool:
        list(pool.map(lambda u: compile_unit(u, verbose), stale))
    tmp = LIB_PATH.with_suffix(".so.tmp")
    began = min((OBJ_DIR / (u.stem + ".o")).stat().st_mtime for u in stale) if stale else time.time()
    run([nvcc(), *flags(), "-shared", *[str(OBJ_DIR / (u.stem + ".o")) for u in UNITS], "-o", str(tmp)], verbose)
    os.utime(tmp, (began, began))
    tmp.replace(LIB_PATH)
    return LIB_PATH


if __name__ == "__main__":
    print(build_library(force="--force" in sys.argv, verbose="-v" in sys.argv))
