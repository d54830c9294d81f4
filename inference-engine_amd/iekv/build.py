"""Build libiekv.so and libiekv_ops.so (the HIP kernels and their C-ABIs) in-tree for gfx950.

The libraries are compiled with hipcc straight from ``csrc/`` into ``iekv/`` next to
this file, so they travel with the source tree and are the files ``iekv._native`` (the
handoff, from ``csrc/kv_handoff.hip``) and ``iekv._ops`` (attention and scoring, from
``csrc/attention.hip`` and ``csrc/logprobs.hip``) load. Run ``python -m iekv.build`` (with
``inference-engine_amd`` on ``sys.path``) or call :func:`build`.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
from pathlib import Path

PACKAGE_DIR = Path(__file__).resolve().parent
SOURCE_DIR = PACKAGE_DIR.parent / "csrc"
REPO_ROOT = PACKAGE_DIR.parent.parent
INCLUDE_DIR = REPO_ROOT / "include"
LIBRARY = PACKAGE_DIR / "libiekv.so"
SOURCES = [SOURCE_DIR / "kv_handoff.hip"]
OPS_LIBRARY = PACKAGE_DIR / "libiekv_ops.so"
OPS_SOURCES = [SOURCE_DIR / "attention.hip", SOURCE_DIR / "logprobs.hip"]
ARCH = "gfx950"


def hipcc() -> str:
    found = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not Path(found).exists():
        raise RuntimeError("hipcc not found: install ROCm or put hipcc on PATH")
    return found


def command(output: Path = LIBRARY, sources: list[Path] = SOURCES) -> list[str]:
    return [
        hipcc(),
        f"--offload-arch={ARCH}",
        "-O3",
        "-std=c++17",
        "-fPIC",
        "-shared",
        # Packed FP32 instructions stay disabled in every HIP build here.
        "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
        "-Wall",
        f"-I{INCLUDE_DIR}",
        *[str(s) for s in sources],
        "-o", str(output),
    ]


def _compile(library: Path, sources: list[Path], verbose: bool) -> Path:
    tmp = library.with_name(library.name + f".tmp{os.getpid()}")
    cmd = command(tmp, sources)
    if verbose:
        print(" ".join(cmd), flush=True)
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        tmp.unlink(missing_ok=True)
        raise RuntimeError(f"hipcc failed ({proc.returncode}):\n{proc.stdout}\n{proc.stderr}")
    os.replace(tmp, library)
    return library


def build(verbose: bool = False) -> Path:
    """Compile libiekv.so; raises RuntimeError with the compiler output on failure."""
    return _compile(LIBRARY, SOURCES, verbose)


def build_ops(verbose: bool = False) -> Path:
    """Compile libiekv_ops.so, as :func:`build` does libiekv.so."""
    return _compile(OPS_LIBRARY, OPS_SOURCES, verbose)


if __name__ == "__main__":
    for make in (build, build_ops):
        print(make(verbose="-v" in sys.argv))
