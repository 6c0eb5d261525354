"""Build recipe for the in-tree sm_100a shared library and its torch binding.

``python -m testfiles_b200.build`` (or ``build_native()``) compiles the
``csrc/*.cu`` translation units with nvcc for ``sm_100a`` only into
``testfiles_b200/libwelm_rope_b200.so``.  The CUDA runtime is linked
statically, so the library loads on a machine without a GPU (the host-only
entry points then work; the device ones report a CUDA error).
``build_binding()`` compiles ``csrc/torch_binding.cpp`` against the installed
torch into the Python module ``testfiles_b200/_welm_torch.so``, which calls the
library; ``build_native()`` builds it too.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PACKAGE_DIR = Path(__file__).resolve().parent
REPO_ROOT = PACKAGE_DIR.parent
CSRC = PACKAGE_DIR / "csrc"
# one translation unit per kernel family; the .cuh headers hold what they share
SOURCES = tuple(CSRC / name for name in (
    "rope_ordinary.cu", "rope_mirror.cu", "rope_kv_write.cu", "rope_tiles.cu", "rope_host_memory.cu",
    "rope_ceiling.cu", "rope_multi_axis.cu", "rope_kv_append.cu", "rope_attend.cu", "rope_abi.cu"))
HEADERS = (REPO_ROOT / "include" / "welm_rope.h", *(CSRC / name for name in (
    "rope_device.cuh", "rope_host.cuh", "rope_axes.cuh", "rope_rows.h", "rope_tma.cuh")))
LIBRARY = PACKAGE_DIR / "libwelm_rope_b200.so"
BINDING_SOURCE = CSRC / "torch_binding.cpp"
BINDING = PACKAGE_DIR / "_welm_torch.so"

NVCC_FLAGS = (
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo",
    "-O3",
    "-std=c++17",
    "-Xcompiler", "-fPIC,-O2,-Wall",
    "-shared",
)


def _nvcc() -> str:
    for candidate in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if candidate and Path(candidate).exists():
            return candidate
    raise RuntimeError("nvcc not found: the sm_100a library cannot be built")


def _stale() -> bool:
    if not LIBRARY.exists():
        return True
    built = LIBRARY.stat().st_mtime
    return any(src.stat().st_mtime > built for src in SOURCES + HEADERS)


def build_native(force: bool = False, verbose: bool = False, extra_flags: tuple[str, ...] = ()) -> Path:
    """Compile the library and the binding if they are missing or older than their sources."""
    if force or _stale():
        _build_library(verbose, extra_flags)
    build_binding(force, verbose)
    return LIBRARY


def _build_library(verbose: bool, extra_flags: tuple[str, ...]) -> None:
    tmp = LIBRARY.with_suffix(".so.tmp")
    cmd = [
        _nvcc(), *NVCC_FLAGS, *extra_flags,
        "-I", str(REPO_ROOT / "include"),
        *(str(s) for s in SOURCES),
        "-o", str(tmp),
    ]
    if verbose:
        print(" ".join(cmd), flush=True)
    _run("nvcc", cmd, verbose)
    os.replace(tmp, LIBRARY)


def build_binding(force: bool = False, verbose: bool = False) -> Path:
    """Compile the torch binding if it is missing or older than its source or the installed torch."""
    import torch

    torch_dir = Path(torch.__file__).resolve().parent
    newer = (BINDING_SOURCE, CSRC / "rope_rows.h", REPO_ROOT / "include" / "welm_rope.h", torch_dir / "version.py")
    if not force and BINDING.exists() and all(p.stat().st_mtime <= BINDING.stat().st_mtime for p in newer):
        return BINDING
    cuda = Path(_nvcc()).resolve().parent.parent
    tmp = BINDING.with_suffix(".so.tmp")
    cmd = [
        shutil.which("g++") or "c++", "-std=c++17", "-O2", "-Wall", "-fPIC", "-shared", "-fvisibility=hidden",
        f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
        "-I", str(REPO_ROOT / "include"),
        "-I", str(CSRC),
        "-isystem", str(torch_dir / "include"),
        "-isystem", str(torch_dir / "include" / "torch" / "csrc" / "api" / "include"),
        "-isystem", str(cuda / "include"),
        "-isystem", sysconfig.get_paths()["include"],
        str(BINDING_SOURCE),
        "-L", str(torch_dir / "lib"), "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10_cuda", "-lc10",
        "-L", str(PACKAGE_DIR), f"-l:{LIBRARY.name}", "-Wl,-rpath,$ORIGIN",
        "-o", str(tmp),
    ]
    if verbose:
        print(" ".join(cmd), flush=True)
    _run("g++", cmd, verbose)
    os.replace(tmp, BINDING)
    return BINDING


def _run(tool: str, cmd: list[str], verbose: bool) -> None:
    result = subprocess.run(cmd, capture_output=True, text=True)
    if result.returncode != 0:
        raise RuntimeError(f"{tool} failed ({result.returncode}):\n{result.stdout}\n{result.stderr}")
    if verbose and (result.stdout or result.stderr):
        print(result.stdout + result.stderr, flush=True)


if __name__ == "__main__":
    args = set(sys.argv[1:])
    path = build_native(force="--force" in args, verbose=True,
                        extra_flags=("-Xptxas", "-v") if "--ptxas-v" in args else ())
    print(path)
