"""Build the in-tree CUDA library ``librnn_kernel_b200.so`` for sm_100a.

``python -m rnn_kernel_b200.build`` (or ``build()``) compiles every ``.cu`` in
``csrc/`` with nvcc into one shared library next to this file.  The library
has a plain C ABI (``include/rnn_kernel_b200.h``) and is loaded with ctypes.
``csrc/host_*.cpp`` become the Python module ``_host`` beside it
(``build_host()``), which reads torch tensors' addresses for AdamW and makes the
usual calls of the newer operators.  The library needs nvcc alone; the module
needs a C++ compiler and the headers of the installed Python and torch (and of
CUDA, for the newer operators), and carries both versions in its file's name, so
that after an upgrade of either a new one is built and the old one left alone.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
# RNN_KERNEL_B200_VARIANT=timeline selects an instrumented build of the same
# sources (-DGRU_TIMELINE: the time loops record clock64() at the phases of a
# few steps, read back by gru_timeline_read) in a library of its own; it is
# slower by a few percent and only used for profiling (bench.py --timeline).
VARIANT = os.environ.get("RNN_KERNEL_B200_VARIANT", "")
if VARIANT not in ("", "timeline"):
    raise ValueError(f"RNN_KERNEL_B200_VARIANT must be unset or 'timeline', got {VARIANT!r}")
LIB_NAME = "librnn_kernel_b200_timeline.so" if VARIANT else "librnn_kernel_b200.so"
LIB_PATH = PKG / LIB_NAME
HOST_SOURCES = [CSRC / "host_tensors.cpp", CSRC / "host_operators.cpp"]
VARIANT_FLAGS = ["-DGRU_TIMELINE"] if VARIANT == "timeline" else []

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC", "-shared",
    "--expt-relaxed-constexpr",
]


def nvcc_path() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(cand).exists():
        raise RuntimeError("nvcc not found; the CUDA toolkit is required to build rnn_kernel_b200")
    return cand


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def _stale(built: Path, deps) -> bool:
    if not built.exists():
        return True
    mtime = built.stat().st_mtime
    return any(p.stat().st_mtime > mtime for p in [*deps, *(ROOT / "include").glob("*.h")])


def needs_build() -> bool:
    return _stale(LIB_PATH, CSRC.glob("*.cu*"))


def host_path() -> Path:
    """The module's file for this Python and this torch."""
    import torch

    return PKG / f"_host-torch{torch.__version__}{sysconfig.get_config_var('EXT_SUFFIX')}"


def host_parts(torch_base: Path) -> tuple[list[Path], list[str]]:
    """The module's sources and what they need besides torch: AdamW's part alone, without CUDA's headers or torch's part for it."""
    try:
        headers = Path(nvcc_path()).resolve().parent.parent / "include"
    except RuntimeError:
        headers = Path("/usr/local/cuda/include")
    if (headers / "cuda_runtime_api.h").exists() and (torch_base / "lib" / "libc10_cuda.so").exists():
        return HOST_SOURCES, [f"-I{headers}", "-lc10_cuda"]
    return HOST_SOURCES[:1], ["-DGRU_TENSORS_ONLY"]


def build_host(force: bool = False, verbose: bool = False) -> Path:
    """Compiles the module ``_host`` if it is missing or older than a source of its."""
    import torch

    path = host_path()
    if not force and not _stale(path, [*HOST_SOURCES, *CSRC.glob("host_*.h")]):
        return path
    base = Path(torch.__file__).parent
    tmp = path.with_name(f"{path.name}.{os.getpid()}.so.tmp")  # ranks may build at the same time
    include = [base / "include", base / "include/torch/csrc/api/include", sysconfig.get_paths()["include"]]
    files, cuda = host_parts(base)
    cmd = [shutil.which("g++") or "c++", "-O2", "-std=c++17", "-fPIC", "-shared",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", *(f"-I{i}" for i in include),
           *map(str, files), f"-L{base / 'lib'}", "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", *cuda, "-o", str(tmp)]
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    subprocess.run(cmd, check=True)
    os.replace(tmp, path)
    return path


def build(force: bool = False, verbose: bool = False, extra: list[str] | None = None) -> Path:
    """Compiles the CUDA library if it is missing or older than a source."""
    if not force and not needs_build():
        return LIB_PATH
    tmp = LIB_PATH.with_suffix(".so.tmp")
    cmd = [nvcc_path(), *NVCC_FLAGS, *VARIANT_FLAGS, *(extra or []), "-I", str(ROOT / "include"),
           *map(str, sources()), "-o", str(tmp)]
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    subprocess.run(cmd, check=True)
    os.replace(tmp, LIB_PATH)
    return LIB_PATH


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True,
          extra=["-Xptxas", "-v"] if "--ptxas" in sys.argv else None)
    try:
        build_host(force="--force" in sys.argv, verbose=True)
    except (OSError, subprocess.CalledProcessError) as e:
        print(f"the module _host was not built ({e}); its calls are made in Python", file=sys.stderr)
