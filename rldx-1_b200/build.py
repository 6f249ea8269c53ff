"""Builds librldx_b200.so (all sm_100a kernels + the C ABI) and the Python binding of the token-decoding
operators in this package directory.

The library is one nvcc translation unit (csrc/rldx_b200.cu) compiled for sm_100a only:
no PTX for other architectures is embedded, so it loads only on B200-class GPUs.  The binding is
host C++ against the installed torch's headers; it is good for that torch and that Python only, so its file
name says which, and without torch the library is built alone.
"""

from __future__ import annotations

import importlib.metadata
import importlib.util
import os
import re
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
CSRC = PKG_DIR / "csrc"
LIB_NAME = "librldx_b200.so"
LIB_PATH = PKG_DIR / LIB_NAME
BINDING_SOURCES = [CSRC / "torch_binding.cpp", PKG_DIR.parent / "include" / "rldx_b200.h"]

NVCC_FLAGS = [
    "-gencode",
    "arch=compute_100a,code=sm_100a",
    "-O3",
    "-lineinfo",
    "-std=c++17",
    "-Xcompiler",
    "-fPIC",
    "-shared",
]


def _sources() -> list[Path]:
    return sorted(list(CSRC.glob("*.cu")) + list(CSRC.glob("*.cuh")) + list(CSRC.glob("*.h"))) + [
        PKG_DIR.parent / "include" / "rldx_b200.h"
    ]


def _nvcc() -> str:
    cand = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    return cand


def needs_build() -> bool:
    if not LIB_PATH.exists():
        return True
    lib_mtime = LIB_PATH.stat().st_mtime
    return any(p.stat().st_mtime > lib_mtime for p in _sources() if p.exists())


def torch_version() -> str | None:
    """Of the installed torch, without importing it; None: there is none."""
    try:
        return importlib.metadata.version("torch")
    except importlib.metadata.PackageNotFoundError:
        return None


def binding_path() -> Path:
    """The binding of this Python and the installed torch, whose C++ interfaces it is compiled against."""
    tag = f"{sysconfig.get_config_var('SOABI')}-torch{torch_version()}"
    return PKG_DIR / f"_torch_binding.{re.sub(r'[^A-Za-z0-9_.+-]', '_', tag)}.so"


def binding_needs_build() -> bool:
    path = binding_path()
    if not path.exists():
        return True
    mtime = path.stat().st_mtime
    return any(p.stat().st_mtime > mtime for p in BINDING_SOURCES if p.exists())


def _temporary(path: Path) -> Path:
    """Where this process compiles `path`: ranks that build at once do not share it."""
    return path.with_name(f"{path.name}.{os.getpid()}.tmp")


def _compile(cmd: list[str], tmp: Path, path: Path) -> str:
    """Runs a compiler that writes `tmp`, which then takes the place of `path`; returns what it had to say."""
    try:
        res = subprocess.run(cmd, cwd=str(CSRC), capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"{cmd[0]} failed ({res.returncode}):\n{res.stdout}\n{res.stderr}")
        os.replace(tmp, path)
    finally:
        tmp.unlink(missing_ok=True)
    return res.stderr


def build_binding(force: bool = False) -> Path:
    """Compiles the Python binding if a source is newer than it (or when forced)."""
    path = binding_path()
    if not force and not binding_needs_build():
        return path
    spec = importlib.util.find_spec("torch")
    if spec is None or spec.origin is None:
        raise RuntimeError("torch is not installed: its headers are needed to build the binding")
    torch_dir = Path(spec.origin).parent
    nvcc = Path(_nvcc()).resolve()
    include = [torch_dir / "include", torch_dir / "include" / "torch" / "csrc" / "api" / "include",
               Path(sysconfig.get_paths()["include"]), nvcc.parents[1] / "include"]
    tmp = _temporary(path)
    cmd = [os.environ.get("CXX") or "g++", "-O2", "-std=c++17", "-shared", "-fPIC", *[f"-I{p}" for p in include],
           str(BINDING_SOURCES[0]), "-o", str(tmp), f"-L{torch_dir / 'lib'}", "-lc10", "-lc10_cuda", "-ltorch_cpu",
           "-ltorch_cuda", "-ltorch_python", "-ltorch"]
    _compile(cmd, tmp, path)
    return path


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compiles the library and, where torch is installed, the binding if a source is newer than the .so (or when
    forced)."""
    if torch_version() is not None:
        build_binding(force)
    if not force and not needs_build():
        return LIB_PATH
    tmp = _temporary(LIB_PATH)
    cmd = [_nvcc(), *NVCC_FLAGS, str(CSRC / "rldx_b200.cu"), "-o", str(tmp)]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
        print(" ".join(cmd), file=sys.stderr)
    err = _compile(cmd, tmp, LIB_PATH)
    if verbose and err:
        print(err, file=sys.stderr)
    return LIB_PATH


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(LIB_PATH)
