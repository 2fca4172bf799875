"""Build libeas_cuda.so in-tree with nvcc for sm_100a.

Run ``python -m easy_as_b200.build``.  The library lands in
``easy_as_b200/_lib/libeas_cuda.so`` so that it ships with the source tree
(no site-packages install, no JIT cache).  Where torch is installed, the
extension ``_lib/eas_ops.so`` (the quick way of :mod:`easy_as_b200.ops` for
torch tensors, host code only) is built beside it against that torch.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
LIB_DIR = PKG / "_lib"
LIB = LIB_DIR / "libeas_cuda.so"
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found (set NVCC or put /usr/local/cuda/bin on PATH)")


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def _flags(ptxas_verbose: bool = False) -> list[str]:
    return [*ARCH, "-O3", "-lineinfo", "-std=c++17", "-shared", "-Xcompiler", "-fPIC", "-cudart", "static", "-t0",
            *(["-Xptxas", "-v"] if ptxas_verbose else [])]


def source_hash() -> str:
    """sha256 over every source and header the library is built from, and the nvcc flags."""
    import hashlib

    h = hashlib.sha256()
    deps = sources() + sorted(CSRC.glob("*.h")) + sorted(CSRC.glob("*.cuh")) + [PKG.parent / "include" / "eas_cuda.h"]
    for p in deps:
        if p.exists():
            h.update(p.name.encode() + b"\0" + p.read_bytes() + b"\0")
    h.update(" ".join(_flags()).encode())
    return h.hexdigest()


STAMP = LIB.with_name(LIB.name + ".sha256")


def needs_build() -> bool:
    """Rebuild unless the library exists and its stamp (written beside it by the build that made it)
    matches the current sources and flags; file times play no part."""
    if not LIB.exists() or not STAMP.exists():
        return True
    return STAMP.read_text().strip() != source_hash()


OPS_SOURCE = CSRC / "ops_torch.cpp"
OPS = LIB_DIR / "eas_ops.so"
OPS_STAMP = OPS.with_name(OPS.name + ".sha256")


def ops_hash() -> str | None:
    """sha256 over the extension's source and what it is built against; None without torch."""
    import hashlib
    import importlib.metadata

    try:
        torch = importlib.metadata.version("torch")
    except importlib.metadata.PackageNotFoundError:
        return None
    h = hashlib.sha256(OPS_SOURCE.read_bytes())
    h.update(f"{torch} {sys.version} {' '.join(_OPS_FLAGS)}".encode())
    return h.hexdigest()


_OPS_FLAGS = ["-O2", "-std=c++17", "-shared", "-fPIC", "-w"]


def build_ops(verbose: bool = False, force: bool = False) -> Path | None:
    """Build the torch extension of ``eas.ops`` (None without torch)."""
    digest = ops_hash()
    if digest is None:
        return None
    if not force and OPS.exists() and OPS_STAMP.exists() and OPS_STAMP.read_text().strip() == digest:
        return OPS
    import sysconfig

    import torch

    root = Path(torch.__file__).resolve().parent
    cuda = Path(nvcc()).resolve().parent.parent
    LIB_DIR.mkdir(parents=True, exist_ok=True)
    tmp = OPS.with_suffix(".so.tmp")
    include = [root / "include", root / "include" / "torch" / "csrc" / "api" / "include", cuda / "include",
               sysconfig.get_paths()["include"]]
    cmd = [os.environ.get("CXX", "g++"), *_OPS_FLAGS, f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *[f"-I{d}" for d in include], str(OPS_SOURCE), "-o", str(tmp), "-L", str(root / "lib"), "-lc10", "-lc10_cuda",
           "-ltorch_cpu", "-ltorch_python"]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"{cmd[0]} failed ({res.returncode}):\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, OPS)
    OPS_STAMP.write_text(digest + "\n")
    return OPS


def build(verbose: bool = False, force: bool = False, ptxas_verbose: bool = False) -> Path:
    try:
        build_ops(verbose, force)
    except Exception as e:   # whatever a broken torch raises: the library does not need it, eas.ops then takes its full path
        print(f"eas_ops extension not built: {e}", file=sys.stderr)
    if not force and not needs_build():
        return LIB
    LIB_DIR.mkdir(parents=True, exist_ok=True)
    tmp = LIB.with_suffix(".so.tmp")
    digest = source_hash()
    cmd = [nvcc(), *_flags(ptxas_verbose), "-I", str(PKG.parent / "include"), "-I", str(CSRC),
           *map(str, sources()), "-o", str(tmp), "-ldl", "-lpthread"]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed ({res.returncode}):\n{res.stdout}\n{res.stderr}")
    if verbose or ptxas_verbose:
        sys.stdout.write(res.stdout + res.stderr)
    os.replace(tmp, LIB)
    STAMP.write_text(digest + "\n")
    return LIB


if __name__ == "__main__":
    args = sys.argv[1:]
    print(build(verbose=True, force="--force" in args, ptxas_verbose="-v" in args))
