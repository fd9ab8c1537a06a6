"""In-tree build of the sm_100a kernel library ``tokenforge_b200/lib/libtokenforge_b200.so``.

Every ``csrc/*.cu`` file is compiled by ``nvcc`` for ``sm_100a`` (``-gencode
arch=compute_100a,code=sm_100a``) into ``_build/`` and linked into one shared library with the
CUDA runtime linked statically, so the library has no dependency beyond the driver. The C ABI
it exports is declared in ``include/tokenforge_b200.h``.

Beside it, ``lib/fp8_host.*.so`` is the host fast path of the FP8 operators (``csrc/host``), a
CPython extension compiled by the host compiler against PyTorch's headers (a file for each PyTorch
and CPython it is built against).

    python -m tokenforge_b200._build [--force] [--verbose]
"""

from __future__ import annotations

import argparse
import concurrent.futures as cf
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
BUILD = PKG / "_build"
LIB = PKG / "lib" / "libtokenforge_b200.so"
HOST_SRC = CSRC / "host" / "fp8_host.cpp"
INCLUDE = ROOT / "include"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = [
    *ARCH,
    "-lineinfo",
    "-O3",
    "-std=c++17",
    "-Xcompiler",
    "-fPIC",
    "-Xcompiler",
    "-fvisibility=hidden",
    "--expt-relaxed-constexpr",
    f"-I{INCLUDE}",
]


def nvcc() -> str:
    path = shutil.which("nvcc")
    if path is None:
        cand = Path("/usr/local/cuda/bin/nvcc")
        if cand.exists():
            return str(cand)
        raise RuntimeError("nvcc not found: the CUDA toolkit is required to build tokenforge_b200")
    return path


def _sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def _headers() -> list[Path]:
    return sorted([*CSRC.glob("*.cuh"), *CSRC.glob("*.h"), *INCLUDE.glob("*.h")])


def _stale(target: Path, deps: list[Path]) -> bool:
    if not target.exists():
        return True
    t = target.stat().st_mtime
    return any(d.stat().st_mtime > t for d in deps)


def _compile(src: Path, verbose: bool) -> Path:
    obj = BUILD / (src.stem + ".o")
    cmd = [nvcc(), *NVCC_FLAGS, "-c", str(src), "-o", str(obj)]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src.name}:\n{proc.stderr}")
    if verbose and proc.stderr:
        print(proc.stderr, file=sys.stderr)
    return obj


def _build_host(force: bool) -> None:
    """The CPython extension: linked against PyTorch and the kernel library next to it."""
    import torch

    from tokenforge_b200 import _lib

    target = _lib.host_path()
    if not force and not _stale(target, [HOST_SRC, LIB, *INCLUDE.glob("*.h")]):
        return
    cxx = os.environ.get("CXX") or shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        raise RuntimeError("g++ not found: a C++ compiler is required to build tokenforge_b200")
    pt = Path(torch.__file__).resolve().parent
    cuda = Path(nvcc()).resolve().parent.parent
    tmp = target.with_suffix(".so.tmp")
    cmd = [
        cxx, "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
        f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
        f"-I{pt / 'include'}", f"-I{pt / 'include/torch/csrc/api/include'}",
        f"-I{cuda / 'include'}", f"-I{sysconfig.get_paths()['include']}", str(HOST_SRC),
        "-o", str(tmp), f"-L{LIB.parent}", "-ltokenforge_b200", f"-L{pt / 'lib'}",
        "-ltorch_python", "-ltorch_cuda", "-ltorch_cpu", "-ltorch", "-lc10", "-lc10_cuda",
        "-Wl,-rpath,$ORIGIN",
    ]  # fmt: skip
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"{cxx} failed on {HOST_SRC.name}:\n{proc.stderr}")
    os.replace(tmp, target)


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile and link the kernel library if any source is newer than it. Returns its path."""
    BUILD.mkdir(exist_ok=True)
    LIB.parent.mkdir(exist_ok=True)
    headers = _headers()
    todo = [s for s in _sources() if force or _stale(BUILD / (s.stem + ".o"), [s, *headers])]
    if todo:
        workers = min(len(todo), os.cpu_count() or 4)
        with cf.ThreadPoolExecutor(workers) as pool:
            list(pool.map(lambda s: _compile(s, verbose), todo))
    objs = [BUILD / (s.stem + ".o") for s in _sources()]
    if force or todo or _stale(LIB, objs):
        tmp = LIB.with_suffix(".so.tmp")
        cmd = [nvcc(), *ARCH, "-shared", "-cudart", "static", "-o", str(tmp), *map(str, objs)]
        proc = subprocess.run(cmd, capture_output=True, text=True)
        if proc.returncode != 0:
            raise RuntimeError(f"link failed:\n{proc.stderr}")
        os.replace(tmp, LIB)
    _build_host(force)
    return LIB


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    args = ap.parse_args()
    print(build(force=args.force, verbose=args.verbose))


if __name__ == "__main__":
    main()
