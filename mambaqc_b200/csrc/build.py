"""Build ``mambaqc_b200/libmambaqc_b200.so`` from the CUDA/C++ sources in this folder.

Plain nvcc, in-tree, for sm_100a only:

    python -m mambaqc_b200.csrc.build            # incremental
    python -m mambaqc_b200.csrc.build --force    # rebuild everything
    MQC_PTXAS_VERBOSE=1 python -m mambaqc_b200.csrc.build --force   # -Xptxas -v

The library has a pure C ABI (``include/mambaqc_b200.h``) and links the CUDA
runtime statically, so it carries no torch dependency; the Python package loads
it with ctypes. The operators of the training step are bound by a small torch
extension beside it (``csrc/torch/ops.cpp`` -> ``mambaqc_b200/_torch_ops.so``, built
with g++ against the installed torch), which calls the same C ABI.
"""

from __future__ import annotations

import argparse
import concurrent.futures as cf
import importlib.util
import os
import shutil
import subprocess
import sys
from pathlib import Path

CSRC = Path(__file__).resolve().parent
PKG = CSRC.parent
ROOT = PKG.parent
INCLUDE = ROOT / "include"
BUILD_DIR = PKG / "_build"
LIB = PKG / "libmambaqc_b200.so"
OPS_SOURCE = CSRC / "torch" / "ops.cpp"
OPS_LIB = PKG / "_torch_ops.so"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-std=c++17", "-lineinfo", "--expt-relaxed-constexpr",
              "-Xcompiler", "-fPIC,-O3,-fvisibility=hidden", "-Xfatbin", "-compress-all"]


def _nvcc() -> str:
    cuda_home = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    cand = Path(cuda_home) / "bin" / "nvcc"
    if cand.exists():
        return str(cand)
    found = shutil.which("nvcc")
    if not found:
        raise RuntimeError("nvcc not found (set CUDA_HOME)")
    return found


def _sources() -> list[Path]:
    return sorted([*CSRC.glob("*.cu"), *CSRC.glob("*.cpp")])


def _headers() -> list[Path]:
    return sorted([*CSRC.glob("*.cuh"), *CSRC.glob("*.h"), *INCLUDE.glob("*.h")])


def _compile(src: Path, verbose_ptxas: bool) -> tuple[Path, str]:
    obj = BUILD_DIR / (src.name + ".o")
    cmd = [_nvcc(), *ARCH, *NVCC_FLAGS, f"-I{INCLUDE}", f"-I{CSRC}", "-c", str(src), "-o", str(obj)]
    if verbose_ptxas:
        cmd[1:1] = ["-Xptxas", "-v"]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src.name}:\n{proc.stdout}\n{proc.stderr}")
    return obj, proc.stdout + proc.stderr


def build(force: bool = False, jobs: int | None = None, quiet: bool = False) -> Path:
    BUILD_DIR.mkdir(exist_ok=True)
    srcs = _sources()
    newest_header = max((h.stat().st_mtime for h in _headers()), default=0.0)
    verbose_ptxas = os.environ.get("MQC_PTXAS_VERBOSE") == "1"
    todo = []
    for s in srcs:
        obj = BUILD_DIR / (s.name + ".o")
        if (force or verbose_ptxas or not obj.exists()
                or obj.stat().st_mtime < max(s.stat().st_mtime, newest_header)):
            todo.append(s)
    jobs = jobs or min(len(todo) or 1, os.cpu_count() or 4)
    with cf.ThreadPoolExecutor(max_workers=jobs) as ex:
        for obj, log in ex.map(lambda s: _compile(s, verbose_ptxas), todo):
            if log.strip() and (verbose_ptxas or not quiet):
                print(f"[{obj.name}]\n{log}", file=sys.stderr)
    objs = [BUILD_DIR / (s.name + ".o") for s in srcs]
    if todo or not LIB.exists() or LIB.stat().st_mtime < max(o.stat().st_mtime for o in objs):
        tmp = LIB.with_suffix(".so.tmp")
        cmd = [_nvcc(), *ARCH, "-shared", "-o", str(tmp), *map(str, objs), "-cudart", "static"]
        proc = subprocess.run(cmd, capture_output=True, text=True)
        if proc.returncode != 0:
            raise RuntimeError(f"link failed:\n{proc.stdout}\n{proc.stderr}")
        os.replace(tmp, LIB)
        if not quiet:
            print(f"built {LIB}", file=sys.stderr)
    build_torch_ops(force=force, quiet=quiet)
    return LIB


def build_torch_ops(force: bool = False, quiet: bool = False) -> Path | None:
    """The torch extension; compiled again when its source or the header is newer, or
    when it was built for another torch or Python. None, with a message, where torch, its
    headers or g++ are missing: the C library does without them."""
    missing = None
    if importlib.util.find_spec("torch") is None:
        missing = "torch"
    elif shutil.which("g++") is None:
        missing = "g++"
    else:
        import torch

        root = Path(torch.__file__).resolve().parent
        if not (root / "include" / "torch" / "extension.h").exists():
            missing = "torch's headers"
    if missing:
        print(f"{OPS_LIB.name} is not built: no {missing} (the C library is; the operators of "
              "the training stack need both)", file=sys.stderr)
        return None
    built_for = f"torch {torch.__version__}, Python {sys.version_info[0]}.{sys.version_info[1]}"
    newest = max(p.stat().st_mtime for p in (OPS_SOURCE, INCLUDE / "mambaqc_b200.h"))
    if not force and OPS_LIB.exists() and OPS_LIB.stat().st_mtime >= newest \
            and f"mqc built for {built_for};".encode() in OPS_LIB.read_bytes():
        return OPS_LIB
    import sysconfig

    cuda_home = Path(_nvcc()).resolve().parents[1]
    include = [root / "include", root / "include" / "torch" / "csrc" / "api" / "include",
               cuda_home / "include", Path(sysconfig.get_paths()["include"]), INCLUDE]
    tmp = OPS_LIB.with_suffix(".so.tmp")
    cmd = ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           "-DTORCH_EXTENSION_NAME=_torch_ops", f'-DMQC_BUILT_FOR="mqc built for {built_for};"', *[f"-I{p}" for p in include], str(OPS_SOURCE),
           "-o", str(tmp), f"-L{root / 'lib'}", "-lc10", "-lc10_cuda", "-ltorch_cpu",
           "-ltorch_cuda", "-ltorch", "-ltorch_python", "-ldl"]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"g++ failed for {OPS_SOURCE.name}:\n{proc.stdout}\n{proc.stderr}")
    os.replace(tmp, OPS_LIB)
    if not quiet:
        print(f"built {OPS_LIB}", file=sys.stderr)
    return OPS_LIB


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--force", action="store_true")
    ap.add_argument("-j", "--jobs", type=int, default=None)
    args = ap.parse_args()
    build(force=args.force, jobs=args.jobs)


if __name__ == "__main__":
    main()
