"""Build libsonata_b200.so in-tree with nvcc for sm_100a.

    python -m sonata_b200.build [--force] [--jobs N]

Each .cu under csrc/ is compiled to an object in sonata_b200/_build/ (in
parallel), then linked into sonata_b200/libsonata_b200.so with the CUDA
runtime linked statically, so the library only needs the driver at run time.
bind/fastcall.cpp, the short way from torch tensors to the C ABI, becomes
sonata_b200/_fastcall.*.so against the torch of this interpreter, which its
name says (host code only; the wrappers work without it, with more host time
a call, so a failure to build it is a warning).
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import os
import shutil
import subprocess
import sys
import sysconfig
import warnings
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
BUILD = PKG / "_build"
LIB = PKG / "libsonata_b200.so"
INCLUDE = PKG.parent / "include"
BIND_SRC = PKG / "bind" / "fastcall.cpp"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
              "-Xptxas", "-v", "-I", str(INCLUDE)]


def nvcc() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(cand).exists():
        raise RuntimeError("nvcc not found; the CUDA toolkit is required to build sonata_b200")
    return cand


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def _deps_mtime() -> float:
    files = list(CSRC.glob("*.cu")) + list(CSRC.glob("*.cuh")) + list(INCLUDE.glob("*.h"))
    return max(f.stat().st_mtime for f in files)


def _compile(src: Path) -> tuple[Path, str]:
    obj = BUILD / (src.stem + ".o")
    cmd = [nvcc(), *ARCH, *NVCC_FLAGS, "-c", str(src), "-o", str(obj)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src.name}:\n{r.stdout}\n{r.stderr}")
    (BUILD / (src.stem + ".ptxas.txt")).write_text(r.stderr)
    return obj, r.stderr


def bind_path() -> Path:
    """The short way's file for this interpreter and its torch: one built for others is never taken for it."""
    import torch
    return PKG / f"_fastcall.{sysconfig.get_config_var('SOABI')}-torch{torch.__version__}-abi{int(torch._C._GLIBCXX_USE_CXX11_ABI)}.so"


def build_bind(force: bool = False) -> Path:
    out = bind_path()
    if not force and out.exists() and out.stat().st_mtime >= max(
            f.stat().st_mtime for f in (BIND_SRC, *INCLUDE.glob("*.h"))):
        return out
    import torch
    from torch.utils import cpp_extension as ext
    cuda = Path(nvcc()).resolve().parent.parent
    include = [a for d in (*ext.include_paths(), cuda / "include", sysconfig.get_path("include")) for a in ("-isystem", str(d))]
    tmp = out.with_suffix(f".{os.getpid()}.tmp")
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-I", str(INCLUDE), *include, str(BIND_SRC),
           "-o", str(tmp), *["-L" + d for d in ext.library_paths()], "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed on {BIND_SRC.name}:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, out)
    return out


def build(force: bool = False, jobs: int | None = None, verbose: bool = False) -> Path:
    lib = _build_lib(force, jobs, verbose)
    try:
        build_bind(force)
    except Exception as e:  # no compiler, no headers of torch or Python, ...
        warnings.warn(f"the short way from torch tensors was not built, calls take more host time: {e}")
    return lib


def _build_lib(force: bool, jobs: int | None, verbose: bool) -> Path:
    if not force and LIB.exists() and LIB.stat().st_mtime >= _deps_mtime():
        return LIB
    BUILD.mkdir(exist_ok=True)
    srcs = sources()
    jobs = jobs or min(len(srcs), os.cpu_count() or 4)
    with cf.ThreadPoolExecutor(jobs) as ex:
        results = list(ex.map(_compile, srcs))
    if verbose:
        for obj, log in results:
            print(f"== {obj.name}\n{log}")
    tmp = LIB.with_suffix(f".{os.getpid()}.tmp")
    cmd = [nvcc(), *ARCH, "-shared", "-cudart", "static", "-o", str(tmp), *[str(o) for o, _ in results],
           ]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, LIB)
    return LIB


def main() -> int:
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--jobs", type=int, default=None)
    ap.add_argument("-v", "--verbose", action="store_true")
    a = ap.parse_args()
    print(build(force=a.force, jobs=a.jobs, verbose=a.verbose))
    return 0


if __name__ == "__main__":
    sys.exit(main())
