"""Build the sm_100a C-ABI library ``libh3b200.so`` in-tree with nvcc.

Each ``csrc/*.cu`` compiles to an object under ``_build/`` (rebuilt only when it
or a header is newer), in parallel, then nvcc links the shared library next to
this file.  The CUDA runtime is linked statically; driver entry points
(cuTensorMapEncodeTiled) are resolved at run time through
cudaGetDriverEntryPoint, so the library needs no libcuda at link time.
"""
from __future__ import annotations

import concurrent.futures
import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
INCLUDE = PKG.parent / "include"
BUILD = PKG.parent / "_build"
LIB = PKG / "libh3b200.so"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-Xcompiler", "-O3",
         "--expt-relaxed-constexpr", "-I", str(INCLUDE), "-I", str(CSRC)]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found")


def _headers() -> list[Path]:
    return sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.h")) + sorted(INCLUDE.glob("*.h"))


def _compile(nvcc: str, src: Path, obj: Path, newest_header: float, verbose: bool) -> Path:
    if obj.exists() and obj.stat().st_mtime >= max(src.stat().st_mtime, newest_header):
        return obj
    cmd = [nvcc, *ARCH, *FLAGS, "-c", str(src), "-o", str(obj)]
    if verbose:
        cmd += ["-Xptxas", "-v"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src.name}:\n{res.stdout}\n{res.stderr}")
    if verbose and res.stderr:
        sys.stderr.write(res.stderr)
    return obj


def build(verbose: bool = False, jobs: int | None = None) -> Path:
    nvcc = _nvcc()
    BUILD.mkdir(exist_ok=True)
    sources = sorted(CSRC.glob("*.cu"))
    newest_header = max((h.stat().st_mtime for h in _headers()), default=0.0)
    objs = [BUILD / (s.stem + ".o") for s in sources]
    with concurrent.futures.ThreadPoolExecutor(max_workers=jobs or min(8, os.cpu_count() or 1)) as ex:
        list(ex.map(lambda so: _compile(nvcc, so[0], so[1], newest_header, verbose), zip(sources, objs)))
    if not LIB.exists() or LIB.stat().st_mtime < max(o.stat().st_mtime for o in objs):
        tmp = LIB.with_suffix(".so.tmp")
        cmd = [nvcc, *ARCH, "-shared", "-Xcompiler", "-fPIC", "-o", str(tmp), *map(str, objs),
               "-cudart", "static"]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
        os.replace(tmp, LIB)
    return LIB


def host_path() -> Path:
    """The extension of csrc/host_calls.cpp for this Python and this torch, whose C++ layouts it
    is compiled against: under another of either it is another file, and built again."""
    import torch
    return PKG / f"_h3host.{sys.implementation.cache_tag}-torch{torch.__version__}.so"


def build_host(verbose: bool = False) -> Path:
    """The Python extension over torch's C++ headers (the host compiler, no nvcc)."""
    import sysconfig

    import torch
    src, out = CSRC / "host_calls.cpp", host_path()
    newest = max(src.stat().st_mtime, (INCLUDE / "h3_b200.h").stat().st_mtime)
    if out.exists() and out.stat().st_mtime >= newest:
        return out
    root = Path(torch.__path__[0])
    cuda = Path(_nvcc()).resolve().parent.parent / "include"
    includes = [sysconfig.get_path("include"), root / "include", root / "include/torch/csrc/api/include", cuda]
    tmp = out.with_suffix(".tmp")
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-w",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *[f"-I{i}" for i in includes], str(src), "-o", str(tmp), f"-L{root / 'lib'}",
           "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda", f"-Wl,-rpath,{root / 'lib'}"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"building {out.name} failed:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, out)
    if verbose:
        print(out)
    return out


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
    print(build_host())
