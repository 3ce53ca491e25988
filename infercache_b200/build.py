"""Build the sm_100a C-ABI library and its Python binding in-tree.

    python -m infercache_b200.build [--force] [--verbose]

Compiles every ``csrc/*.cu`` with nvcc for ``sm_100a`` (cross-compiles on a
machine without a GPU) and links ``lib/libinfercache_b200.so`` with the CUDA
runtime linked statically, so the library does not depend on which
libcudart the host process loaded first.  Then compiles ``csrc/binding.cpp``
(the paged serving tick's calls on torch tensors) with g++ against the torch
that runs this, as ``lib/_binding.so``; without a CUDA build of torch or
Python's headers the library is built alone.
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import os
import shutil
import subprocess
import sys
from pathlib import Path
from typing import Optional

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
OBJ = PKG / "_build"
LIBDIR = PKG / "lib"
LIB = LIBDIR / "libinfercache_b200.so"
BINDING = LIBDIR / "_binding.so"
HEADERS = [ROOT / "include" / "infercache.h"] + sorted(CSRC.glob("*.cuh"))

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC,-O3",
              "--expt-relaxed-constexpr", "-I", str(ROOT / "include")]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found")


def _stale(target: Path, deps) -> bool:
    if not target.exists():
        return True
    t = target.stat().st_mtime
    return any(d.stat().st_mtime > t for d in deps)


def build(force: bool = False, verbose: bool = False) -> Path:
    sources = sorted(CSRC.glob("*.cu"))
    OBJ.mkdir(exist_ok=True)
    LIBDIR.mkdir(exist_ok=True)
    cc = nvcc()
    jobs = []
    for src in sources:
        obj = OBJ / (src.stem + ".o")
        if force or _stale(obj, [src] + HEADERS):
            cmd = [cc, *ARCH, *NVCC_FLAGS, "-c", str(src), "-o", str(obj)]
            if verbose:
                cmd += ["-Xptxas", "-v"]
            jobs.append((src, cmd))
    if jobs:
        with cf.ThreadPoolExecutor(max_workers=min(len(jobs), os.cpu_count() or 4)) as ex:
            futs = {ex.submit(subprocess.run, cmd, capture_output=True, text=True): src for src, cmd in jobs}
            for f in cf.as_completed(futs):
                r = f.result()
                if verbose or r.returncode != 0:
                    sys.stderr.write(r.stdout + r.stderr)
                if r.returncode != 0:
                    raise RuntimeError(f"nvcc failed on {futs[f].name}")
    objs = [OBJ / (s.stem + ".o") for s in sources]
    if force or jobs or _stale(LIB, objs):
        cmd = [cc, *ARCH, "-shared", "-cudart", "static", "-o", str(LIB), *map(str, objs)]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            sys.stderr.write(r.stdout + r.stderr)
            raise RuntimeError("link failed")
    build_binding(force)
    return LIB


def _python_include() -> Path:
    import sysconfig
    return Path(sysconfig.get_paths()["include"])


def _no_binding() -> str:
    """Why the binding cannot be built here ('' when it can)."""
    import torch
    if torch.version.cuda is None:
        return f"torch {torch.__version__} is not a CUDA build"
    if not (_python_include() / "Python.h").exists():
        return f"Python's headers are not in {_python_include()}"
    if not shutil.which("g++"):
        return "g++ not found"
    return ""


def build_binding(force: bool = False) -> Optional[Path]:
    """The binding, or None, with a line on stderr, where torch, Python's headers
    or g++ do not allow it; the C-ABI library does not need them."""
    why = _no_binding()
    if why:
        sys.stderr.write(f"the paged serving tick's binding is not built: {why}\n")
        return None
    import torch
    from torch.utils.cpp_extension import include_paths, library_paths
    src = CSRC / "binding.cpp"
    cmd = [shutil.which("g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", f'-DIC_TORCH_VERSION="{torch.__version__}"',
           *(f"-I{d}" for d in [*include_paths(), _python_include(), Path(nvcc()).resolve().parents[1] / "include"]), str(src),
           "-o", str(BINDING), f"-L{LIBDIR}", "-linfercache_b200", "-Wl,-rpath,$ORIGIN",
           *(f"-L{d}" for d in library_paths()), *(f"-Wl,-rpath,{d}" for d in library_paths()),
           "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python"]
    # the command names the torch, Python and compiler that it is built for: with
    # others it is another one
    OBJ.mkdir(exist_ok=True)
    made_by = OBJ / "binding.cmd"
    if (not force and not _stale(BINDING, [src, ROOT / "include" / "infercache.h"]) and made_by.exists()
            and made_by.read_text() == "\n".join(cmd)):
        return BINDING
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise RuntimeError("g++ failed on binding.cpp")
    made_by.write_text("\n".join(cmd))
    return BINDING


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    args = ap.parse_args()
    print(build(args.force, args.verbose))


if __name__ == "__main__":
    main()
