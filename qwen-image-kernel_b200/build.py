"""Build libqik.so (the C-ABI CUDA library) in-tree for sm_100a.

    python qwen-image-kernel_b200/build.py [--force] [--verbose-ptxas]

Each .cu under csrc/ is compiled by nvcc to an object (in csrc/_build/) and linked
into qik/libqik.so with the CUDA runtime linked statically, so the library has no
dependency beyond the driver.  Objects are rebuilt when their source or any header
is newer.

The host calls of the decoder operators (csrc/calls.cpp) are a CPython module over torch's
C++ tensors, compiled by g++ to qik/_calls.so and linked against libqik.so beside it; it is made again
when the Python or the torch that it was compiled against is another one.
"""
from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys
from pathlib import Path

HERE = Path(__file__).resolve().parent
CSRC = HERE / "csrc"
OBJ = CSRC / "_build"
INCLUDE = HERE.parent / "include"
OUT = HERE / "qik" / "libqik.so"
CALLS = HERE / "qik" / "_calls.so"
CALLS_MADE_FOR = OBJ / "_calls.made_for"   # the Python and torch that _calls.so was compiled against

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr", "-Xptxas",
         "-warn-spills", "-I", str(INCLUDE)]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found")


def build(force: bool = False, verbose_ptxas: bool = False) -> Path:
    OBJ.mkdir(parents=True, exist_ok=True)
    headers = list(CSRC.glob("*.cuh")) + list(CSRC.glob("*.h")) + list(INCLUDE.glob("*.h"))
    newest_header = max((h.stat().st_mtime for h in headers), default=0.0)
    objs = []
    changed = force or not OUT.exists()
    for src in sorted(CSRC.glob("*.cu")):
        obj = OBJ / (src.stem + ".o")
        objs.append(obj)
        if (not force and obj.exists() and obj.stat().st_mtime >= src.stat().st_mtime
                and obj.stat().st_mtime >= newest_header):
            continue
        cmd = [nvcc(), *ARCH, *FLAGS, "-c", str(src), "-o", str(obj)]
        if verbose_ptxas:
            cmd[1:1] = ["-Xptxas", "-v"]
        print("[qik build]", " ".join(cmd[-4:]), flush=True)
        subprocess.run(cmd, check=True)
        changed = True
    if changed:
        cmd = [nvcc(), *ARCH, "-shared", "-cudart", "static", "-o", str(OUT), *map(str, objs)]
        print("[qik build] link", OUT.name, flush=True)
        subprocess.run(cmd, check=True)
    build_calls(force)
    return OUT


def build_calls(force: bool = False) -> Path:
    import sysconfig

    import torch
    src, header = CSRC / "calls.cpp", INCLUDE / "qik.h"
    made_for = f"Python {sys.version} ({sysconfig.get_config_var('SOABI')}), torch {torch.__version__} ({torch.version.git_version})"
    if (not force and CALLS.exists() and CALLS.stat().st_mtime >= max(src.stat().st_mtime, header.stat().st_mtime)
            and CALLS_MADE_FOR.exists() and CALLS_MADE_FOR.read_text() == made_for):
        return CALLS
    root = Path(torch.__file__).resolve().parent
    cuda = Path(nvcc()).resolve().parent.parent
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           "-I", str(INCLUDE), "-isystem", str(root / "include"), "-isystem", str(root / "include/torch/csrc/api/include"),
           "-isystem", sysconfig.get_paths()["include"], "-isystem", str(cuda / "include"), str(src), "-o", str(CALLS),
           "-L", str(root / "lib"), "-ltorch_python", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-lc10", "-lc10_cuda",
           "-L", str(OUT.parent), "-l:libqik.so", "-Wl,-rpath,$ORIGIN"]
    print("[qik build] g++", src.name, flush=True)
    CALLS_MADE_FOR.unlink(missing_ok=True)
    subprocess.run(cmd, check=True)
    OBJ.mkdir(parents=True, exist_ok=True)
    CALLS_MADE_FOR.write_text(made_for)
    return CALLS


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose-ptxas", action="store_true")
    a = ap.parse_args()
    print(build(a.force, a.verbose_ptxas))
    sys.exit(0)
