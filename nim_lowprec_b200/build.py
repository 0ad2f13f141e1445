"""Build liblowprec_cuda.so in-tree with nvcc for sm_100a.

    python nim_lowprec_b200/build.py [--force] [-v]

(Run it by path: importing the package itself loads the built library.)

Every .cu under csrc/ is compiled for `sm_100a` only (the library uses
tcgen05/TMA-era PTX: bulk copies, mbarrier waits, f32x2 arithmetic) and
linked into one shared object next to this file, with the CUDA runtime linked
statically.  Where torch is installed, csrc/torch_binding.cpp becomes the
CPython module _torch_binding beside it (the entry points of the cache and the experts for
torch tensors).  The result travels with the repository snapshot; nothing is
installed into site-packages.
"""
from __future__ import annotations

import glob
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(ROOT, "include")
OUT = os.path.join(HERE, "liblowprec_cuda.so")
OBJDIR = os.path.join(HERE, "_build")

NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
# -fmad=false: ptxas may otherwise contract a multiply feeding an add into one
# FMA even across the explicit mul.rn/add.rn f32x2 pairs of the bit-exact
# paths (measured on sm_100a); this is the device-side twin of the
# reference's -ffp-contract=off (simd/dequant.nim:36).
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-fmad=false", "-Xcompiler", "-fPIC", "-Xcompiler", "-Wall",
         "--expt-relaxed-constexpr", "-I", CSRC, "-I", INCLUDE]


BINDING = os.path.join(HERE, "_torch_binding.so")


def build_binding(force: bool = False) -> None:
    """_torch_binding.so against the installed torch; skipped without torch, and with a torch
    that has no CUDA.  A binding for another torch or Python is built again."""
    try:
        import torch
        from torch.utils import cpp_extension
    except ImportError:
        return
    if torch.version.cuda is None:
        print("_torch_binding: skipped, the installed torch is without CUDA")
        return
    src = os.path.join(CSRC, "torch_binding.cpp")
    stamp = os.path.join(OBJDIR, "torch_binding.for")
    this = f"torch {torch.__version__}, Python {sys.version}"
    known = open(stamp).read() if os.path.exists(stamp) else ""
    if not force and known == this and not _stale(
            BINDING, [src, OUT, os.path.join(INCLUDE, "lowprec_cuda.h")]):
        return
    import sysconfig
    cuda = os.path.dirname(os.path.dirname(NVCC))
    inc = [INCLUDE, os.path.join(cuda, "include"), sysconfig.get_paths()["include"],
           *cpp_extension.include_paths()]
    lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    cmd = ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-Wall",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *(f"-isystem{i}" for i in inc), src, "-o", BINDING, f"-L{HERE}", f"-L{lib}",
           "-l:" + os.path.basename(OUT), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python",
           "-Wl,-rpath,$ORIGIN"]
    subprocess.run(cmd, check=True)
    with open(stamp, "w") as f:
        f.write(this)


def sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def _stale(obj: str, deps) -> bool:
    if not os.path.exists(obj):
        return True
    t = os.path.getmtime(obj)
    return any(os.path.getmtime(d) > t for d in deps)


def build(force: bool = False, verbose: bool = False) -> str:
    os.makedirs(OBJDIR, exist_ok=True)
    headers = glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(CSRC, "*.h")) + \
        glob.glob(os.path.join(INCLUDE, "*.h"))
    objs = []
    for src in sources():
        obj = os.path.join(OBJDIR, os.path.basename(src)[:-3] + ".o")
        objs.append(obj)
        if force or _stale(obj, [src, *headers]):
            cmd = [NVCC, *ARCH, *FLAGS, "-c", src, "-o", obj]
            if verbose:
                cmd.insert(1, "-Xptxas=-v")
                print(" ".join(cmd), flush=True)
            subprocess.run(cmd, check=True)
    if force or _stale(OUT, objs):
        cmd = [NVCC, *ARCH, "-shared", "-o", OUT, *objs, "-ldl"]
        subprocess.run(cmd, check=True)
    build_binding(force)
    return OUT


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(OUT)
