"""Build libdsa_b200.so (all CUDA kernels of the package) for sm_100a with nvcc, and the Python
binding of its serving operators (csrc/binding.cpp) with the host compiler.

Both are built in-tree (next to this file) so they travel with the source tree;
there is no JIT cache.  Usage: ``python -m dsa_triton_ascend_b200.build``.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
LIB = os.path.join(PKG, "libdsa_b200.so")
BINDING = os.path.join(PKG, "_binding" + sysconfig.get_config_var("EXT_SUFFIX"))
SOURCES = ["capi.cu", "sfa_fwd.cu", "sfa_bwd.cu", "li.cu", "sli.cu", "dense.cu", "attn_paged.cu",
           "rotary.cu", "page_cache.cu"]
FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-std=c++17", "-lineinfo",
         "-Xcompiler", "-fPIC", "-shared", "--expt-relaxed-constexpr"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def _stale() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    deps = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f != "binding.cpp"] + [
        os.path.join(ROOT, "include", "dsa_b200.h")]
    return any(os.path.getmtime(d) > t for d in deps)


def _built_for(version: str) -> bool:
    """Whether the binding carries the stamp of this torch (csrc/binding.cpp)."""
    with open(BINDING, "rb") as f:
        return b"dsa binding for torch " + version.encode() + b"\0" in f.read()


def build_binding(force: bool = False) -> str:
    """The CPython module that calls the serving operators' C entries (see csrc/binding.cpp), built
    anew where its sources are newer or another torch is installed."""
    import torch
    src, header = os.path.join(CSRC, "binding.cpp"), os.path.join(ROOT, "include", "dsa_b200.h")
    if not force and os.path.exists(BINDING) and os.path.getmtime(BINDING) > max(
            os.path.getmtime(src), os.path.getmtime(header)) and _built_for(torch.__version__):
        return BINDING
    from torch.utils import cpp_extension
    inc = [ROOT + "/include", sysconfig.get_paths()["include"], *cpp_extension.include_paths(),
           os.path.join(os.path.dirname(os.path.dirname(nvcc())), "include")]
    libs = cpp_extension.library_paths()
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           f'-DDSA_TORCH_VERSION="{torch.__version__}"',
           *[f for i in inc for f in ("-isystem", i)], src, *[f"-L{p}" for p in libs],
           "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda", "-o", BINDING + ".tmp"]
    subprocess.run(cmd, check=True)
    os.replace(BINDING + ".tmp", BINDING)
    return BINDING


def build(force: bool = False, verbose: bool = False) -> str:
    build_binding(force)
    if not force and not _stale():
        return LIB
    cmd = [nvcc(), *FLAGS, "-I", os.path.join(ROOT, "include"), "-I", CSRC,
           *[os.path.join(CSRC, s) for s in SOURCES], "-o", LIB + ".tmp"]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
        print(" ".join(cmd))
    subprocess.run(cmd, check=True)
    os.replace(LIB + ".tmp", LIB)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
