"""Build libruntimed_b200.so in-tree with nvcc for sm_100a.

    python -m runtimed_b200.build            # incremental
    python -m runtimed_b200.build --force    # rebuild everything

Each source compiles to an object under runtimed_b200/_build/ (git-ignored);
the shared library lands next to this file so it travels with the tree, and beside
it _rtd_torch.so, the binding that hands torch tensors to it (csrc/rtd_torch.cpp).
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
BUILD = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libruntimed_b200.so")
TORCH_LIB = os.path.join(HERE, "_rtd_torch.so")
INCLUDE = os.path.join(ROOT, "include")

SOURCES = ["rtd_api.cu", "rtd_gemv.cu", "rtd_gemm.cu", "rtd_gemm_ts.cu", "rtd_tp.cu", "rtd_model.cu", "rtd_kv4.cu", "rtd_kv4_wide.cu",
           "rtd_sample.cu", "rtd_dequant.cu", "rtd_repack.cpp"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found (set NVCC)")


def host_cxx() -> str:
    return "/usr/bin/g++" if os.path.exists("/usr/bin/g++") else "g++"


def _deps() -> list[str]:
    out = []
    for d in (CSRC, INCLUDE):
        for f in os.listdir(d):
            if f.endswith((".h", ".cuh", ".hpp")):
                out.append(os.path.join(d, f))
    return out


def _stale(target: str, inputs: list[str]) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(i) > t for i in inputs)


def compile_one(src: str, force: bool, verbose: bool) -> str:
    path = os.path.join(CSRC, src)
    obj = os.path.join(BUILD, src + ".o")
    if not force and not _stale(obj, [path] + _deps()):
        return obj
    cmd = [nvcc(), "-ccbin", host_cxx(), *ARCH, "-std=c++17", "-O3", "-lineinfo", "-Xcompiler", "-fPIC",
           "-Xcompiler", "-fvisibility=hidden", f"-I{CSRC}", f"-I{INCLUDE}", "-c", path, "-o", obj]
    if src.endswith(".cu"):
        cmd[1:1] = ["-Xptxas", "-v"] if verbose else []
    else:
        cmd += ["-x", "c++"]
    subprocess.run(cmd, check=True)
    return obj


def build(force: bool = False, verbose: bool = False) -> str:
    os.makedirs(BUILD, exist_ok=True)
    with cf.ThreadPoolExecutor(max_workers=len(SOURCES)) as ex:
        objs = list(ex.map(lambda s: compile_one(s, force, verbose), SOURCES))
    if force or _stale(LIB, objs):
        cmd = [nvcc(), "-ccbin", host_cxx(), *ARCH, "-shared", "-o", LIB, *objs, "-cudart", "static"]
        subprocess.run(cmd, check=True)
    torch_binding(force)
    return LIB


def torch_binding(force: bool = False) -> str:
    """_rtd_torch.so next to the library: torch tensors into the C ABI (csrc/rtd_torch.cpp)."""
    import sysconfig

    src = os.path.join(CSRC, "rtd_torch.cpp")
    if not force and not _stale(TORCH_LIB, [src, os.path.join(INCLUDE, "rtd.h")]):
        return TORCH_LIB
    import torch
    from torch.utils import cpp_extension as ext

    inc = [f"-isystem{d}" for d in ext.include_paths() + [sysconfig.get_paths()["include"], "/usr/local/cuda/include"]]
    lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    cmd = [host_cxx(), "-std=c++17", "-O2", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f"-I{INCLUDE}", *inc, src, "-o", TORCH_LIB,
           f"-L{HERE}", "-l:libruntimed_b200.so", f"-L{lib}", "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda",
           "-Wl,-rpath,$ORIGIN"]
    subprocess.run(cmd, check=True)
    return TORCH_LIB


def main() -> int:
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true", help="print ptxas register/smem usage")
    args = ap.parse_args()
    print(build(args.force, args.verbose))
    return 0


if __name__ == "__main__":
    sys.exit(main())
