"""Build the sm_100a kernel library in-tree.

    python llama-efficient-inference_b200/build.py [--force] [-v]

Compiles csrc/*.cu with nvcc for sm_100a (cross-compiles without a GPU) and
links lib/libllama_int4_b200.so -- a plain C-ABI shared library (see
include/llama_int4_b200.h) with the CUDA runtime linked statically, so it
loads with or without torch in the process -- and compiles csrc/li4_torch.cpp
against this interpreter's torch into lib/li4_torch.so, the binding of the
paged-cache entry points to torch tensors (it links the C-ABI library).  Without
g++, torch or their headers the library is built alone, and llama.paged raises
when it is used.
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import glob
import os
import shutil
import subprocess
import sys
import sysconfig

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(PKG_DIR)
CSRC = os.path.join(PKG_DIR, "csrc")
BUILD_DIR = os.path.join(PKG_DIR, "_build")
LIB_DIR = os.path.join(PKG_DIR, "lib")
LIB_PATH = os.path.join(LIB_DIR, "libllama_int4_b200.so")
EXT_PATH = os.path.join(LIB_DIR, "li4_torch.so")

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ARCH_FLAGS + ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-Xcompiler", "-Wall",
                           f"-I{os.path.join(REPO, 'include')}"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found (set NVCC or put CUDA's bin/ on PATH)")


def sources() -> list[str]:
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def _deps() -> list[str]:
    return sources() + glob.glob(os.path.join(CSRC, "*.cpp")) + glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(CSRC, "*.h")) + \
        glob.glob(os.path.join(REPO, "include", "*.h")) + [os.path.abspath(__file__)]


def up_to_date() -> bool:
    if not os.path.exists(LIB_PATH):
        return False
    t = os.path.getmtime(LIB_PATH)
    if os.path.exists(EXT_PATH):
        t = min(t, os.path.getmtime(EXT_PATH))
    elif not why_no_binding():
        return False
    return all(os.path.getmtime(d) <= t for d in _deps())


def why_no_binding() -> str:
    """What the binding cannot be built without, "" if it can."""
    if shutil.which("g++") is None:
        return "no g++"
    try:
        import torch
    except ImportError as e:
        return f"no torch ({e})"
    headers = [os.path.join(os.path.dirname(torch.__file__), "include", "ATen", "ATen.h"),
               os.path.join(sysconfig.get_paths()["include"], "Python.h")]
    missing = [h for h in headers if not os.path.exists(h)]
    return f"no {missing[0]}" if missing else ""


def compile_binding(verbose: bool) -> str:
    """csrc/li4_torch.cpp as an object file (host code only)."""
    import torch

    root = os.path.dirname(torch.__file__)
    obj = os.path.join(BUILD_DIR, "li4_torch.o")
    cuda = os.path.join(os.path.dirname(os.path.dirname(nvcc())), "include")
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-Wall", "-fvisibility=hidden", f"-I{os.path.join(REPO, 'include')}",
           f"-I{root}/include", f"-I{root}/include/torch/csrc/api/include", f"-I{sysconfig.get_paths()['include']}",
           f"-I{cuda}", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", "-c",
           os.path.join(CSRC, "li4_torch.cpp"), "-o", obj]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed on li4_torch.cpp:\n{r.stdout}\n{r.stderr}")
    return obj


def link_binding(obj: str, verbose: bool) -> None:
    import torch

    tmp = EXT_PATH + ".tmp"
    cmd = ["g++", "-shared", "-o", tmp, obj, f"-L{LIB_DIR}", "-l:libllama_int4_b200.so", "-Wl,-rpath,$ORIGIN",
           f"-L{os.path.join(os.path.dirname(torch.__file__), 'lib')}", "-lc10", "-lc10_cuda", "-ltorch_cpu",
           "-ltorch_cuda", "-ltorch_python"]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, EXT_PATH)


def build(force: bool = False, verbose: bool = False, ptxas_info: bool = False) -> str:
    """Compile every .cu in csrc/ and link the library; returns its path."""
    if not force and not ptxas_info and up_to_date():
        return LIB_PATH
    os.makedirs(BUILD_DIR, exist_ok=True)
    os.makedirs(LIB_DIR, exist_ok=True)
    cc = nvcc()
    extra = ["-Xptxas", "-v"] if ptxas_info else []

    shared = [d for d in _deps() if not d.endswith((".cu", ".cpp"))]

    def compile_one(src: str) -> str:
        obj = os.path.join(BUILD_DIR, os.path.basename(src)[:-3] + ".o")
        if not force and not ptxas_info and os.path.exists(obj) and \
                all(os.path.getmtime(d) <= os.path.getmtime(obj) for d in [src] + shared):
            return obj  # newer than its source, every header and this file
        cmd = [cc] + NVCC_FLAGS + extra + ["-c", src, "-o", obj]
        if verbose:
            print(" ".join(cmd), flush=True)
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed on {os.path.basename(src)}:\n{r.stdout}\n{r.stderr}")
        if ptxas_info or verbose:
            sys.stdout.write(r.stderr)
        return obj

    missing = why_no_binding()
    with cf.ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
        binding = None if missing else ex.submit(compile_binding, verbose)
        objs = list(ex.map(compile_one, sources()))
    tmp = LIB_PATH + ".tmp"
    cmd = [cc] + ARCH_FLAGS + ["-shared", "-o", tmp] + objs
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, LIB_PATH)
    if binding is None:
        print(f"build.py: li4_torch.so is not built ({missing}); llama.paged needs it", file=sys.stderr)
        if os.path.exists(EXT_PATH):
            os.remove(EXT_PATH)  # (made for another build of the library)
    else:
        link_binding(binding.result(), verbose)
    return LIB_PATH


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("-v", "--verbose", action="store_true")
    ap.add_argument("--ptxas-info", action="store_true", help="print registers / spills / smem per kernel")
    a = ap.parse_args()
    print(build(force=a.force, verbose=a.verbose, ptxas_info=a.ptxas_info))
