"""Build the CUDA extension in-tree: unum_ops_b200/lib/libunum_ops_b200.so, and its
binding to torch's tensors, unum_ops_b200/lib/_binding.<Python ABI>-torch<version>.so.

nvcc compiles every ``csrc/*.cu`` for sm_100a only (``-gencode
arch=compute_100a,code=sm_100a``) and links one shared library exposing the C
ABI declared in ``include/unum_ops_b200.h``.  The CUDA runtime is linked as a
shared library so the extension shares the runtime state (current device,
streams) of the PyTorch process that loads it.  ``csrc/binding.cpp`` (the native
half of ``paged_cache``) is host code against torch's headers, linked to that library; it
fits the torch and the Python that it was compiled for, and its file is named after them.

Usage: ``python -m unum_ops_b200._build [--force]``.
"""
from __future__ import annotations

import concurrent.futures as cf
import os
import shutil
import subprocess
import sys
import sysconfig

import torch

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT_DIR = os.path.join(HERE, "lib")
LIB = os.path.join(OUT_DIR, "libunum_ops_b200.so")
ROOT = os.path.dirname(HERE)

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-Xcompiler", "-O3",
    "-Xptxas", "-v", "--expt-relaxed-constexpr",
    "-I" + os.path.join(ROOT, "include"),
]


def binding_path() -> str:
    return os.path.join(OUT_DIR, f"_binding.{sysconfig.get_config_var('SOABI')}-torch{torch.__version__}.so")


def _nvcc() -> str:
    cand = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    return cand


def _sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cu"))


def _deps():
    return [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh", ".cpp"))] + [
        os.path.join(ROOT, "include", "unum_ops_b200.h")]


def needs_build() -> bool:
    if not os.path.exists(LIB) or not os.path.exists(binding_path()):
        return True
    t = min(os.path.getmtime(LIB), os.path.getmtime(binding_path()))
    return any(os.path.getmtime(d) > t for d in _deps())


def _binding_command(src, out):
    from torch.utils import cpp_extension

    cxx = os.environ.get("CXX") or shutil.which("g++") or "c++"
    cuda = os.path.dirname(os.path.dirname(_nvcc()))
    inc = [*cpp_extension.include_paths(), sysconfig.get_paths()["include"], os.path.join(cuda, "include")]
    libs = cpp_extension.library_paths()
    return [cxx, "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *[f"-isystem{i}" for i in inc], src, "-o", out,
            *[f"-L{d}" for d in libs], "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda",
            "-L" + OUT_DIR, "-l:" + os.path.basename(LIB), "-Wl,-rpath,$ORIGIN"]


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and not needs_build():
        return LIB
    os.makedirs(OUT_DIR, exist_ok=True)
    obj_dir = os.path.join(OUT_DIR, "obj")
    os.makedirs(obj_dir, exist_ok=True)
    nvcc = _nvcc()

    def compile_one(src):
        obj = os.path.join(obj_dir, os.path.basename(src)[:-3] + ".o")
        cmd = [nvcc, *NVCC_FLAGS, "-c", src, "-o", obj]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed for {src}:\n{r.stderr}")
        return obj, r.stderr

    with cf.ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
        results = list(ex.map(compile_one, _sources()))
    if verbose:
        for _, log in results:
            sys.stderr.write(log)
    objs = [o for o, _ in results]
    tmp = LIB + ".tmp"
    cmd = [nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-shared", "-cudart", "shared",
           "-o", tmp, *objs]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stderr}")
    os.replace(tmp, LIB)
    tmp = binding_path() + ".tmp"
    r = subprocess.run(_binding_command(os.path.join(CSRC, "binding.cpp"), tmp), capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"binding failed:\n{r.stderr}")
    os.replace(tmp, binding_path())
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
