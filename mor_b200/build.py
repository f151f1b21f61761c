"""In-tree build of the three native artefacts of mor_b200.

``libmor_b200.so``     the CUDA kernels behind the C ABI of ``include/mor_b200.h``
                       (nvcc, sm_100a only, no torch headers; a few seconds).
``libmor_b200_mx.so``  the operators on microscaled operands, behind ``include/mor_b200_mx.h``.
``_C.*.so``            the PyTorch shim that registers ``torch.ops.mor.*`` and forwards
                       to the C ABIs (g++ against the torch headers; about a minute).

All land next to this file so that they travel with the source tree; nothing is
installed into site-packages.  nvcc cross-compiles without a GPU.
"""
from __future__ import annotations

import os
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
BUILD = os.path.join(HERE, "build")
LIB = os.path.join(HERE, "libmor_b200.so")
CU_SOURCES = ["fq_elementwise.cu", "fq_reduce.cu", "fq_scaling.cu", "fq_block.cu", "fq_group.cu", "fq_resident.cu", "p2p.cu", "api.cu"]
MX_LIB = os.path.join(HERE, "libmor_b200_mx.so")
MX_SOURCES = ["mx_quant.cu", "mx_matmul.cu", "mx_grad.cu", "mx_api.cu"]
NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
              "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden"]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", "nvcc"):
        if cand and (os.path.isabs(cand) and os.path.exists(cand) or not os.path.isabs(cand)):
            return cand
    return "nvcc"


def _newer(target: str, deps) -> bool:
    if not os.path.exists(target):
        return False
    t = os.path.getmtime(target)
    return all(os.path.getmtime(d) <= t for d in deps)


def _headers():
    hs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    hs += [os.path.join(os.path.dirname(HERE), "include", f) for f in ("mor_b200.h", "mor_b200_mx.h")]
    return hs


def shim_path() -> str:
    return os.path.join(HERE, "_C" + (sysconfig.get_config_var("EXT_SUFFIX") or ".so"))


def build_library(force: bool = False, verbose: bool = False) -> str:
    """Compile the kernels into libmor_b200.so and libmor_b200_mx.so."""
    os.makedirs(BUILD, exist_ok=True)
    hdrs = _headers()

    def compile_one(src):
        s = os.path.join(CSRC, src)
        o = os.path.join(BUILD, src.replace(".cu", ".o"))
        if force or not _newer(o, [s] + hdrs):
            cmd = [_nvcc()] + NVCC_FLAGS + (["-Xptxas", "-v"] if verbose else []) + ["-c", s, "-o", o]
            r = subprocess.run(cmd, capture_output=True, text=True)
            if r.returncode != 0:
                raise RuntimeError(f"nvcc failed on {src}:\n{r.stdout}\n{r.stderr}")
            if verbose:
                sys.stderr.write(r.stderr)
        return o

    sources = CU_SOURCES + MX_SOURCES
    with ThreadPoolExecutor(max_workers=len(sources)) as ex:
        objs = dict(zip(sources, ex.map(compile_one, sources)))
    for lib, parts in ((LIB, CU_SOURCES), (MX_LIB, MX_SOURCES)):
        parts = [objs[p] for p in parts]
        if force or not _newer(lib, parts):
            cmd = [_nvcc(), "-shared", "-o", lib] + parts + ["-gencode", "arch=compute_100a,code=sm_100a", "-lcudart"]
            r = subprocess.run(cmd, capture_output=True, text=True)
            if r.returncode != 0:
                raise RuntimeError(f"link of {os.path.basename(lib)} failed:\n{r.stdout}\n{r.stderr}")
    return LIB


def build_extension(force: bool = False) -> str:
    """Compile csrc/torch_shim.cpp into mor_b200/_C.<abi>.so, linked against both libraries."""
    import torch
    from torch.utils import cpp_extension

    build_library(force=False)
    out = shim_path()
    src = os.path.join(CSRC, "torch_shim.cpp")
    if not force and _newer(out, [src, LIB, MX_LIB] + _headers()):
        return out
    tdir = os.path.dirname(torch.__file__)
    inc = [f"-I{p}" for p in cpp_extension.include_paths("cuda")] + [f"-I{sysconfig.get_paths()['include']}"]
    cxx = "/usr/bin/g++" if os.path.exists("/usr/bin/g++") else "g++"
    abi = int(torch._C._GLIBCXX_USE_CXX11_ABI)
    cmd = [cxx, "-O2", "-std=c++17", "-fPIC", "-shared", "-DTORCH_EXTENSION_NAME=_C", "-DTORCH_API_INCLUDE_EXTENSION_H",
           f"-D_GLIBCXX_USE_CXX11_ABI={abi}", *inc, src, "-o", out,
           f"-L{HERE}", "-lmor_b200", "-lmor_b200_mx", "-Wl,-rpath,$ORIGIN",
           f"-L{os.path.join(tdir, 'lib')}", f"-Wl,-rpath,{os.path.join(tdir, 'lib')}",
           "-lc10", "-lc10_cuda", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python",
           "-L/usr/local/cuda/lib64", "-lcudart"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed on torch_shim.cpp:\n{r.stdout}\n{r.stderr}")
    return out


def build_all(force: bool = False) -> None:
    build_library(force=force)
    build_extension(force=force)


if __name__ == "__main__":
    build_all(force="--force" in sys.argv)
    print(LIB)
    print(MX_LIB)
    print(shim_path())
