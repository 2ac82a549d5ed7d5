"""Build libemberglass_cuda.so in-tree for sm_100a.

nvcc compiles the CUDA sources for `-gencode arch=compute_100a,code=sm_100a`
(cross-compiles without a GPU); g++ compiles the host quantiser/generator
with -ffp-contract=off so its arithmetic matches the reference's JS doubles
operation by operation.  Objects go to _build/ beside this file, the shared
library next to the package so it ships with the source tree, and beside it the
Python binding of the ops on torch tensors (_ops, against the installed torch;
left out where there is none: the library itself does not need it).
"""
from __future__ import annotations

import importlib.metadata
import importlib.util
import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
BUILD = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libemberglass_cuda.so")
OPS = os.path.join(HERE, "_ops" + sysconfig.get_config_var("EXT_SUFFIX"))  # one for each Python
OPS_TORCH = os.path.join(BUILD, "_ops.torch")  # the torch that it was built against
INCLUDE = os.path.join(ROOT, "include")

NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
CXX = "/usr/bin/g++"
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVFLAGS = ["-O3", "-std=c++17", "-lineinfo", "--expt-relaxed-constexpr", "-Xcompiler", "-fPIC",
           "-ccbin", CXX, "-I", INCLUDE, "-I", CSRC]
CXXFLAGS = ["-O3", "-std=c++17", "-fPIC", "-fopenmp", "-ffp-contract=off", "-march=x86-64-v3",
            "-I", INCLUDE, "-I", CSRC, "-I", "/usr/local/cuda/include"]

CU = ["eg_kernels.cu", "eg_batch.cu", "eg_tc.cu", "eg_prefill.cu", "eg_fused.cu", "eg_runtime.cu", "eg_noalloc.cu",
      "eg_paged.cu", "eg_sample.cu"]
CPP = ["eg_host.cpp", "eg_safetensors.cpp"]
HEADERS = ["eg_common.cuh", "eg_device.cuh", "eg_stream.cuh", "eg_tc.cuh", "eg_kernels.h", "eg_batch.h", "eg_prefill.h", "eg_fused.h",
           "eg_host.h"]


def _stale(target: str, deps: list[str]) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def _run(cmd: list[str], verbose: bool):
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)


def build(verbose: bool = False, extra_nvflags: list[str] | None = None) -> str:
    os.makedirs(BUILD, exist_ok=True)
    hdrs = [os.path.join(CSRC, h) for h in HEADERS] + [os.path.join(INCLUDE, "emberglass.h")]
    objs = []
    for src in CU:
        s = os.path.join(CSRC, src)
        o = os.path.join(BUILD, src + ".o")
        if _stale(o, [s, __file__] + hdrs):
            _run([NVCC, *ARCH, *NVFLAGS, *(extra_nvflags or []), "-c", s, "-o", o], verbose)
        objs.append(o)
    for src in CPP:
        s = os.path.join(CSRC, src)
        o = os.path.join(BUILD, src + ".o")
        if _stale(o, [s, __file__] + hdrs):
            _run([CXX, *CXXFLAGS, "-c", s, "-o", o], verbose)
        objs.append(o)
    if _stale(LIB, objs):
        _run([NVCC, *ARCH, "-shared", "-ccbin", CXX, "-o", LIB, *objs, "-Xcompiler", "-fopenmp",
              "-lgomp", "-Xlinker", "--no-undefined"], verbose)
    build_ops(verbose)
    return LIB


def _torch() -> str | None:
    """The installed torch, by version and place (not imported); None without one."""
    spec = importlib.util.find_spec("torch")
    return f"{importlib.metadata.version('torch')} {spec.origin}" if spec else None


def build_ops(verbose: bool = False) -> str | None:
    """The binding: csrc/eg_torch.cpp against torch's headers and libraries and the
    library above (found beside it at run time).  Built again for another torch."""
    src = os.path.join(CSRC, "eg_torch.cpp")
    have = _torch()
    if have is None:
        print("torch is not installed: the library is built without the Python binding of its paged serving ops",
              file=sys.stderr)
        return None
    built = open(OPS_TORCH).read() if os.path.exists(OPS_TORCH) else ""
    if built != have or _stale(OPS, [src, __file__, os.path.join(INCLUDE, "emberglass.h")]):
        import torch
        from torch.utils.cpp_extension import include_paths, library_paths
        inc = [f for p in include_paths() + ["/usr/local/cuda/include"] for f in ("-isystem", p)]
        libs = [f for p in library_paths() for f in ("-L", p, f"-Wl,-rpath,{p}")]
        _run([CXX, "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
              "-I", INCLUDE, *inc, "-isystem", sysconfig.get_paths()["include"], src, "-o", OPS, "-L", HERE,
              "-l:" + os.path.basename(LIB), *libs, "-lc10",
              "-lc10_cuda", "-ltorch_cpu", "-ltorch_python", "-Wl,-rpath,$ORIGIN"], verbose)
        with open(OPS_TORCH, "w") as f:
            f.write(have)
    return OPS


if __name__ == "__main__":
    build(verbose="-v" in sys.argv)
    print(LIB)
