"""Build the B200 ConvRot library (libconvrot_b200.so) with nvcc for sm_100a.

Counterpart of the reference's hipcc build (_int4/build.py:73-86): one nvcc
call on the package's CUDA sources, output next to this file, and one g++ call for
the Python binding of the MX4 entries, which links against it. It is run by
``__graft_entry__.build()`` and, when a file is missing, once by the loaders.
"""
from __future__ import annotations

import glob
import hashlib
import os
import shutil
import subprocess
import sys

_HERE = os.path.dirname(os.path.abspath(__file__))
_CSRC = os.path.join(os.path.dirname(_HERE), "csrc")
SOURCES = ["convrot_b200.cu", "noalloc.cu", "mx4.cu", "rope.cu", "mx4_tree.cu", "rms_linear.cu"]
HEADERS = ["sm100_ptx.cuh", "gemm_pair.cuh", "gemm_a8t.cuh", "lora_down.cuh", "linear_api.cuh", "hadamard.cuh",
           "host_launch.cuh", "mx4_common.cuh", "mx4_unit.cuh", "mx4_quant.cuh", "mx4_gemm.cuh", "mx4_few.cuh", "mx4_cache.cuh", "mx4_attn.cuh",
           "mx4_host.cuh", "mx4_attn_host.cuh", "rope.cuh", "mx4_cache_rope.cuh", "mx4_tree.cuh", "rms_quant.cuh"]
ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]


def lib_name() -> str:
    return "libconvrot_b200.so"


def lib_path() -> str:
    return os.path.join(_HERE, lib_name())


def src_paths() -> list[str]:
    return [os.path.join(_CSRC, s) for s in SOURCES]


def is_stale() -> bool:
    """True when the library is missing or older than any CUDA source."""
    out = lib_path()
    if not os.path.exists(out):
        return True
    newest = max(os.path.getmtime(p) for p in src_paths() + [os.path.join(_CSRC, h) for h in HEADERS])
    return newest > os.path.getmtime(out)


def binding_sources() -> list[str]:
    return [os.path.join(_CSRC, "mx4_binding.cpp"),
            os.path.join(os.path.dirname(os.path.dirname(_HERE)), "include", "convrot_b200.h")]


def binding_path() -> str:
    """The binding's file, named after its sources and the torch and Python it is built for:
    one that does not fit is not found."""
    import torch
    key = hashlib.sha1(f"{torch.__version__} {sys.implementation.cache_tag}".encode())
    for path in binding_sources():
        with open(path, "rb") as f:
            key.update(f.read())
    return os.path.join(_HERE, f"_mx4_binding_{key.hexdigest()[:12]}.so")


def find_nvcc() -> str | None:
    cand = shutil.which("nvcc")
    if cand:
        return cand
    home = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    p = os.path.join(home, "bin", "nvcc")
    return p if os.path.exists(p) else None


def build(verbose: bool = False) -> str:
    nvcc = find_nvcc()
    if not nvcc:
        raise RuntimeError("nvcc not found; cannot build libconvrot_b200.so")
    out = lib_path()
    tmp = f"{out}.{os.getpid()}.tmp"
    cmd = [nvcc, *ARCH_FLAGS, "-O3", "-lineinfo", "-std=c++17", "-shared", "--threads", "0",
           "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
           "-o", tmp, *src_paths()]
    if verbose:
        print("building:", " ".join(cmd))
    cp = subprocess.run(cmd, capture_output=True, text=True)
    if cp.returncode != 0 or not os.path.exists(tmp):
        raise RuntimeError(f"nvcc build failed:\n{cp.stderr}")
    os.replace(tmp, out)
    return out


def build_binding(verbose: bool = False) -> str:
    """The Python module of the MX4 entries (needs the built library and torch's headers)."""
    import sysconfig

    import torch
    root = os.path.dirname(torch.__file__)
    home = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    out = binding_path()
    tmp = f"{out}.{os.getpid()}.tmp"
    include = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
               os.path.join(home, "include"), sysconfig.get_paths()["include"],
               os.path.join(os.path.dirname(os.path.dirname(_HERE)), "include")]
    cmd = [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *[f"-I{d}" for d in include],
           binding_sources()[0], "-o", tmp, f"-L{os.path.join(root, 'lib')}", f"-L{_HERE}",
           "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda", f"-l:{lib_name()}", "-Wl,-rpath,$ORIGIN"]
    if verbose:
        print("building:", " ".join(cmd))
    cp = subprocess.run(cmd, capture_output=True, text=True)
    if cp.returncode != 0 or not os.path.exists(tmp):
        raise RuntimeError(f"the binding's build failed:\n{cp.stderr}")
    os.replace(tmp, out)
    for old in glob.glob(os.path.join(os.path.dirname(out), "_mx4_binding*.so")):
        if old != out:
            os.remove(old)
    return out


if __name__ == "__main__":
    print("built:", build(verbose=True))
    print("built:", build_binding(verbose=True))
