"""Builds ``_lib/libflasheq.so`` from ``csrc/*.hip`` with hipcc for gfx950.

Every translation unit is compiled to an object under ``_build/`` (git-ignored)
and linked into one shared library with a plain C ABI (``include/flasheq.h``).
Packed-FP32 instructions are disabled for all device code.

``_lib/flasheq_torch.so`` is the PyTorch module over that library
(``csrc/torch_nodes.cpp``): host code only, compiled with g++ against the
installed PyTorch's headers.
"""
from __future__ import annotations

import concurrent.futures as cf
import glob
import importlib.util
import os
import subprocess
import sys
import sysconfig

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG_DIR)                      # flash-eq_amd/
REPO = os.path.dirname(ROOT)
CSRC = os.path.join(ROOT, "csrc")
INCLUDE = os.path.join(REPO, "include")
BUILD_DIR = os.path.join(ROOT, "_build")
LIB_DIR = os.path.join(PKG_DIR, "_lib")
LIB_PATH = os.path.join(LIB_DIR, "libflasheq.so")
NODES_PATH = os.path.join(LIB_DIR, "flasheq_torch.so")
ARCH = os.environ.get("FEQ_OFFLOAD_ARCH", "gfx950")

HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
CFLAGS = [
    f"--offload-arch={ARCH}", "-O3", "-fPIC", "-std=c++17",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wall", "-Wno-unused-function",
    f"-I{INCLUDE}", f"-I{CSRC}",
]


def _compile(src: str) -> str:
    obj = os.path.join(BUILD_DIR, os.path.basename(src).replace(".hip", ".o"))
    cmd = [HIPCC, *CFLAGS, "-c", src, "-o", obj]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src}:\n{res.stdout}\n{res.stderr}")
    return obj


def _compile_nodes() -> str:
    torch_dir = importlib.util.find_spec("torch").submodule_search_locations[0]
    obj = os.path.join(BUILD_DIR, "torch_nodes.o")
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-fPIC", "-std=c++17", "-Wall", "-Wno-sign-compare",
           "-D__HIP_PLATFORM_AMD__", "-DUSE_ROCM", f"-isystem{torch_dir}/include",
           f"-isystem{torch_dir}/include/torch/csrc/api/include", "-isystem/opt/rocm/include",
           f"-I{sysconfig.get_paths()['include']}", f"-I{INCLUDE}", "-c",
           os.path.join(CSRC, "torch_nodes.cpp"), "-o", obj]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"compiling torch_nodes.cpp failed:\n{res.stdout}\n{res.stderr}")
    return obj


def _link_nodes(obj: str) -> None:
    torch_dir = importlib.util.find_spec("torch").submodule_search_locations[0]
    tmp = NODES_PATH + ".tmp"
    cmd = [os.environ.get("CXX", "g++"), "-shared", "-o", tmp, obj, f"-L{torch_dir}/lib", "-ltorch_python", "-ltorch",
           "-ltorch_cpu", "-lc10", "-lc10_hip", f"-L{LIB_DIR}", "-l:libflasheq.so", "-Wl,-rpath,$ORIGIN"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"linking flasheq_torch.so failed:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, NODES_PATH)


def build(verbose: bool = False) -> str:
    """Compile every source and link the shared library and the PyTorch module; returns the library's path.

    The library is in place before anything of the module can fail, and is built alone where there is
    no PyTorch.  A module that could not be built leaves none of an earlier library behind."""
    os.makedirs(BUILD_DIR, exist_ok=True)
    os.makedirs(LIB_DIR, exist_ok=True)
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.hip")))
    with cf.ThreadPoolExecutor(max_workers=min(8, len(srcs) + 1)) as ex:
        nodes = ex.submit(_compile_nodes) if importlib.util.find_spec("torch") else None
        objs = list(ex.map(_compile, srcs))
    tmp = LIB_PATH + ".tmp"
    cmd = [HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", tmp, *objs,
           "-L/opt/rocm/lib", "-Wl,-rpath,/opt/rocm/lib"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, LIB_PATH)
    if os.path.exists(NODES_PATH):
        os.remove(NODES_PATH)
    if nodes is not None:
        _link_nodes(nodes.result())
    if verbose:
        built = f"{LIB_PATH} and {NODES_PATH}" if nodes is not None else f"{LIB_PATH} (no PyTorch: no {NODES_PATH})"
        print(f"built {built}", file=sys.stderr)
    return LIB_PATH


if __name__ == "__main__":
    build(verbose=True)
