"""Build libk3moe.so (every sm_100a kernel + the C ABI) in-tree with nvcc."""
from __future__ import annotations

import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
SRC = os.path.join(HERE, "csrc", "capi.cu")
OUT = os.path.join(HERE, "libk3moe.so")
HEADER = os.path.join(HERE, "..", "include", "k3moe.h")
TORCH_SRC = os.path.join(HERE, "csrc", "torch_ops.cpp")
TORCH_OUT = os.path.join(HERE, "k3moe_torch.so")
TORCH_STAMP = os.path.join(HERE, "k3moe_torch.stamp")  # the torch and Python that k3moe_torch.so was built against
NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-lineinfo", "-std=c++17", "-shared",
              "-Xcompiler", "-fPIC", "-Xptxas", "-v"]


def sources():
    d = os.path.join(HERE, "csrc")
    return [os.path.join(d, f) for f in sorted(os.listdir(d)) if not f.endswith(".cpp")] + [HEADER]


def up_to_date() -> bool:
    if not os.path.exists(OUT):
        return False
    t = os.path.getmtime(OUT)
    return all(os.path.getmtime(s) <= t for s in sources())


CUBIN = os.path.join(HERE, "k3moe_module.cubin")


def build_cubin(nvcc: str) -> str:
    """The drop-in kernel module (csrc/module.cu: the extern "C" entries with the reference's names)."""
    cmd = [nvcc, "-cubin", "-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-lineinfo", "-std=c++17",
           os.path.join(HERE, "csrc", "module.cu"), "-o", CUBIN + ".tmp"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise RuntimeError("nvcc failed for k3moe_module.cubin")
    os.replace(CUBIN + ".tmp", CUBIN)
    return CUBIN


def torch_stamp() -> str:
    import torch

    return f"torch {torch.__version__}, {sysconfig.get_config_var('SOABI')}\n"


def torch_up_to_date() -> bool:
    """Newer than its sources, and built against this torch and Python (their binary interfaces change)."""
    if not os.path.exists(TORCH_OUT) or not os.path.exists(TORCH_STAMP):
        return False
    with open(TORCH_STAMP) as f:
        same = f.read() == torch_stamp()
    return same and all(os.path.getmtime(s) <= os.path.getmtime(TORCH_OUT) for s in (TORCH_SRC, HEADER))


def build_torch(force: bool = False) -> str:
    """The compiled torch side of the newer entries (csrc/torch_ops.cpp), linked to libk3moe.so beside it."""
    if not force and torch_up_to_date():
        return TORCH_OUT
    import torch
    from torch.utils import cpp_extension

    lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    inc = [*cpp_extension.include_paths(), os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "include"),
           sysconfig.get_paths()["include"]]
    abi = int(torch._C._GLIBCXX_USE_CXX11_ABI)
    cmd = ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden", f"-D_GLIBCXX_USE_CXX11_ABI={abi}",
           *(f for d in inc for f in ("-isystem", d)), TORCH_SRC, "-o", TORCH_OUT + ".tmp",
           "-L" + HERE, "-l:libk3moe.so", "-L" + lib, "-ltorch_python", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-lc10", "-lc10_cuda", "-Wl,-rpath,$ORIGIN"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise RuntimeError("g++ failed for k3moe_torch.so")
    os.replace(TORCH_OUT + ".tmp", TORCH_OUT)
    with open(TORCH_STAMP, "w") as f:
        f.write(torch_stamp())
    return TORCH_OUT


def build(force: bool = False, verbose: bool = False) -> str:
    out = build_library(force, verbose)
    build_torch(force)
    return out


def build_library(force: bool = False, verbose: bool = False) -> str:
    nvcc = os.environ.get("NVCC", "nvcc")
    if not force and up_to_date():
        if not os.path.exists(CUBIN) or os.path.getmtime(CUBIN) < os.path.getmtime(OUT):
            build_cubin(nvcc)
        return OUT
    build_cubin(nvcc)
    cmd = [nvcc, *NVCC_FLAGS, SRC, "-o", OUT + ".tmp"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise RuntimeError("nvcc failed for libk3moe.so")
    os.replace(OUT + ".tmp", OUT)
    with open(os.path.join(HERE, "ptxas.txt"), "w") as f:
        f.write(r.stderr)
    if verbose:
        sys.stderr.write(r.stderr)
    return OUT


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
