"""Builds the sm_100a shared library (batch_topk_b200/lib/libbatch_topk_b200.so) with nvcc, and the
tensor-level Python module over it (batch_topk_b200/_tensors.so) with g++.

Run as ``python -m batch_topk_b200.build``.  The library is built in-tree so that it
travels with the repository; nothing is installed into site-packages.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(HERE)
SRC = os.path.join(HERE, "csrc", "batch_topk.cu")
GEN_SRC = os.path.join(HERE, "csrc", "gen.cu")  # device-side input generation
LOGITS_SRC = os.path.join(HERE, "csrc", "bt_logits.cu")  # logits producer, fused top-k epilogue
SAMPLE_SRC = os.path.join(HERE, "csrc", "bt_sample.cu")  # sampling
EXPERTS_SRC = os.path.join(HERE, "csrc", "bt_experts.cu")  # routing and experts' rows
HEADERS = [os.path.join(HERE, "csrc", f) for f in ("bt_device.cuh", "bt_kernels.cuh", "bt_body.cuh",
                                                   "bt_elem.cuh", "bt_small.cuh",
                                                   "bt_large.cuh", "bt_common.cuh", "bt_f32.cuh",
                                                   "bt_values.cuh")] + [
    os.path.join(REPO, "include", "batch_topk_b200.h"),
    os.path.join(REPO, "include", "batch_topk_b200_gen.h"),
]
SOURCES = [SRC, GEN_SRC, LOGITS_SRC, SAMPLE_SRC, EXPERTS_SRC]
LIB_DIR = os.path.join(HERE, "lib")
LIB = os.path.join(LIB_DIR, "libbatch_topk_b200.so")
TENSORS_SRC = os.path.join(HERE, "csrc", "tensors.cpp")  # needs torch's headers
TENSORS = os.path.join(HERE, "_tensors.so")
TENSORS_STAMP = os.path.join(HERE, "_build", "torch")  # the torch that TENSORS was built for

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC", "-shared",
]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: set NVCC or put the CUDA toolkit on PATH")


def up_to_date() -> bool:
    if not os.path.exists(LIB):
        return False
    t = os.path.getmtime(LIB)
    return all(os.path.getmtime(p) <= t for p in [*SOURCES, *HEADERS])


def torch_dir() -> str | None:
    """Where torch is installed, without importing it."""
    from importlib.util import find_spec

    spec = find_spec("torch")
    return os.path.dirname(spec.origin) if spec else None


def torch_version() -> str:
    with open(os.path.join(torch_dir(), "version.py")) as f:
        return f.read()


def tensors_up_to_date() -> bool:
    if not os.path.exists(TENSORS) or not os.path.exists(TENSORS_STAMP):
        return False
    with open(TENSORS_STAMP) as f:
        if f.read() != torch_version():
            return False
    t = os.path.getmtime(TENSORS)
    return all(os.path.getmtime(p) <= t for p in [TENSORS_SRC, *HEADERS])


def _run(cmd: list[str], verbose: bool = False) -> None:
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"{cmd[0]} failed ({res.returncode}):\n{res.stdout}\n{res.stderr}")
    if verbose:
        sys.stderr.write(res.stderr)


def build_tensors(force: bool = False) -> str:
    """The Python module, which needs torch; LIB has to be there (it is linked, and found beside the
    module)."""
    if not force and tensors_up_to_date():
        return TENSORS
    import sysconfig

    torch = torch_dir()
    cuda = os.path.dirname(os.path.dirname(nvcc()))
    tmp = TENSORS + ".tmp"
    # the g++ that nvcc compiles host code with: another one may bring its own C++ library
    _run(["g++", "-O2", "-std=c++17", "-fPIC", "-shared",
          "-D_GLIBCXX_USE_CXX11_ABI=1",
          "-I" + os.path.join(torch, "include"),
          "-I" + os.path.join(torch, "include", "torch", "csrc", "api", "include"),
          "-I" + sysconfig.get_paths()["include"], "-I" + os.path.join(cuda, "include"),
          TENSORS_SRC, "-o", tmp,
          "-L" + os.path.join(torch, "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu",
          "-ltorch_python", "-L" + LIB_DIR, "-lbatch_topk_b200", "-Wl,-rpath,$ORIGIN/lib"])
    os.makedirs(os.path.dirname(TENSORS_STAMP), exist_ok=True)
    with open(TENSORS_STAMP, "w") as f:
        f.write(torch_version())
    os.replace(tmp, TENSORS)
    return TENSORS


def build(force: bool = False, verbose: bool = False) -> str:
    if force or not up_to_date():
        os.makedirs(LIB_DIR, exist_ok=True)
        tmp = LIB + ".tmp"
        cmd = [nvcc(), *NVCC_FLAGS, "--threads", "0", "-o", tmp, *SOURCES]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
        _run(cmd, verbose)
        os.replace(tmp, LIB)
    if torch_dir():  # C callers of the library need no torch
        build_tensors(force)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
