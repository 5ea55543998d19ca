"""Builds libindecis_b200.so (the C-ABI library) in-tree with nvcc for sm_100a.

The library links the CUDA runtime statically and resolves the driver's
tensor-map encoder at run time, so it carries no dependency on torch or on
libcuda at link time. _torch_ops.so beside it is what Python calls the training
operators through, and links torch. Run ``python -m indecis_b200.build`` or call ``build()``.
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
LIB = os.path.join(HERE, "libindecis_b200.so")
TORCH_OPS = os.path.join(HERE, "_torch_ops.so")  # the training operators' calls from Python (torch_ops.cpp)
TORCH_OPS_STAMP = os.path.join(HERE, "_build", "torch_ops.txt")  # the torch and Python it was built for
SOURCES = ["libindecis_b200.cu", "adamw.cu", "spans.cpp", "batcher.cpp"]
HEADERS = ["common.cuh", "exactmath.cuh", "internal.h", "gemm_i8.cu", "gemm_persist.cu", "gemm_pair.cu", "rows_fast.cu", "rows.cu", "rows_ln.cu", "attention.cu", "attention_tc.cu", "attention_short.cu", "siglip.cu", "encoder_f32.cu", "capi.cu", "multi.cu", "siglip_capi.cu", "spans_device.cu", "noalloc.cu", "selfcheck.cu",
           "vocab_rows.cu", "vocab_gemm.cu", "vocab_capi.cu", "train.h", "layer_norm.cu", "gated_ff.cu", "train_capi.cu"]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
    "--expt-relaxed-constexpr",
    "-rdc=false",
]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", "nvcc"):
        if cand and (os.path.isabs(cand) and os.path.exists(cand) or not os.path.isabs(cand)):
            return cand
    return "nvcc"


def _stale(target: str, deps: list[str]) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def _torch_and_python() -> str:
    return f"torch {importlib.metadata.version('torch')}, {sysconfig.get_config_var('SOABI')}"


def _torch_ops_stale() -> bool:
    if _stale(TORCH_OPS, [os.path.join(CSRC, "torch_ops.cpp"), os.path.join(ROOT, "include", "indecis_b200.h")]):
        return True
    if not os.path.exists(TORCH_OPS_STAMP):
        return True
    with open(TORCH_OPS_STAMP) as f:
        return f.read() != _torch_and_python()


def _torch_ops_command() -> list[str]:
    torch = list(importlib.util.find_spec("torch").submodule_search_locations)[0]
    cuda = os.path.dirname(os.path.dirname(_nvcc())) if os.path.isabs(_nvcc()) else "/usr/local/cuda"
    inc = [os.path.join(torch, "include"), os.path.join(torch, "include", "torch", "csrc", "api", "include"),
           sysconfig.get_paths()["include"], os.path.join(cuda, "include")]
    return ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", *[f"-I{i}" for i in inc],
            os.path.join(CSRC, "torch_ops.cpp"), "-o", TORCH_OPS, f"-L{torch}/lib", "-ltorch_python", "-ltorch_cpu", "-lc10",
            "-lc10_cuda", f"-L{HERE}", "-l:libindecis_b200.so", "-Wl,-rpath,$ORIGIN"]


def build(verbose: bool = False, force: bool = False, extra: list[str] | None = None) -> str:
    """Compiles every .cu into objects, then links the shared library."""
    objdir = os.path.join(HERE, "_build")
    os.makedirs(objdir, exist_ok=True)
    inc = [os.path.join(ROOT, "include"), CSRC]
    header_paths = [os.path.join(CSRC, h) for h in HEADERS] + [os.path.join(ROOT, "include", "indecis_b200.h")]
    objs, running = [], []
    for src in SOURCES:
        sp = os.path.join(CSRC, src)
        op = os.path.join(objdir, os.path.splitext(src)[0] + ".o")
        objs.append(op)
        if force or _stale(op, [sp] + header_paths):
            cmd = [_nvcc(), *NVCC_FLAGS, *(extra or []), *[f"-I{i}" for i in inc], "-c", sp, "-o", op]
            if verbose:
                print(" ".join(cmd), flush=True)
            running.append((cmd, subprocess.Popen(cmd)))  # the objects side by side
    for cmd, p in [(cmd, p.wait()) for cmd, p in running]:
        if p:
            raise subprocess.CalledProcessError(p, cmd)
    if force or _stale(LIB, objs):
        cmd = [_nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-shared", "-Xcompiler", "-fPIC",
               "-o", LIB, *objs, "-cudart", "static", "-lpthread", "-ldl", "-lrt"]
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.run(cmd, check=True)
    if force or _torch_ops_stale():
        cmd = _torch_ops_command()
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.run(cmd, check=True)
        with open(TORCH_OPS_STAMP, "w") as f:
            f.write(_torch_and_python())
    return LIB


if __name__ == "__main__":
    build(verbose=True, force="--force" in sys.argv,
          extra=["-Xptxas", "-v"] if "--ptxas" in sys.argv else None)
