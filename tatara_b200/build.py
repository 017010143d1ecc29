"""Builds libtatara_b200.so (sm_100a) in-tree with nvcc.

    python -m tatara_b200.build [--force]

nvcc cross-compiles without a GPU.  The library links the CUDA runtime statically and has no other
link-time dependency (NCCL is opened at run time only when world_size > 1).

Where torch is installed, the binding of the operators on torch tensors (_ops.so, csrc/torch_ops.cpp, plain C++) is built too.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ_DIR = os.path.join(HERE, "build")
LIB_PATH = os.path.join(HERE, "libtatara_b200.so")
SOURCES = ["ft_kernels.cu", "ft_slice_bwd.cu", "sort_kernels.cu", "dense_kernels.cu", "tail_kernels.cu", "opt_kernels.cu", "psv.cu", "host_util.cu", "host_mem.cu", "trainer.cu", "noalloc.cu", "microbench.cu", "l1_tc.cu", "peer_exchange.cu",
           "norm_kernels.cu", "route_kernels.cu", "orth_kernels.cu", "orth_tc.cu", "rms_kernels.cu", "rms_quantised.cu", "expert_kernels.cu", "embed_kernels.cu"]
# every object depends on every header: csrc/*.cuh and the public C header
HEADERS = sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))) + [
    os.path.join(os.path.dirname(HERE), "include", "tatara_b200.h")]
NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC",
              "-diag-suppress", "68"]


def _nvcc():
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found (set NVCC)")


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def build(force: bool = False, verbose: bool = False) -> str:
    nvcc = _nvcc()
    os.makedirs(OBJ_DIR, exist_ok=True)
    objs, jobs = [], []
    for src in SOURCES:
        s = os.path.join(CSRC, src)
        o = os.path.join(OBJ_DIR, src.replace(".cu", ".o"))
        objs.append(o)
        if force or _stale(o, [s] + HEADERS):
            cmd = [nvcc] + NVCC_FLAGS + (["-Xptxas", "-v"] if verbose else []) + ["-c", s, "-o", o]
            jobs.append(cmd)

    def run(cmd):
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError("nvcc failed: %s\n%s" % (" ".join(cmd), r.stderr))
        return r.stderr

    with ThreadPoolExecutor(max_workers=max(1, min(len(jobs), os.cpu_count() or 1))) as ex:
        for out in ex.map(run, jobs):
            if verbose and out:
                sys.stderr.write(out)
    if jobs or force or _stale(LIB_PATH, objs):
        run([nvcc, "-shared", "-o", LIB_PATH] + objs + ["-gencode", "arch=compute_100a,code=sm_100a", "-Xcompiler",
             "-fPIC", "-Xlinker", "--exclude-libs=ALL", "-ldl"])
    return LIB_PATH


OPS_PATH = os.path.join(HERE, "_ops.so")


def build_ops(force: bool = False) -> str | None:
    """Builds the torch binding beside the library it calls; None where torch is not installed."""
    try:
        import torch
    except ImportError:
        return None
    root = os.path.dirname(torch.__file__)
    src, libs = os.path.join(CSRC, "torch_ops.cpp"), os.path.join(root, "lib")
    stamp = os.path.join(OBJ_DIR, "torch_version")  # the binding belongs to one torch
    same = os.path.exists(stamp) and open(stamp).read() == torch.__version__
    if force or not same or _stale(OPS_PATH, [src, HEADERS[-1]]):
        cmd = [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-w", "-D_GLIBCXX_USE_CXX11_ABI=%d" % torch._C._GLIBCXX_USE_CXX11_ABI,
               "-I" + sysconfig.get_paths()["include"], "-I" + os.path.join(root, "include"), "-I" + os.path.join(root, "include", "torch", "csrc", "api", "include"),
               "-I" + os.path.join(os.path.dirname(os.path.dirname(_nvcc())), "include"), src, "-o", OPS_PATH, "-L" + libs, "-ltorch_python", "-ltorch_cuda", "-ltorch_cpu",
               "-ltorch", "-lc10_cuda", "-lc10", "-L" + HERE, "-l:libtatara_b200.so", "-Wl,-rpath,$ORIGIN", "-Wl,-rpath," + libs]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError("g++ failed: %s\n%s" % (" ".join(cmd), r.stderr))
        with open(stamp, "w") as f:
            f.write(torch.__version__)
    return OPS_PATH


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
    print(build_ops(force="--force" in sys.argv) or "torch is not installed: no _ops.so")
