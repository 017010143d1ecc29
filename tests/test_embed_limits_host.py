"""The table gradient's host side at the largest sizes: built with the compiler's check for signed overflow, whose reports are this test's failures.

No kernel runs: the addresses are never read, and without a GPU the launches are refused.
"""
import os
import subprocess
import sys

import pytest

import tatara_b200 as tb
from helpers import ROOT
from tatara_b200 import build

CALLS = r"""
import ctypes as C, sys
lib = C.CDLL(sys.argv[1])
i64, vp = C.c_int64, C.c_void_p
lib.tb_embedding_backward_workspace.restype = i64
lib.tb_embedding_backward_workspace.argtypes = [i64, i64, C.c_int]
lib.tb_embedding_backward.argtypes = [vp, i64, C.c_int, vp, C.c_int, i64, i64, C.c_int, C.c_float, vp, i64, C.c_int, vp, i64, vp, C.c_char_p, C.c_size_t]
lib.tb_embedding_forward.argtypes = [vp, C.c_int, i64, vp, i64, C.c_int, i64, C.c_int, C.c_float, vp, i64, vp, C.c_char_p, C.c_size_t]
codes = set()
for n in (1, 255, 768, 4097, 1 << 20, 1 << 29, (1 << 30) - 4, 1 << 30):
    for count, rows in ((1, 1), (5000, 2), (131072, 73305), ((1 << 31) - 1024, 2), (1, (1 << 31) - 1), ((1 << 31) - 1024, (1 << 31) - 1)):
        for kind, out in ((0, 0), (1, 1), (2, 0)):
            err = C.create_string_buffer(300)
            work = lib.tb_embedding_backward_workspace(count, rows, n)
            codes.add(lib.tb_embedding_backward(1 << 60, n, kind, 1 << 20, 8, count, rows, n, 1.0, 1 << 62, n, out, 1 << 40, max(work, 0), None, err, 300))
            codes.add(lib.tb_embedding_forward(1 << 20, 8, count, 1 << 60, n, kind, rows, n, 1.0, 1 << 62, n, None, err, 300))
assert codes <= {-1, -6}, codes   # refused, or no device
"""


@pytest.mark.skipif(tb.load_library().tb_device_count() > 0, reason="the addresses are not real")
def test_sizes_do_not_overflow(tmp_path):
    try:
        nvcc = build._nvcc()
    except RuntimeError:
        pytest.skip("nvcc is not installed")
    lib = str(tmp_path / "checked.so")
    r = subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-O0", "-Xcicc", "-O0", "-Xptxas", "-O0", "-std=c++17", "-Xcompiler", "-fPIC,-fsanitize=signed-integer-overflow",
                        "-diag-suppress", "68", "-shared", "-Xlinker", "-Bsymbolic", os.path.join(ROOT, "tatara_b200", "csrc", "embed_kernels.cu"), "-o", lib, "-lubsan"], capture_output=True, text=True)
    if r.returncode != 0 and "ubsan" in r.stderr:
        pytest.skip("the compiler's check is not installed")
    assert r.returncode == 0, r.stderr[-2000:]
    r = subprocess.run([sys.executable, "-c", CALLS, lib], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "runtime error" not in r.stderr, r.stderr[-2000:]
