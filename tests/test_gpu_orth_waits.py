"""Waits of the tensor-core products that run out: what comes out is right or NaN, and the device is left as it was.

The products' source is built once more with the tries of every kind of wait in a table.  With no tries for one kind, the warp that waits so gives up at once and stops;
the others then wait in vain, for 2000 tries each.  Nothing is taken out of the kernels: every access keeps its bounds, every wait ends, copies and products under
way are waited for before a block stores or ends.
"""
import ctypes as C
import os
import subprocess

import pytest

from helpers import ROOT

torch = pytest.importorskip("torch")
from tatara_b200 import build  # noqa: E402

pytestmark = pytest.mark.gpu
SOURCE = r"""
#include <cuda_runtime.h>
static __device__ int wait_tries[5];
#define OT_WAIT_LIMIT(role) (wait_tries[role])
#include "orth_tc.cu"

extern "C" long long waits_workspace(int batch, int rows, int cols, int limbs) { return orth_tc_workspace(batch, rows, cols, limbs); }
extern "C" int waits_run(const int* tries, const void* x, void* out, int type, int limbs, int batch, int rows, int cols, void* work) {
    if (cudaMemcpyToSymbol(wait_tries, tries, sizeof wait_tries) != cudaSuccess) return 1;
    OrthIo io = {};
    io.g = x;
    io.out = out;
    io.g_batch = io.out_batch = (long long)rows * cols;
    io.g_stride = io.out_stride = cols;
    io.rows = rows;
    io.cols = cols;
    io.batch = batch;
    const OrthPoly poly = {5, 3.4445f, -4.7750f, 2.0315f, 1e-7f};
    launch_orth_tc(nullptr, io, poly, type, limbs, work);
    return cudaDeviceSynchronize() == cudaSuccess && cudaGetLastError() == cudaSuccess ? 0 : 2;
}
"""
COPIES, PRODUCTS, RELAY, SUMS, END = range(5)
# one block per tile of 64 columns, with K in parts and whole; of 128; pairs of blocks with 256; several tiles per block
SHAPES = [(1, 70, 2500), (1, 359, 785), (1, 1500, 1100), (4, 1000, 777), (6, 1024, 1024), (1, 2600, 2700)]


@pytest.fixture(scope="module")
def waits(tmp_path_factory):
    try:
        nvcc = build._nvcc()
    except RuntimeError:
        pytest.skip("nvcc is not installed")
    at = tmp_path_factory.mktemp("waits")
    (at / "waits.cu").write_text(SOURCE)
    lib = str(at / "waits.so")  # bound to its own functions: the package's library has the same ones in the global scope
    r = subprocess.run([nvcc] + build.NVCC_FLAGS + ["-I", os.path.join(ROOT, "tatara_b200", "csrc"), "-shared", "-Xlinker", "-Bsymbolic", str(at / "waits.cu"), "-o", lib],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    lib = C.CDLL(lib)
    lib.waits_workspace.restype = C.c_longlong
    lib.waits_run.argtypes = [C.POINTER(C.c_int), C.c_void_p, C.c_void_p] + [C.c_int] * 5 + [C.c_void_p]
    return lib


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("batch,rows,cols", SHAPES)
def test_waits_that_run_out(waits, batch, rows, cols, dtype):
    from tatara_b200 import ops
    limbs, kind = (2, 0) if dtype == torch.float32 else (1, 2)
    x = torch.randn(batch, rows, cols, generator=torch.Generator("cuda").manual_seed(rows), device="cuda").to(dtype)
    want = ops.orthogonalise(x)
    assert want.isfinite().all()
    work = torch.empty(waits.waits_workspace(batch, rows, cols, limbs), dtype=torch.uint8, device="cuda")

    def run(tries):
        out = torch.full_like(x, 7.0)
        torch.cuda.synchronize()
        assert waits.waits_run((C.c_int * 5)(*tries), x.data_ptr(), out.data_ptr(), kind, limbs, batch, rows, cols, work.data_ptr()) == 0
        return out

    enough = [1 << 20] * 4 + [1 << 22]
    assert torch.equal(run(enough), want)
    for role in (COPIES, PRODUCTS, RELAY, SUMS):
        got = run([0 if r == role else 2000 for r in range(4)] + [1 << 22])
        assert ((got == want) | got.isnan()).all(), role
        # only pairs of blocks have a relay
        assert got.isnan().all() or role == RELAY, role
    assert torch.equal(run(enough), want)          # nothing of it is left: tensor memory, barriers
    assert torch.equal(ops.orthogonalise(x), want)
