"""Waits for the copies of a table gradient that run out: what comes out is right or NaN, and the device is left as it was.

The gradient's source is built once more with the tries of its waits in a table.  With none or a few for a copy, warps give up while their copies, all of them ordinary ones inside the
tensors, are on their way.  Nothing is taken out of the kernels: every wait ends, and copies under way are waited for before their memory holds sums or the block ends.
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
static __device__ int wait_tries[2];
#define BULK_WAIT_LIMIT(role) (wait_tries[role])
#include "embed_kernels.cu"

extern "C" int waits_run(const int* tries, const void* dy, int type, const void* tokens, long long count, long long rows, int n, void* dtable, void* work, long long work_bytes) {
    if (cudaMemcpyToSymbol(wait_tries, tries, sizeof wait_tries) != cudaSuccess) return 1;
    char err[256];
    if (tb_embedding_backward(dy, n, type, tokens, 8, count, rows, n, 0.5f, dtable, n, TB_TYPE_F32, work, work_bytes, nullptr, err, sizeof err) != TB_OK) return 2;
    return cudaDeviceSynchronize() == cudaSuccess && cudaGetLastError() == cudaSuccess ? 0 : 3;
}
extern "C" long long waits_workspace(long long count, long long rows, int n) { return tb_embedding_backward_workspace(count, rows, n); }
"""
KINDS = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
ENOUGH = 1 << 22


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
    lib.waits_workspace.argtypes = [C.c_longlong, C.c_longlong, C.c_int]
    lib.waits_run.argtypes = [C.POINTER(C.c_int), C.c_void_p, C.c_int, C.c_void_p, C.c_longlong, C.c_longlong, C.c_int, C.c_void_p, C.c_void_p, C.c_longlong]
    return lib


# rows by copies: whole 16-byte accesses in tiles of six and of four, rows that start anywhere in tiles of eight and of sixteen
@pytest.mark.parametrize("dtype,n", [(torch.float32, 768), (torch.float32, 2000), (torch.float16, 1200), (torch.bfloat16, 3000), (torch.float32, 201), (torch.float16, 1001)])
@pytest.mark.parametrize("tokens", ["one", "few", "many"])
def test_waits_that_run_out(waits, tokens, dtype, n):
    from tatara_b200 import ops
    g = torch.Generator("cuda").manual_seed(n)
    count, rows = 9000, 400
    # one: a list of all tokens; few: lists of many pieces, several of them to a block; many: lists of one piece or less beside two long ones
    token = {"one": lambda: torch.full((count,), 7, device="cuda"), "few": lambda: torch.randint(0, 50, (count,), generator=g, device="cuda"),
             "many": lambda: torch.randint(0, 350, (count,), generator=g, device="cuda")}[tokens]()
    if tokens == "many":
        token[::9], token[5::11] = 3, 349
    dy = torch.randn(count, n, generator=g, device="cuda").to(dtype)
    want = ops.embedding_backward(dy, token, rows, scale=0.5, dtype=torch.float32)
    assert want.isfinite().all()
    work = torch.empty(waits.waits_workspace(count, rows, n), dtype=torch.uint8, device="cuda")
    asked = torch.bincount(token, minlength=rows) > 0

    def run(tries):
        out = torch.full((rows, n), 7.0, device="cuda")
        torch.cuda.synchronize()
        assert waits.waits_run((C.c_int * 2)(tries, ENOUGH), dy.data_ptr(), KINDS[dtype], token.data_ptr(), count, rows, n, out.data_ptr(), work.data_ptr(), work.numel()) == 0
        return out

    assert torch.equal(run(ENOUGH), want)
    assert run(0)[asked].isnan().all()   # every warp that needs a row gives up on its first one
    for tries in (0, 1, 2, 3, 0):
        got = run(tries)
        assert ((got == want) | got.isnan()).all(), tries
    assert torch.equal(run(ENOUGH), want)          # nothing of it is left
    assert torch.equal(ops.embedding_backward(dy, token, rows, scale=0.5, dtype=torch.float32), want)
