"""Rows of a table by token and the table's gradient, on device tensors, against the definition in 64 bits.

Tolerances count roundings of fp32 (u = 2^-24): a row's sum over c tokens passes at most c + 40 additions (its pieces' shares and the shares' sums included), the
scale one more.
"""
import math

import pytest

import tatara_b200 as tb

torch = pytest.importorskip("torch")
from op_plain import HALF, TINY, U32  # noqa: E402

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def ops():
    from tatara_b200 import ops as o
    return o


def tokens_of(count, rows, seed, missing=0.0, skew=True, dtype=torch.int64):
    g = torch.Generator("cuda").manual_seed(seed)
    u = torch.rand(count, generator=g, device="cuda", dtype=torch.float64)
    t = (torch.exp(u * math.log(rows + 1)) - 1 if skew else u * rows).long().clamp(0, rows - 1)
    return torch.where(torch.rand(count, generator=g, device="cuda") < missing, -1, t).to(dtype)


def values(rows, n, dtype, seed, pad=0, offset=0):
    g = torch.Generator("cuda").manual_seed(seed)
    return torch.randn(rows, n + pad + offset, generator=g, device="cuda").to(dtype)[:, offset:offset + n]


def check_forward(tokens, table, scale, out):
    ok = (tokens >= 0) & (tokens < len(table))
    want = torch.where(ok[..., None], table.double()[torch.where(ok, tokens, 0).long()] * float(torch.tensor(scale, dtype=torch.float32)), 0.0)
    assert out.dtype == table.dtype and out.shape == want.shape
    assert ((out.double() - want).abs() <= (U32 + HALF[out.dtype]) * want.abs() * 1.01 + TINY[out.dtype]).all()
    assert (out[~ok] == 0).all()


def check_backward(dy, tokens, rows, scale, got):
    ok = ((tokens >= 0) & (tokens < rows)).flatten()
    t, d = tokens.flatten()[ok].long(), dy.reshape(-1, dy.shape[-1])[ok].double()
    s = float(torch.tensor(scale, dtype=torch.float32))
    zero = torch.zeros(rows, d.shape[1], dtype=torch.float64, device="cuda")
    want, size = zero.index_add(0, t, d) * s, zero.index_add(0, t, d.abs()) * abs(s)
    many = torch.bincount(t, minlength=rows)[:, None].double()
    assert got.shape == want.shape
    assert ((got.double() - want).abs() <= U32 * (many + 41) * size + HALF[got.dtype] * want.abs() * 1.01 + TINY[got.dtype]).all()
    assert (got[many[:, 0] == 0] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("count,rows,n", [(1, 1, 1), (3, 5, 2), (100, 9, 8), (77, 50, 33), (300, 81, 64), (64, 1000, 136), (33, 7, 256), (50, 40, 264), (40, 12, 520), (21, 30, 1024), (9, 3, 1537), (5, 4, 4100)])
def test_forward(count, rows, n, dtype):
    table = values(rows, n, dtype, n)
    for tokens in (tokens_of(count, rows, count, 0.2), tokens_of(count, rows, count, 0.0, False, torch.int32)):
        for scale in (1.0, math.sqrt(n), -0.37):
            check_forward(tokens, table, scale, ops().embedding_forward(tokens, table, scale=scale))


# one block's sort and several, one to three passes, short lists and long ones, tiles of every width
BACK = [(1, 1, 1), (3, 5, 2), (100, 9, 8), (1000, 81, 64), (31, 40, 33), (33, 1, 96), (500, 2, 100), (300, 5000, 136), (4096, 1024, 40), (4097, 1025, 40), (6000, 300, 256), (2000, 73305, 264), (700, 40, 520),
        (900, 30, 777), (300, 20, 1030), (64, 6, 4100), (20000, 3, 24), (70000, 2000, 20), (100, 2_000_000, 8), (5000, 1_048_577, 16), (150000, 11, 6)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("count,rows,n", BACK)
def test_backward(count, rows, n, dtype):
    dy = values(count, n, dtype, count + n)
    tokens = tokens_of(count, rows, count, 0.1 if count % 2 else 0.0)
    check_backward(dy, tokens, rows, 1.0, ops().embedding_backward(dy, tokens, rows))
    even = tokens_of(count, rows, count + 1, 0.3, False, torch.int32)
    check_backward(dy, even, rows, 0.7, got := ops().embedding_backward(dy, even, rows, scale=0.7, dtype=torch.float32))
    assert got.dtype == torch.float32


@pytest.mark.parametrize("count", [31, 32, 33, 63, 64, 65, 96, 97, 127, 1000, 65536, 65537, 140000])
def test_lists_that_end_at_a_piece(count):
    """All tokens in one row, in two, and lists of 32, 33 and 64 tokens that begin and end around the pieces' bounds."""
    for n, dtype in ((4, torch.float32), (40, torch.bfloat16)):
        dy = values(count, n, dtype, count)
        for tokens in (torch.zeros(count, dtype=torch.int64, device="cuda"), (torch.arange(count, device="cuda") >= count // 2).long(), torch.arange(count, device="cuda") // 33,
                       torch.arange(count, device="cuda") // 32, torch.arange(count, device="cuda") // 64, (torch.arange(count, device="cuda") + 17) // 65):
            rows = int(tokens.max()) + 2
            check_backward(dy, tokens, rows, 1.0, ops().embedding_backward(dy, tokens, rows))


# tiles of every width, one and several, rows on 16-byte boundaries and not, with lists that go over a piece, a chunk of pieces and much of the whole
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("count,rows,n", [(5000, 30, 777), (4000, 7, 768), (3000, 5, 1030), (2500, 3, 4100), (9000, 2, 513), (20000, 400, 96), (9000, 60, 128), (6000, 50, 200), (6000, 70, 250), (6000, 40, 1536),
                                          (30000, 900, 768), (800_000, 5000, 4), (700_000, 3, 9)])
def test_long_lists_of_wide_rows(count, rows, n, dtype):
    dy, tokens = values(count, n, dtype, count + n), tokens_of(count, rows, n, 0.1)
    got = ops().embedding_backward(dy, tokens, rows)
    check_backward(dy, tokens, rows, 1.0, got)
    assert torch.equal(ops().embedding_backward(dy, tokens.int(), rows), got)


def test_a_first_call_may_be_captured():
    """Nothing has to be set up before: a process of its own whose first calls go into a graph."""
    import subprocess
    import sys
    from helpers import ROOT
    code = ("import torch; from tatara_b200 import ops\n"
            "t = torch.arange(5000, device='cuda') % 40; dy = torch.ones(5000, 768, device='cuda'); torch.cuda.synchronize()\n"
            "g = torch.cuda.CUDAGraph()\n"
            "with torch.cuda.graph(g):\n"
            "    d = ops.embedding_backward(dy, t, 41); o = ops.expert_order(t.int()[:, None].contiguous(), 40); y = ops.rms_norm_forward(dy)[0]\n"
            "g.replay(); torch.cuda.synchronize()\n"
            "assert (d[:40] == 125).all() and (d[40] == 0).all() and (o.offsets.cpu() == torch.arange(41) * 125).all() and ((y - 1).abs() < 1e-5).all()\n")
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset", [1, 8])
def test_rows_of_a_wider_buffer(dtype, offset):
    table, tokens = values(50, 96, dtype, 3, 8, offset), tokens_of(200, 50, 4, 0.1)
    out = torch.full((200, 120), 3.0, dtype=dtype, device="cuda")
    check_forward(tokens, table, 2.0, ops().embedding_forward(tokens, table, scale=2.0, out=out[:, offset:offset + 96]))
    assert (out[:, :offset] == 3).all() and (out[:, offset + 96:] == 3).all()
    dy = values(200, 96, dtype, 5, 8, offset)
    check_backward(dy, tokens, 50, 2.0, ops().embedding_backward(dy, tokens, 50, scale=2.0))


def test_tokens_of_any_shape():
    table = values(30, 24, torch.float32, 1)
    tokens = tokens_of(60, 30, 2, 0.1).view(3, 4, 5)
    out = ops().embedding_forward(tokens, table)
    assert out.shape == (3, 4, 5, 24)
    check_forward(tokens, table, 1.0, out)
    check_backward(out, tokens, 30, 1.0, ops().embedding_backward(out, tokens, 30))
    one = torch.tensor(7, device="cuda")
    assert torch.equal(ops().embedding_forward(one, table), table[7])
    d = ops().embedding_backward(table[7], one, 30)
    assert torch.equal(d[7], table[7]) and (d[:7] == 0).all() and (d[8:] == 0).all()


def test_tokens_outside_the_table():
    table = values(10, 16, torch.float16, 1)
    tokens = torch.tensor([0, -1, 10, 9, 2 ** 31, 2 ** 40 + 3, -2 ** 63, 2 ** 63 - 1, 2 ** 32 + 5], device="cuda")
    out = ops().embedding_forward(tokens, table)
    assert torch.equal(out[[0, 3]], table[[0, 9]]) and (out[[1, 2, 4, 5, 6, 7, 8]] == 0).all()
    dy = values(9, 16, torch.float16, 2)
    dy[[1, 2, 4, 5, 6, 7, 8]] = math.nan   # not looked at
    d = ops().embedding_backward(dy, tokens, 10)
    assert torch.equal(d[[0, 9]], dy[[0, 3]]) and (d[1:9] == 0).all()
    d = ops().embedding_backward(dy, torch.full((9,), -1, device="cuda"), 10)
    assert (d == 0).all()


def test_values_that_are_not_numbers_stay_in_their_rows():
    tokens = torch.arange(200, device="cuda") % 4
    dy = values(200, 40, torch.float32, 3)
    dy[6, 5] = math.inf
    dy[9, 7] = math.nan
    d = ops().embedding_backward(dy, tokens, 5)
    assert d[2, 5] == math.inf and d[1, 7].isnan()
    d[2, 5] = d[1, 7] = 0
    assert d.isfinite().all() and (d[4] == 0).all()


def test_no_tokens():
    table = values(10, 16, torch.float32, 1)
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    assert ops().embedding_forward(none, table).shape == (0, 16)
    d = ops().embedding_backward(torch.empty(0, 16, device="cuda"), none, 10)
    assert d.shape == (10, 16) and (d == 0).all()


def test_repeated_calls_agree():
    tokens, dy = tokens_of(50000, 3000, 1), values(50000, 72, torch.float32, 2)
    first = ops().embedding_backward(dy, tokens, 3000)
    for _ in range(4):
        assert torch.equal(ops().embedding_backward(dy, tokens, 3000), first)


def test_gradient_against_differences():
    tokens, table, dy = tokens_of(90, 12, 3, 0.1), values(12, 20, torch.float32, 1), values(90, 20, torch.float32, 2)
    grad = ops().embedding_backward(dy, tokens, 12, scale=1.5)
    ok = tokens >= 0
    value = lambda t: float((torch.where(ok[:, None], 1.5 * t[tokens.clamp(min=0)], 0.0) * dy.double()).sum())  # noqa: E731
    d = torch.randn(12, 20, device="cuda", dtype=torch.float64)
    want = (value(table.double() + 1e-3 * d) - value(table.double() - 1e-3 * d)) / 2e-3   # linear
    assert abs(float((grad.double() * d).sum()) - want) <= U32 * 150 * float((grad.double() * d).abs().sum()) + 1e-9


def test_offsets_beyond_32_bits():
    rows, n = 600_000, 4096
    table = torch.empty(rows, n, dtype=torch.float16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(1))
    tokens = torch.arange(rows - 1, -1, -1, device="cuda")
    out = ops().embedding_forward(tokens, table, scale=2.0)
    for i in (0, 1, rows // 2, rows - 1):
        assert torch.equal(out[i], (2 * table[rows - 1 - i].float()).half())
    d = ops().embedding_backward(out, tokens, rows, scale=0.5)
    for i in (0, rows // 2 + 1, rows - 2, rows - 1):
        assert torch.equal(d[i], table[i])
    del table, out, d


def test_refusals():
    o = ops()
    table, tokens, dy = torch.zeros(5, 8, device="cuda"), torch.zeros(6, dtype=torch.int64, device="cuda"), torch.zeros(6, 8, device="cuda")
    for bad in (lambda: o.embedding_forward(tokens.cpu(), table), lambda: o.embedding_forward(tokens, table.cpu()), lambda: o.embedding_forward(tokens.float(), table), lambda: o.embedding_forward(tokens, table.double()),
                lambda: o.embedding_forward(tokens, table[0]), lambda: o.embedding_forward(tokens, table[:0]), lambda: o.embedding_forward(tokens, table[:, :0]), lambda: o.embedding_forward(tokens[::2], table),
                lambda: o.embedding_forward(tokens, table.t()), lambda: o.embedding_forward(tokens, table, out=dy[:5]), lambda: o.embedding_forward(tokens, table, out=dy.half()),
                lambda: o.embedding_forward(tokens, table, scale="a"), lambda: o.embedding_forward(tokens[:5], table, out=table), lambda: o.embedding_backward(dy[:5], tokens, 5),
                lambda: o.embedding_backward(dy, tokens, 0), lambda: o.embedding_backward(dy, tokens, 1 << 31), lambda: o.embedding_backward(dy, tokens, "a"), lambda: o.embedding_backward(dy.double(), tokens, 5),
                lambda: o.embedding_backward(dy, tokens, 5, dtype=torch.float16), lambda: o.embedding_backward(dy, tokens.view(2, 3), 5), lambda: o.embedding_backward(dy, tokens.short(), 5),
                lambda: o.embedding_backward(None, tokens, 5), lambda: o.embedding_backward(dy, None, 5)):
        with pytest.raises(tb.TrainerError):
            bad()
