"""Layer norm on device tensors against the definition in 64 bits.

Tolerances count roundings of fp32 (u = 2^-24).  A row's sum runs through at most n / 32 + 1 terms of a thread and ten more
additions, so L = n / 32 + 11 bounds its relative error in u; a column's sum through at most `rows` + 40 terms.
"""
import ctypes as C
import math

import pytest

import tatara_b200 as tb

torch = pytest.importorskip("torch")
from op_plain import HALF, TINY, U32, norm_backward, norm_forward  # noqa: E402

pytestmark = pytest.mark.gpu
EPS = 1e-5
TYPES = [torch.float32, torch.float16, torch.bfloat16]
# widths around every change of layout: warps, several warps, the longest rows in registers (8192 back, 16384 forward) and beyond, odd ones
SIZES = [(1, 1), (3, 2), (37, 8), (5, 31), (129, 256), (64, 257), (40, 512), (33, 520), (9, 777), (70, 1536), (21, 2048), (7, 2056), (6, 4104),
         (5, 8192), (3, 8200), (2, 16384), (3, 16400), (300, 20), (2000, 64)]


def ops():
    from tatara_b200 import ops as o
    return o


def make(rows, n, dtype, seed, strided=False, offset=0):
    g = torch.Generator("cuda").manual_seed(seed)
    wide = torch.randn(rows, (n + 13 if strided else n) + offset, generator=g, device="cuda") * (0.1 + torch.rand(rows, 1, generator=g, device="cuda")) + 0.7
    return wide.to(dtype)[:, offset:offset + n]


def check_forward(x, w, b, got, eps=EPS):
    y, mean, rstd = got
    want, m, r = norm_forward(x, w, b, eps)
    n = x.shape[1]
    length = n / 32 + 11
    size = x.double().abs().mean(1)
    wa = w.double().abs() if w is not None else 1.0
    ba = b.double().abs() if b is not None else 0.0
    assert (mean.double() - m).abs().le(U32 * length * size + 1e-45).all()
    # the variance: its own sum, and the mean's error once more for the squared distance
    off = U32 * length * size * r
    rel = U32 * (length + 6) + off ** 2
    assert ((rstd.double() - r).abs() <= rel * r).all()
    xh = (x.double() - m[:, None]).abs() * r[:, None]
    tol = off[:, None] * wa + (rel[:, None] + 4 * U32) * xh * wa + 2 * U32 * ba + HALF[y.dtype] * want.abs() * 1.01 + TINY[y.dtype]
    assert ((y.double() - want).abs() <= tol).all(), float(((y.double() - want).abs() / tol).max())


def check_backward(dy, x, mean, rstd, w, got):
    dx, dw, db = got
    want, ww, wb, xh, t = norm_backward(dy, x, mean, rstd, w)
    rows, n = x.shape
    length = n / 32 + 11
    ta, r = t.abs(), rstd.double()[:, None]
    tol = U32 * r * (6 * ta + (length + 6) * (ta.mean(1, keepdim=True) + xh.abs() * (ta * xh.abs()).mean(1, keepdim=True)))
    tol = tol + HALF[dx.dtype] * want.abs() * 1.01 + TINY[dx.dtype]
    assert ((dx.double() - want).abs() <= tol).all(), float(((dx.double() - want).abs() / tol).max())
    g = dy.double().abs()
    assert ((dw.double() - ww).abs() <= U32 * (rows + 43) * (g * xh.abs()).sum(0) + 1e-44).all()
    assert ((db.double() - wb).abs() <= U32 * (rows + 43) * g.sum(0) + 1e-44).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n", SIZES)
def test_both_directions(rows, n, dtype):
    x = make(rows, n, dtype, rows + n)
    dy = make(rows, n, dtype, rows + n + 1) * 0.01
    w, b = 1 + 0.2 * torch.randn(n, device="cuda"), torch.randn(n, device="cuda")
    y, mean, rstd = ops().layer_norm_forward(x, w, b, eps=EPS)
    check_forward(x, w, b, (y, mean, rstd))
    check_backward(dy, x, mean, rstd, w, ops().layer_norm_backward(dy, x, mean, rstd, w))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n,offset", [(50, 512, 0), (50, 512, 1), (17, 1000, 3), (9, 9000, 5), (1, 40, 2)])
def test_rows_of_a_wider_buffer(rows, n, offset, dtype):
    x, dy = make(rows, n, dtype, 1, True, offset), make(rows, n, dtype, 2, True, offset)
    got = ops().layer_norm_forward(x, eps=EPS)
    check_forward(x, None, None, got)
    check_backward(dy, x, got[1], got[2], None, ops().layer_norm_backward(dy, x, got[1], got[2]))
    # results into columns of a wider buffer leave their neighbours alone
    wide = torch.full((rows, n + 9), 3.0, dtype=dtype, device="cuda")
    ops().layer_norm_forward(x, eps=EPS, out=wide[:, 4:4 + n])
    assert (wide[:, 4:4 + n] == got[0]).all() and (wide[:, :4] == 3).all() and (wide[:, 4 + n:] == 3).all()


def test_in_place_and_repeated():
    x, dy = make(700, 384, torch.float32, 5), make(700, 384, torch.float32, 6)
    y, mean, rstd = ops().layer_norm_forward(x)
    first = ops().layer_norm_backward(dy, x, mean, rstd)
    again = ops().layer_norm_backward(dy, x, mean, rstd)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    z = x.clone()
    assert torch.equal(ops().layer_norm_forward(z, out=z)[0], y)
    assert torch.equal(ops().layer_norm_backward(g := dy.clone(), x, mean, rstd, out=g)[0], first[0])


def test_constant_rows_large_offsets_and_values_that_are_not_numbers():
    x = torch.full((4, 300), 7.25, device="cuda")
    y, mean, rstd = ops().layer_norm_forward(x, eps=EPS)
    assert (y == 0).all() and (mean == 7.25).all()
    big = make(8, 512, torch.float32, 9) + 4096.0   # a variance far below the squared mean
    check_forward(big, None, None, ops().layer_norm_forward(big, eps=EPS))
    x = make(5, 96, torch.float32, 3)
    x[1, 7], x[3, 95] = float("inf"), float("nan")
    y = ops().layer_norm_forward(x)[0]
    assert y[1].isnan().any() and y[3].isnan().all()
    check_forward(x[[0, 2, 4]], None, None, tuple(t[[0, 2, 4]] for t in ops().layer_norm_forward(x)), 1e-5)


def test_no_rows():
    x = torch.empty(0, 40, device="cuda")
    y, mean, rstd = ops().layer_norm_forward(x)
    dx, dw, db = ops().layer_norm_backward(x, x, mean, rstd)
    assert y.shape == dx.shape == (0, 40) and (dw == 0).all() and (db == 0).all()


@pytest.mark.parametrize("n", [100, 1000, 1001, 5000, 9001, 20000])
def test_in_place_at_every_length(n):
    x, dy = make(40, n, torch.float32, 31), make(40, n, torch.float32, 32)
    w = 1 + 0.2 * torch.randn(n, device="cuda")
    y, mean, rstd = ops().layer_norm_forward(x, w, eps=EPS)
    want = ops().layer_norm_backward(dy, x, mean, rstd, w)
    z = x.clone()
    assert torch.equal(ops().layer_norm_forward(z, w, eps=EPS, out=z)[0], y)
    for same in ("dy", "x"):
        t = {"dy": dy.clone(), "x": x.clone()}
        got = ops().layer_norm_backward(t["dy"], t["x"], mean, rstd, w, out=t[same])
        assert all(torch.equal(a, b) for a, b in zip(got, want)), same


def test_outputs_beside_and_over_the_inputs():
    n = 24
    wide = make(50, 2 * n + 3, torch.float32, 33)
    x, dy = wide[:, :n].clone(), make(50, n, torch.float32, 34)
    y, mean, rstd = ops().layer_norm_forward(wide[:, :n], eps=EPS)   # strides decide the order of a row's sum
    assert torch.equal(ops().layer_norm_forward(wide[:, :n], eps=EPS, out=wide[:, n:2 * n])[0], y)   # other columns of the same rows
    rows = torch.cat([x, x])
    assert torch.equal(ops().layer_norm_forward(rows[::2], eps=EPS, out=rows[1::2])[0], ops().layer_norm_forward(torch.cat([x, x])[::2].clone(), eps=EPS)[0])
    with pytest.raises(tb.TrainerError, match="overlaps"):
        ops().layer_norm_forward(wide[:, :n], eps=EPS, out=wide[:, 1:n + 1])
    with pytest.raises(tb.TrainerError, match="overlaps"):
        ops().layer_norm_backward(dy, wide[:, :n], mean, rstd, out=wide[:, 1:n + 1])
    with pytest.raises(tb.TrainerError, match="overlaps"):
        ops().layer_norm_forward(rows[:50], eps=EPS, out=rows[1:51])
    with pytest.raises(tb.TrainerError, match="overlaps"):
        ops().layer_norm_backward(rows[:50], x, mean, rstd, out=rows[1:51])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [127, 128, 129, 255, 257, 511, 769, 1175, 2561, 3071, 3073, 4095, 4097, 8191])
def test_columns_around_the_kernels_bounds(n, dtype):
    rows = 37
    for offset in (0, 1):
        x, dy = make(rows, n, dtype, n, True, offset), make(rows, n, dtype, n + 1, False, offset)
        w, b = 1 + 0.2 * torch.randn(n, device="cuda"), torch.randn(n, device="cuda")
        got = ops().layer_norm_forward(x, w, b, eps=EPS)
        check_forward(x, w, b, got)
        check_backward(dy, x, got[1], got[2], w, ops().layer_norm_backward(dy, x, got[1], got[2], w))


@pytest.mark.parametrize("rows,n", [(6, 33), (4, 512)])
def test_gradient_against_differences(rows, n):
    x, dy = make(rows, n, torch.float32, 21), make(rows, n, torch.float32, 22)
    w, b = 1 + 0.2 * torch.randn(n, device="cuda"), torch.randn(n, device="cuda")
    _, mean, rstd = ops().layer_norm_forward(x, w, b, eps=EPS)
    dx, dw, db = ops().layer_norm_backward(dy, x, mean, rstd, w)
    value = lambda x, w, b: float((norm_forward(x, w, b, EPS)[0] * dy.double()).sum())  # noqa: E731
    g = torch.Generator("cuda").manual_seed(4)
    h = 1e-5  # central differences in 64 bits: error h^2 ~ 1e-10 of the third derivative, rounding 1e-16 / h
    for at, grad in (("x", dx), ("w", dw), ("b", db)):
        d = torch.randn(grad.shape, generator=g, device="cuda", dtype=torch.float64)
        moved = [{"x": x.double(), "w": w.double(), "b": b.double()} for _ in range(2)]
        moved[0][at] = moved[0][at] + h * d
        moved[1][at] = moved[1][at] - h * d
        want = (value(**moved[0]) - value(**moved[1])) / (2 * h)
        # 2^-24 times the chains of the sums, with mean and rstd themselves rounded
        tol = U32 * (n + rows + 60) * float((grad.double() * d).abs().sum()) + 1e-6
        assert abs(float((grad.double() * d).sum()) - want) <= tol


def test_offsets_beyond_32_bits():
    rows, n = 1_100_000, 2048
    x = torch.empty(rows, n, dtype=torch.float16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(1))
    tail, keep = x[-5:].clone(), x[:5].clone()
    want = ops().layer_norm_forward(tail, eps=EPS)
    y, mean, rstd = ops().layer_norm_forward(x, eps=EPS, out=x)
    assert torch.equal(y[-5:], want[0]) and torch.equal(mean[-5:], want[1])
    assert torch.equal(y[:5], ops().layer_norm_forward(keep, eps=EPS)[0])
    dx, dw, db = ops().layer_norm_backward(y, y, torch.zeros_like(mean), torch.ones_like(rstd), out=y)
    t = want[0].float()
    ref = norm_backward(want[0], want[0], torch.zeros(5, device="cuda"), torch.ones(5, device="cuda"), None)
    assert (dx[-5:].double() - ref[0]).abs().max() <= 2.0 ** -10 * float(t.abs().max())   # one rounding of a value that cancels
    # sums of 1.1e6 squares of unit variance: chains of a few thousand per block, then 600 blocks
    assert (dw / rows - 1).abs().max() <= 0.01


def test_another_stream():
    x = make(5000, 768, torch.float32, 11)
    torch.cuda.synchronize()
    want = ops().layer_norm_forward(x)[0]
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        z = x * 1.0
        y, mean, rstd = ops().layer_norm_forward(z)
        dx = ops().layer_norm_backward(y, z, mean, rstd)[0]
    s.synchronize()
    assert torch.equal(y, want) and dx.isfinite().all()


def test_refusals():
    o = ops()
    x = torch.zeros(4, 8, device="cuda")
    v = torch.zeros(4, device="cuda")
    for bad in (lambda: o.layer_norm_forward(x.double()), lambda: o.layer_norm_forward(x.cpu()), lambda: o.layer_norm_forward(x[0]),
                lambda: o.layer_norm_forward(x.t()), lambda: o.layer_norm_forward(x[:1].expand(4, 8)), lambda: o.layer_norm_forward(x, torch.zeros(7, device="cuda")),
                lambda: o.layer_norm_forward(x, torch.zeros(8)), lambda: o.layer_norm_forward(x, eps=-1.0), lambda: o.layer_norm_forward(x, eps=float("nan")),
                lambda: o.layer_norm_forward(x[:, :0]), lambda: o.layer_norm_forward(x, out=x.half()), lambda: o.layer_norm_backward(x[:3], x, v, v),
                lambda: o.layer_norm_backward(x.half(), x, v, v), lambda: o.layer_norm_backward(x, x, v[:3], v)):
        with pytest.raises(tb.TrainerError):
            bad()
    lib = tb.load_library()
    p = x.data_ptr()
    assert lib.tb_layer_norm_backward(p, 8, p, 8, p, p, None, 0, 4, 8, p, 8, p, p, p, 0, None, None, 0) == -1   # workspace too small
    assert lib.tb_layer_norm_forward(None, 8, None, None, 1e-5, 0, 4, 8, p, 8, None, None, None, None, 0) == -1
    assert lib.tb_layer_norm_forward(p, 7, None, None, 1e-5, 0, 4, 8, p, 8, None, None, None, None, 0) == -1
    assert lib.tb_layer_norm_forward(p, 8, None, None, 1e-5, 3, 4, 8, p, 8, None, None, None, None, 0) == -1
    assert lib.tb_layer_norm_backward_workspace(-1, 8) == -1 and lib.tb_layer_norm_backward_workspace(4, 0) == -1


@pytest.mark.parametrize("rows,n", [(1, 9), (5, 19), (32, 64), (33, 64), (64, 40), (65, 40), (2, 100), (9, 200), (17, 200), (4, 1000), (5, 1001), (2, 5000), (1, 9000), (2, 9000)])
def test_gradients_of_few_rows(rows, n):
    x, dy = make(rows, n, torch.float32, rows + n), make(rows, n, torch.float32, rows + n + 7)
    w = 1 + 0.2 * torch.randn(n, device="cuda")
    _, mean, rstd = ops().layer_norm_forward(x, w, eps=EPS)
    got = ops().layer_norm_backward(dy, x, mean, rstd, w)
    check_backward(dy, x, mean, rstd, w, got)
    # either gradient alone, and gradients that do not start on a wide boundary
    lib, need = tb.load_library(), tb.load_library().tb_layer_norm_backward_workspace(rows, n)
    work, err = torch.empty(need, dtype=torch.uint8, device="cuda"), C.create_string_buffer(200)
    for use_w, use_b, off in ((True, False, 0), (False, True, 0), (False, False, 0), (True, True, 1)):
        dx, dw, db = torch.empty_like(x), torch.full((n + 1,), 7.0, device="cuda"), torch.full((n + 1,), 7.0, device="cuda")
        rc = lib.tb_layer_norm_backward(dy.data_ptr(), n, x.data_ptr(), n, mean.data_ptr(), rstd.data_ptr(), w.data_ptr(), 0, rows, n, dx.data_ptr(), n,
                                        dw[off:].data_ptr() if use_w else None, db[off:].data_ptr() if use_b else None, work.data_ptr(), need,
                                        torch.cuda.current_stream().cuda_stream, err, 200)
        assert rc == 0, err.value
        assert torch.equal(dx, got[0])
        for t, used, want in ((dw, use_w, got[1]), (db, use_b, got[2])):
            assert torch.equal(t[off:off + n], want) if used else (t == 7).all()
            assert (t[:off] == 7).all() and (t[off + n:] == 7).all()


def test_rows_of_two_to_the_31():
    """The longest rows that are taken, 2^31 - 5 columns, in numbers that leave nothing to round: columns of 1 and -1 in turn."""
    n = 2 ** 31 - 5
    if torch.cuda.mem_get_info()[0] < 130 << 30:
        pytest.skip("needs 130 GB of free device memory")
    half = lambda *s: torch.empty(*s, dtype=torch.float16, device="cuda")  # noqa: E731
    x, dy = half(2, n), half(2, n)
    x[:, 0::2], x[:, 1::2] = 1, -1
    x[1].neg_()
    y, mean, rstd = ops().layer_norm_forward(x, eps=EPS)   # mean 1 / n, deviation 1: rounded to 11 bits the row itself
    assert torch.equal(y, x) and mean.abs().max() <= 1e-8 and (rstd - 1 / math.sqrt(1 + EPS)).abs().max() <= 1e-6
    dy[0], dy[1] = x[0], 1
    del mean, rstd
    mean, rstd = torch.zeros(2, device="cuda"), torch.tensor([0.5, 1.0], device="cuda")
    dx, dw, db = ops().layer_norm_backward(dy, x, mean, rstd, out=y)
    # row 0: t = x, xh = x / 2, so dx = (x - x / 4) / 2; row 1: t = 1 and xh of mean zero, so nothing is left
    assert (dx[0, 0::2] == 0.375).all() and (dx[0, 1::2] == -0.375).all() and dx[1].abs().max() <= 1e-6
    assert (dw[0::2] == -0.5).all() and (dw[1::2] == 1.5).all()
    assert (db[0::2] == 2).all() and (db[1::2] == 0).all()
    del x, dy, y, dx, dw, db
    torch.cuda.empty_cache()
