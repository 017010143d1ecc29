"""Root-mean-square norm on device tensors against the definition in 64 bits.

Tolerances count roundings of fp32 (u = 2^-24).  A row's sum of squares runs through at most n / 32 + 1 terms of a thread and ten more additions, a square
brings three roundings (the sum with the residual counts twice): its relative error is at most (n / 32 + 14) u, that of 1 / rms half of it and four more.
"""
import math

import pytest

import tatara_b200 as tb

torch = pytest.importorskip("torch")
from op_plain import HALF, TINY, U32  # noqa: E402

pytestmark = pytest.mark.gpu
EPS = 1e-6
TYPES = [torch.float32, torch.float16, torch.bfloat16]
# widths around every change of layout, odd ones among them, and rows beyond the registers (16384 back, 32768 forward)
SIZES = [(1, 1), (3, 2), (37, 8), (5, 31), (41, 64), (70, 72), (129, 128), (50, 136), (129, 256), (64, 257), (40, 512), (33, 520), (9, 777), (70, 1536), (21, 2048), (7, 2056), (6, 4104), (5, 8192),
         (3, 8200), (2, 16384), (3, 16400), (2, 32768), (2, 32776), (300, 20), (2000, 64)]


def ops():
    from tatara_b200 import ops as o
    return o


def make(rows, n, dtype, seed, pad=0, offset=0):
    g = torch.Generator("cuda").manual_seed(seed)
    wide = torch.randn(rows, n + pad + offset, generator=g, device="cuda") * (0.1 + torch.rand(rows, 1, generator=g, device="cuda"))
    return wide.to(dtype)[:, offset:offset + n]


def vector(n, seed):
    return 1 + 0.2 * torch.randn(n, generator=torch.Generator("cuda").manual_seed(seed), device="cuda")


def plain(x, w, r, eps):
    h = x.double() if r is None else x.double() + r.double()
    rstd = 1 / torch.sqrt((h * h).mean(1) + eps)
    y = h * rstd[:, None]
    return y if w is None else y * w.double(), h, rstd


def error(n):
    return U32 * ((n / 32 + 14) / 2 + 4)


def check_forward(x, w, r, got, eps=EPS):
    y, h, rstd = got
    want, hw, rw = plain(x, w, r, eps)
    rel = error(x.shape[1])
    assert ((rstd.double() - rw).abs() <= rel * rw).all()
    assert ((y.double() - want).abs() <= (rel + 3 * U32 + HALF[y.dtype]) * want.abs() * 1.01 + TINY[y.dtype]).all()
    if r is None:
        assert h is x
    else:
        assert ((h.double() - hw).abs() <= (U32 + HALF[h.dtype]) * hw.abs() * 1.01 + TINY[h.dtype]).all()


def check_quantised(x, w, r, group, got, eps=EPS):
    q, scale, h, rstd = got
    want, hw, rw = plain(x, w, r, eps)
    rows, n = x.shape
    group = n if group is None else group
    rel = error(n) + 3 * U32
    assert q.dtype == torch.float8_e4m3fn and scale.shape == (rows, -(-n // group))
    assert ((rstd.double() - rw).abs() <= rel * rw).all()
    column = torch.arange(n, device="cuda") // group
    most = torch.zeros(scale.shape, dtype=torch.float64, device="cuda").index_reduce_(1, column, want.abs(), "amax")
    sw = (most / 448).clamp(min=2.0 ** -126)
    assert ((scale.double() - sw).abs() <= (rel + 2 * U32) * sw).all()
    s = scale.double()[:, column]
    v = want.abs() / s
    # half a step of e4m3: 2^-4 of a normal number, 2^-10 below 2^-6; what the fp32 arithmetic before may be off
    tol = s * torch.maximum(v * 2.0 ** -4, torch.tensor(2.0 ** -10, device="cuda", dtype=torch.float64)) * 1.001 + (rel + 4 * U32) * want.abs()
    assert ((q.double() * s - want).abs() <= tol).all()
    big = torch.zeros_like(most).index_reduce_(1, column, q.double().abs(), "amax")
    assert (big[most > 448 * 2.0 ** -126] == 448).all()
    if r is not None:
        assert ((h.double() - hw).abs() <= (U32 + HALF[h.dtype]) * hw.abs() * 1.01 + TINY[h.dtype]).all()


def check_backward(dy, h, rstd, w, dres, got):
    dx, dw = got
    rows, n = h.shape
    g, r = dy.double(), rstd.double()[:, None]
    xh = h.double() * r
    t = g if w is None else g * w.double()
    want = r * (t - xh * (t * xh).mean(1, keepdim=True))
    tol = U32 * r * (5 * t.abs() + (n / 32 + 17) * xh.abs() * (t * xh).abs().mean(1, keepdim=True))
    if dres is not None:
        want = want + dres.double()
        tol = tol + U32 * want.abs()
    assert ((dx.double() - want).abs() <= tol + HALF[dx.dtype] * want.abs() * 1.01 + TINY[dx.dtype]).all()
    assert ((dw.double() - (g * xh).sum(0)).abs() <= U32 * (rows + 43) * (g * xh).abs().sum(0) + 1e-44).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n", SIZES)
def test_both_directions(rows, n, dtype):
    x, res, dy, dres = (make(rows, n, dtype, rows + n + i) for i in range(4))
    w = vector(n, n)
    for r in (None, res):
        got = ops().rms_norm_forward(x, w, residual=r, eps=EPS)
        check_forward(x, w, r, got)
        check_backward(dy, got[1], got[2], w, dres if r is not None else None, ops().rms_norm_backward(dy, got[1], got[2], w, dresidual=dres if r is not None else None))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n", SIZES)
def test_eight_bits(rows, n, dtype):
    x, res = make(rows, n, dtype, rows + n), make(rows, n, dtype, rows + n + 1)
    w = vector(n, n)
    for group in (None, 32, 64, 128):
        for r in (None, res):
            check_quantised(x, w, r, group, ops().rms_norm_quantised(x, w, residual=r, eps=EPS, group=group))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n,offset", [(50, 512, 0), (50, 512, 1), (17, 1000, 3), (9, 9000, 5), (5, 17000, 8), (1, 40, 2), (33, 2049, 0), (64, 96, 1)])
def test_rows_of_a_wider_buffer(rows, n, offset, dtype):
    x, res, dy, dres = (make(rows, n, dtype, i, 16 if offset == 0 else 13, offset) for i in range(4))
    got = ops().rms_norm_forward(x, residual=res, eps=EPS)
    check_forward(x, None, res, got)
    check_backward(dy, res, got[2], None, dres, ops().rms_norm_backward(dy, res, got[2], dresidual=dres))
    for group in (None, 32, 128):
        check_quantised(x, None, res, group, ops().rms_norm_quantised(x, residual=res, eps=EPS, group=group))
    # results into columns of a wider buffer leave their neighbours alone
    wide, more = torch.full((rows, n + 9), 3.0, dtype=dtype, device="cuda"), torch.full((rows, n + 9), 5.0, dtype=dtype, device="cuda")
    ops().rms_norm_forward(x, residual=res, eps=EPS, out=wide[:, 4:4 + n], residual_out=more[:, 2:2 + n])
    check_forward(x, None, res, (wide[:, 4:4 + n], more[:, 2:2 + n], got[2]))
    assert (wide[:, :4] == 3).all() and (wide[:, 4 + n:] == 3).all() and (more[:, :2] == 5).all() and (more[:, 2 + n:] == 5).all()


@pytest.mark.parametrize("n", [24, 100, 1000, 1001, 5000, 9001, 20000, 33000])
def test_in_place_at_every_length(n):
    x, res, dy, dres = (make(40, n, torch.float32, 31 + i) for i in range(4))
    w = vector(n, 3)
    y, h, rstd = ops().rms_norm_forward(x, w, residual=res, eps=EPS)
    for y_over in ("x", "r"):
        t = {"x": x.clone(), "r": res.clone()}
        got = ops().rms_norm_forward(t["x"], w, residual=t["r"], eps=EPS, out=t[y_over], residual_out=t["r" if y_over == "x" else "x"])
        assert all(torch.equal(a, b) for a, b in zip(got, (y, h, rstd))), y_over
    q = ops().rms_norm_quantised(x, w, residual=res, eps=EPS, group=32)
    r = res.clone()
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(ops().rms_norm_quantised(x, w, residual=r, eps=EPS, group=32, residual_out=r), q))
    want = ops().rms_norm_backward(dy, h, rstd, w, dresidual=dres)
    again = ops().rms_norm_backward(dy, h, rstd, w, dresidual=dres)
    assert all(torch.equal(a, b) for a, b in zip(again, want))
    for same in ("dy", "h", "dres"):
        t = {"dy": dy.clone(), "h": h.clone(), "dres": dres.clone()}
        got = ops().rms_norm_backward(t["dy"], t["h"], rstd, w, dresidual=t["dres"], out=t[same])
        assert all(torch.equal(a, b) for a, b in zip(got, want)), same


def test_the_norm_is_that_of_the_unrounded_sum():
    x = torch.full((4, 64), 1.0, dtype=torch.bfloat16, device="cuda")
    r = torch.full((4, 64), 2.0 ** -9, dtype=torch.bfloat16, device="cuda")
    r[:, ::2] = -(2.0 ** -9)
    y, h, rstd = ops().rms_norm_forward(x, residual=r, eps=0.0)
    assert (h == 1).all()   # both 1 + 2^-9 and 1 - 2^-9 round to 1
    assert ((rstd.double() - 1 / math.sqrt(1 + 2.0 ** -18)).abs() <= error(64)).all()


@pytest.mark.parametrize("n", [8, 100, 256, 1536, 9000, 33000])
def test_rows_whose_squares_leave_fp32(n):
    """Values of 1e25 and of 1e-25 in rows side by side with ordinary ones, and the type's largest."""
    base = make(9, n, torch.float32, n).abs() + 0.5
    factor = torch.tensor([1.0, 1e25, 1e-25, 1e30, 1.0, 1e-30, 1e37, 1e19, 1e-19], device="cuda")
    x = base * factor[:, None]
    w = vector(n, 4)
    for offset in (0, 1):   # rows that start anywhere too
        v = torch.cat([torch.zeros(9, offset, device="cuda"), x], 1)[:, offset:]
        y, h, rstd = ops().rms_norm_forward(v, w, eps=0.0)
        want, _, rw = plain(v, w, None, 0.0)
        rel = error(n) + 2 * U32
        normal = rw > 2.0 ** -126   # below, 1 / rms itself has fewer bits: 2^-149 of it at worst
        off = torch.where(normal, torch.zeros_like(rw), 2.0 ** -149 / rw)
        assert ((rstd.double() - rw).abs() <= (rel + off) * rw).all()
        assert ((y.double() - want).abs() <= (rel + off[:, None] + 4 * U32) * want.abs()).all()
        q, scale, _, _ = ops().rms_norm_quantised(v, w, eps=0.0, group=32)
        assert q.float().isfinite().all() and ((q.float().abs().amax(1) == 448)).all()
    big = torch.full((2, n), torch.finfo(torch.float32).max, device="cuda")
    y, _, rstd = ops().rms_norm_forward(big, eps=EPS)
    assert ((y - 1).abs() <= 2.0 ** -20).all()


def test_rows_of_zeros_and_values_that_are_not_numbers():
    for dtype in TYPES:
        x = make(7, 300, dtype, 3).clone()
        x[2] = 0
        x[3, 7], x[4, 280] = math.inf, math.nan
        y, _, rstd = ops().rms_norm_forward(x, eps=EPS)
        keep = [0, 1, 2, 5, 6]
        want, _, rw = plain(x[keep], None, None, EPS)
        assert ((y[keep].double() - want).abs() <= (error(300) + 3 * U32 + HALF[dtype]) * want.abs() * 1.01 + TINY[dtype]).all() and (y[2] == 0).all()
        assert y[4].isnan().all() and rstd[4].isnan() and y[3, 7].isnan() and rstd[3] == 0 and (y[3, :7] == 0).all()
        q, scale, _, _ = ops().rms_norm_quantised(x, eps=EPS, group=32)
        v = q.float() * scale.repeat_interleave(32, 1)[:, :300]
        assert (v[2] == 0).all() and (scale[2] == 2.0 ** -126).all() and v[4].isnan().all() and v[3, :32].isnan().all() and (v[3, 32:] == 0).all() and v[keep].isfinite().all()
        dx, dw = ops().rms_norm_backward(x[keep], x[keep], rstd[keep])
        assert (dx[2] == 0).all() and dw.isfinite().all()


def test_no_rows():
    x = torch.empty(0, 40, device="cuda")
    y, h, rstd = ops().rms_norm_forward(x, residual=x)
    q, scale, _, _ = ops().rms_norm_quantised(x, group=32)
    dx, dw = ops().rms_norm_backward(x, x, rstd)
    assert y.shape == h.shape == q.shape == dx.shape == (0, 40) and scale.shape == (0, 2) and (dw == 0).all()


@pytest.mark.parametrize("rows,n", [(6, 33), (4, 512)])
def test_gradient_against_differences(rows, n):
    h, dy = make(rows, n, torch.float32, 21), make(rows, n, torch.float32, 22)
    w = vector(n, 5)
    _, _, rstd = ops().rms_norm_forward(h, w, eps=EPS)
    dx, dw = ops().rms_norm_backward(dy, h, rstd, w)
    value = lambda h, w: float((plain(h, w, None, EPS)[0] * dy.double()).sum())  # noqa: E731
    g = torch.Generator("cuda").manual_seed(4)
    e = 1e-5  # central differences in 64 bits: error e^2 of the third derivative, rounding 1e-16 / e
    for at, grad in (("h", dx), ("w", dw)):
        d = torch.randn(grad.shape, generator=g, device="cuda", dtype=torch.float64)
        up, down = ({"h": h.double(), "w": w.double()} for _ in range(2))
        up[at], down[at] = up[at] + e * d, down[at] - e * d
        want = (value(**up) - value(**down)) / (2 * e)
        assert abs(float((grad.double() * d).sum()) - want) <= U32 * (n + rows + 60) * float((grad.double() * d).abs().sum()) + 1e-6


def test_offsets_beyond_32_bits():
    rows, n = 1_100_000, 2048
    x = torch.empty(rows, n, dtype=torch.float16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(1))
    tail, keep = x[-5:].clone(), x[:5].clone()
    q, scale, _, rstd = ops().rms_norm_quantised(x, eps=EPS, group=128)
    tq = ops().rms_norm_quantised(tail, eps=EPS, group=128)
    assert torch.equal(q[-5:].view(torch.uint8), tq[0].view(torch.uint8)) and torch.equal(scale[-5:], tq[1])
    del q, scale
    want = ops().rms_norm_forward(tail, eps=EPS)
    y, _, rstd = ops().rms_norm_forward(x, eps=EPS, out=x)
    assert torch.equal(y[-5:], want[0]) and torch.equal(rstd[-5:], want[2]) and torch.equal(y[:5], ops().rms_norm_forward(keep, eps=EPS)[0])
    dx, dw = ops().rms_norm_backward(y, y, torch.full_like(rstd, 0.5), out=y)
    t = want[0].double()
    ref = 0.5 * (t - t * 0.5 * (t * t * 0.5).mean(1, keepdim=True))
    assert ((dx[-5:].double() - ref).abs() <= HALF[torch.float16] * ref.abs() * 1.01 + U32 * 100 * t.abs() + TINY[torch.float16]).all()


def test_refusals():
    o = ops()
    x, y = torch.zeros(4, 8, device="cuda"), torch.zeros(4, 8, device="cuda")
    v = torch.zeros(4, device="cuda")
    for bad in (lambda: o.rms_norm_forward(x.double()), lambda: o.rms_norm_forward(x.cpu()), lambda: o.rms_norm_forward(x[0]), lambda: o.rms_norm_forward(x.t()),
                lambda: o.rms_norm_forward(x[:1].expand(4, 8)), lambda: o.rms_norm_forward(x, torch.zeros(7, device="cuda")), lambda: o.rms_norm_forward(x, torch.zeros(8)),
                lambda: o.rms_norm_forward(x, eps=-1.0), lambda: o.rms_norm_forward(x, eps=math.nan), lambda: o.rms_norm_forward(x[:, :0]), lambda: o.rms_norm_forward(x, out=x.half()),
                lambda: o.rms_norm_forward(x, residual=x.half()), lambda: o.rms_norm_forward(x, residual=x[:3]), lambda: o.rms_norm_forward(x, residual_out=y),
                lambda: o.rms_norm_forward(x, residual=y, out=x, residual_out=x), lambda: o.rms_norm_forward(x, residual=y, residual_out=y.half()),
                lambda: o.rms_norm_quantised(x, group=16), lambda: o.rms_norm_quantised(x, group=0), lambda: o.rms_norm_quantised(x, group="a"), lambda: o.rms_norm_quantised(x, residual_out=y),
                lambda: o.rms_norm_backward(x[:3], x, v), lambda: o.rms_norm_backward(x.half(), x, v), lambda: o.rms_norm_backward(x, x, v[:3]), lambda: o.rms_norm_backward(x, x, v, dresidual=x[:, :4]),
                lambda: o.rms_norm_backward(None, x, v), lambda: o.rms_norm_backward(x, x, None)):
        with pytest.raises(tb.TrainerError):
            bad()
    rows = torch.zeros(8, 8, device="cuda")
    for bad in (lambda: o.rms_norm_forward(rows[:4], out=rows[1:5]), lambda: o.rms_norm_forward(x, residual=rows[:4], residual_out=rows[1:5]),
                lambda: o.rms_norm_backward(rows[:4], x, v, out=rows[1:5]), lambda: o.rms_norm_backward(x, x, v, dresidual=rows[:4], out=rows[1:5])):
        with pytest.raises(tb.TrainerError, match="overlaps"):
            bad()
    assert torch.equal(o.rms_norm_quantised(x, group=8)[0].float(), x)   # a group of the whole row


@pytest.mark.parametrize("rows,n", [(1, 9), (5, 19), (32, 64), (33, 64), (64, 40), (65, 40), (2, 100), (9, 200), (17, 200), (4, 1000), (5, 1001), (2, 5000), (1, 9000), (2, 20000)])
def test_gradients_of_few_rows(rows, n):
    h, dy = make(rows, n, torch.float32, rows + n), make(rows, n, torch.float32, rows + n + 7)
    w = vector(n, 8)
    rstd = ops().rms_norm_forward(h, w, eps=EPS)[2]
    check_backward(dy, h, rstd, w, None, ops().rms_norm_backward(dy, h, rstd, w))
