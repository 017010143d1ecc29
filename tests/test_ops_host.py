"""The operators' entry points without a GPU: refused arguments come back as codes and texts before anything is launched, accepted ones as
"no device" where there is none; workspace sizes; the torch binding refuses host tensors."""
import ctypes as C
import math

import pytest

import tatara_b200 as tb
from tatara_b200 import _lib as L

INVALID, NO_DEVICE = -1, -6
P = 0x10000  # an address that is never read: arguments are refused, or the launch fails, before it could be


def lib():
    return tb.load_library()


def err():
    return C.create_string_buffer(200)


def no_gpu():
    return lib().tb_device_count() <= 0


def muon(**kw):
    v = dict(struct_size=C.sizeof(L.Muon), steps=5, nesterov=1, a=3.4445, b=-4.775, c=2.0315, eps=1e-7, lr=0.1, beta=0.9, weight_decay=0.0, scale=1.0, clip=math.inf)
    v.update(kw)
    return L.Muon(**v)


COEF = (C.c_float * 3)(3.4445, -4.775, 2.0315)


def test_layer_norm_arguments():
    f = lambda x=P, xs=8, w=None, b=None, eps=1e-5, t=0, rows=4, n=8, y=P, ys=8: lib().tb_layer_norm_forward(x, xs, w, b, eps, t, rows, n, y, ys, None, None, None, e, 200)  # noqa: E731
    for kw, text in ((dict(x=None), b"NULL"), (dict(y=None), b"NULL"), (dict(xs=7), b"stride"), (dict(ys=7), b"stride"), (dict(t=3), b"type"), (dict(t=-1), b"type"),
                     (dict(rows=-1), b"rows"), (dict(rows=1 << 31), b"rows"), (dict(n=0), b"n positive"), (dict(eps=-1.0), b"eps"), (dict(eps=math.nan), b"eps"),
                     (dict(x=P + 2), b"aligned"), (dict(w=P + 2), b"aligned"), (dict(x=P + 1, t=1), b"aligned")):
        e = err()
        assert f(**kw) == INVALID and text in e.value, (kw, e.value)
    e = err()
    assert f(rows=0, x=None, y=None) == 0 and e.value == b""   # nothing to do
    g = lambda wb, **kw: lib().tb_layer_norm_backward(kw.get("dy", P), 8, P, 8, P, kw.get("rstd", P), None, 0, 4, 8, P, 8, kw.get("dw", P), P, kw.get("work", P), wb, None, e, 200)  # noqa: E731
    need = lib().tb_layer_norm_backward_workspace(4, 8)
    assert need > 0
    for call in (lambda: g(need - 1), lambda: g(need, work=None), lambda: g(need, work=P + 4), lambda: g(need, dy=None), lambda: g(need, rstd=None)):
        e = err()
        assert call() == INVALID and e.value
    assert lib().tb_layer_norm_forward(None, 8, None, None, 1e-5, 0, 4, 8, P, 8, None, None, None, None, 0) == INVALID   # no text wanted


def test_results_that_overlap_an_input_in_part():
    f = lambda x, xs, y, ys, rows=4: lib().tb_layer_norm_forward(x, xs, None, None, 1e-5, 0, rows, 8, y, ys, None, None, None, e, 200)  # noqa: E731
    for x, xs, y, ys in ((P, 8, P + 4, 8), (P, 8, P + 32, 8), (P + 96, 8, P, 8), (P, 16, P + 28, 16), (P, 16, P + 36, 16), (P, 8, P, 16), (P, 16, P + 32, 8)):
        e = err()
        assert f(x, xs, y, ys) == INVALID and b"overlaps" in e.value, (x, xs, y, ys)
    if no_gpu():  # the same memory, memory that follows, other columns of the same rows, rows in between
        for x, xs, y, ys in ((P, 8, P, 8), (P, 8, P + 128, 8), (P + 128, 8, P, 8), (P, 16, P + 32, 16), (P + 32, 16, P, 16), (P, 24, P + 40, 24), (P, 9, P + 4 * 35, 16)):
            e = err()
            assert f(x, xs, y, ys) == NO_DEVICE, (x, xs, y, ys, e.value)
        assert f(P, 8, P, 16, rows=1) == NO_DEVICE
    need = lib().tb_layer_norm_backward_workspace(4, 8)
    g = lambda dy, x, dx: lib().tb_layer_norm_backward(dy, 8, x, 8, P, P, None, 0, 4, 8, dx, 8, None, None, P, need, None, e, 200)  # noqa: E731
    for args in ((P, P + 4096, P + 4), (P + 4096, P, P + 64)):
        e = err()
        assert g(*args) == INVALID and b"overlaps" in e.value
    e = err()
    assert lib().tb_route_backward(P, 9, 0, 100, 9, 2, 1, None, P, P, P, P, P, P, P + 4, 9, None, e, 200) == INVALID and b"overlaps" in e.value
    h = lambda x, xb, out, ob, b=2: lib().tb_orthogonalise(x, xb, 8, 0, b, 4, 8, 5, COEF, 1e-7, out, ob, 8, None, 0, None, e, 200)  # noqa: E731
    for args in ((P, 32, P + 4, 32), (P, 32, P + 128, 32), (P, 32, P, 64)):
        e = err()
        assert h(*args) == INVALID and b"overlaps" in e.value, args


def test_route_arguments():
    need = lib().tb_route_forward_workspace(100, 9)
    assert need > 0 and lib().tb_route_forward_workspace(0, 1) > 0
    f = lambda x=P, s=9, t=0, rows=100, e_=9, k=2, ix=P, work=P, wb=need: lib().tb_route_forward(x, s, t, rows, e_, k, 1, None, ix, P, P, P, P, P, work, wb, None, e, 200)  # noqa: E731
    for kw, text in ((dict(x=None), b"NULL"), (dict(ix=None), b"NULL"), (dict(s=8), b"stride"), (dict(t=9), b"type"), (dict(e_=0), b"experts"), (dict(e_=1025, s=1025), b"experts"),
                     (dict(k=0), b"k must"), (dict(k=10), b"k must"), (dict(k=17, e_=64, s=64), b"k must"), (dict(rows=-1), b"rows"), (dict(rows=1 << 31), b"rows"),
                     (dict(wb=need - 1), b"workspace"), (dict(work=None), b"workspace"), (dict(x=P + 1), b"aligned")):
        e = err()
        assert f(**kw) == INVALID and text in e.value, (kw, e.value)
    for bad in ((-1, 9), (5, 0), (5, 1025)):
        assert lib().tb_route_forward_workspace(*bad) == INVALID
    e = err()
    assert lib().tb_route_backward(P, 9, 0, 100, 9, 2, 1, None, None, P, P, P, P, P, P, 9, None, e, 200) == INVALID
    assert lib().tb_route_backward(P, 9, 0, 100, 9, 2, 1, None, P, P, P, P, P, P, P, 8, None, e, 200) == INVALID
    assert lib().tb_route_backward(None, 9, 0, 0, 9, 2, 1, None, None, None, None, None, None, None, None, 9, None, e, 200) == 0


def test_orthogonalise_arguments():
    need = lib().tb_orthogonalise_workspace(0, 2, 100, 200)
    assert need > 0 and need % 128 == 0 and lib().tb_orthogonalise_workspace(0, 9, 16, 1536) == 0   # short sides of up to 64 need none
    assert lib().tb_orthogonalise_workspace(2, 2, 100, 200) < need                                  # one limb, not two
    f = lambda x=P, xb=20000, xs=200, t=0, b=2, r=100, c=200, steps=5, co=COEF, eps=1e-7, out=P, ob=20000, os=200, work=P, wb=need: lib().tb_orthogonalise(  # noqa: E731
        x, xb, xs, t, b, r, c, steps, co, eps, out, ob, os, work, wb, None, e, 200)
    bad = lambda *v: (C.c_float * 3)(*v)  # noqa: E731
    for kw, text in ((dict(x=None), b"NULL"), (dict(out=None), b"NULL"), (dict(xs=199), b"strides"), (dict(os=199), b"strides"), (dict(xb=19999), b"overlap"), (dict(ob=19999), b"overlap"),
                     (dict(t=5), b"type"), (dict(b=-1), b"batch"), (dict(b=65536), b"batch"), (dict(r=0), b"positive"), (dict(steps=0), b"steps"), (dict(steps=33), b"steps"),
                     (dict(co=None), b"coefficients"), (dict(co=bad(8, 0, 0)), b"coefficients"), (dict(co=bad(math.nan, 0, 0)), b"coefficients"), (dict(co=bad(1, 40, 0)), b"coefficients"),
                     (dict(eps=-1.0), b"eps"), (dict(work=None), b"workspace"), (dict(wb=need - 1), b"workspace"), (dict(work=P + 64), b"workspace"), (dict(x=P + 2), b"aligned")):
        e = err()
        assert f(**kw) == INVALID and text in e.value, (kw, e.value)
    for v in ((9, 1, 1, 1), (0, -1, 1, 1), (0, 1, 0, 1), (0, 1, 1, 0)):
        assert lib().tb_orthogonalise_workspace(*v) == INVALID
    e = err()
    assert f(b=0, x=None, out=None) == 0


def test_coefficients_that_keep_the_range_are_accepted():
    # the quintic of the defaults over many steps, a convergent quintic, the cubic: what stops these calls is the missing workspace, not the coefficients
    e = err()
    for c in ((3.4445, -4.775, 2.0315), (1.875, -1.25, 0.375), (1.5, -0.5, 0.0), (1.0, 0.0, 0.0)):
        assert lib().tb_orthogonalise(P, 20000, 200, 0, 2, 100, 200, 32, (C.c_float * 3)(*c), 1e-7, P, 20000, 200, None, 0, None, e, 200) == INVALID
        assert b"workspace" in e.value, (c, e.value)


def test_muon_arguments():
    need = lib().tb_muon_step_workspace(2, 100, 200)
    size = 4 * 2 * 100 * 200
    w, m, g = P, P + size, P + 2 * size
    work = P + (1 << 30)
    f = lambda cfg=None, w=w, m=m, g=g, t=0, wo=w, mo=m, wb=need: lib().tb_muon_step(C.byref(cfg or muon()), w, m, g, t, 2, 100, 200, wo, mo, work, wb, None, e, 200)  # noqa: E731
    for kw, text in ((dict(cfg=muon(struct_size=8)), b"size"), (dict(cfg=muon(steps=0)), b"steps"), (dict(cfg=muon(clip=0.0)), b"clip"), (dict(cfg=muon(clip=math.nan)), b"clip"),
                     (dict(cfg=muon(eps=-1.0)), b"eps"), (dict(w=None), b"NULL"), (dict(m=None), b"NULL"), (dict(g=None), b"NULL"), (dict(wo=None), b"NULL"), (dict(t=4), b"type"),
                     (dict(wo=m), b"overlaps"), (dict(mo=w), b"overlaps"), (dict(wo=g), b"overlaps"), (dict(mo=g), b"overlaps"), (dict(wo=w + 4), b"overlaps"), (dict(g=m), b"overlaps"),
                     (dict(w=w + 2), b"aligned"), (dict(wb=need - 1), b"workspace")):
        e = err()
        assert f(**kw) == INVALID and text in e.value, (kw, e.value)
    e = err()
    assert lib().tb_muon_step(None, w, m, g, 0, 2, 100, 200, w, m, work, need, None, e, 200) == INVALID


@pytest.mark.skipif("not no_gpu()", reason="a device is present")
def test_no_device_is_an_error_and_not_a_crash():
    e = err()
    assert lib().tb_layer_norm_forward(P, 8, None, None, 1e-5, 0, 4, 8, P, 8, None, None, None, e, 200) == NO_DEVICE and e.value
    assert lib().tb_orthogonalise(P, 0, 8, 0, 1, 8, 8, 5, COEF, 1e-7, P, 0, 8, None, 0, None, e, 200) == NO_DEVICE and e.value


def test_torch_binding_refuses_host_tensors():
    torch = pytest.importorskip("torch")
    from tatara_b200 import ops
    x = torch.zeros(4, 8)
    for bad in (lambda: ops.layer_norm_forward(x), lambda: ops.layer_norm_forward(None), lambda: ops.route_forward(x, 2), lambda: ops.orthogonalise(x),
                lambda: ops.muon_step(x, x, x, lr=0.1), lambda: ops.layer_norm_backward(x, x, x, x)):
        with pytest.raises(tb.TrainerError, match="CUDA tensor"):
            bad()


@pytest.mark.parametrize("type_,limbs", [(0, 2), (1, 2), (2, 1)])
def test_workspaces_of_the_longest_matrices(type_, limbs):
    """What is derived from sides near 2^31 does not wrap: two X of padded tiles, A and Q at least."""
    most = 2 ** 31 - 1
    for rows, cols in ((65, most), (most, 65), (65, most - 255), (500, most), (2 ** 20, 2 ** 20)):
        n, m = min(rows, cols), max(rows, cols)
        need = lib().tb_orthogonalise_workspace(type_, 1, rows, cols)
        assert need >= 2 * 2 * limbs * (n * m + n * n), (rows, cols)
        assert need <= 2 * 2 * limbs * ((n + 255) * (m + 255) + (n + 255) ** 2) + 8 * 65536 * 128 + 8192
        e = err()
        assert lib().tb_orthogonalise(P, 0, cols, type_, 1, rows, cols, 5, COEF, 1e-7, P, 0, cols, P, need - 1, None, e, 200) == INVALID and b"workspace" in e.value
    assert lib().tb_orthogonalise_workspace(type_, 1, 64, most) == 0
    for batch, rows, cols in ((1, most, most), (2, 2 ** 20, 2 ** 20), (65535, 2 ** 20, 64), (1, 2 ** 20 + 1, 2 ** 20)):
        assert lib().tb_orthogonalise_workspace(type_, batch, rows, cols) == INVALID and lib().tb_muon_step_workspace(batch, rows, cols) == INVALID
        e = err()
        assert lib().tb_orthogonalise(P, rows * cols, cols, type_, batch, rows, cols, 5, COEF, 1e-7, P, rows * cols, cols, P, 1 << 62, None, e, 200) == INVALID and b"2^40" in e.value


def test_every_tensor_has_to_be_aligned_to_its_elements():
    """A vector at an odd address would be a misaligned access on the device."""
    at = lambda i: P + 4096 * i  # noqa: E731
    for bad in ("mean", "rstd"):
        for step in (1, 2):
            v = {"mean": at(2), "rstd": at(3)}
            v[bad] += step
            e = err()
            assert lib().tb_layer_norm_forward(at(0), 8, None, None, 1e-5, 1, 4, 8, at(1), 8, v["mean"], v["rstd"], None, e, 200) == INVALID and b"aligned" in e.value, (bad, e.value)
    need = lib().tb_layer_norm_backward_workspace(4, 8)
    for bad in ("mean", "rstd", "weight", "dweight", "dbias"):
        v = {"mean": at(2), "rstd": at(3), "weight": at(4), "dweight": at(5), "dbias": at(6)}
        v[bad] += 2
        e = err()
        assert lib().tb_layer_norm_backward(at(0), 8, at(1), 8, v["mean"], v["rstd"], v["weight"], 1, 4, 8, at(7), 8, v["dweight"], v["dbias"], at(8), need, None, e, 200) == INVALID
        assert b"aligned" in e.value, bad
    need = lib().tb_route_forward_workspace(100, 9)
    for i in range(6):
        v = [at(1 + j) + (2 if j == i else 0) for j in range(6)]
        e = err()
        assert lib().tb_route_forward(at(0), 9, 0, 100, 9, 2, 1, None, *v, at(9), need, None, e, 200) == INVALID and b"aligned" in e.value, i
        e = err()
        index, gate, dgate, counts, n, dlosses = v
        assert lib().tb_route_backward(at(0), 9, 0, 100, 9, 2, 1, None, index, gate, dgate, counts, n, dlosses, at(9), 9, None, e, 200) == INVALID and b"aligned" in e.value, i


def test_results_that_overlap_vectors():
    """mean over the weight, dx over rstd, ..: refused as far as an element is shared, and no further."""
    at = lambda i: P + 65536 * i  # noqa: E731
    rows, n = 4, 8
    fine = NO_DEVICE

    def forward(stride=n, **kw):
        v = dict(x=at(0), y=at(1), w=at(2), b=at(3), mean=at(4), rstd=at(5))
        v.update(kw)
        e = err()
        return lib().tb_layer_norm_forward(v["x"], stride, v["w"], v["b"], 1e-5, 0, rows, n, v["y"], stride, v["mean"], v["rstd"], None, e, 200), e.value

    last = 4 * (rows * n - 1)
    for kw in (dict(w=at(1)), dict(b=at(1) + last), dict(mean=at(1) + last), dict(rstd=at(0)), dict(mean=at(2) + 28), dict(rstd=at(3)), dict(mean=at(5) - 12), dict(w=at(1) - 28)):
        rc, text = forward(**kw)
        assert rc == INVALID and b"overlaps" in text, kw
    need = lib().tb_layer_norm_backward_workspace(rows, n)

    def backward(stride=n, **kw):
        v = dict(dy=at(0), x=at(1), dx=at(2), mean=at(3), rstd=at(4), w=at(5), dw=at(6), db=at(7))
        v.update(kw)
        e = err()
        return lib().tb_layer_norm_backward(v["dy"], stride, v["x"], stride, v["mean"], v["rstd"], v["w"], 0, rows, n, v["dx"], stride, v["dw"], v["db"], at(8), need, None, e, 200), e.value

    for kw in (dict(w=at(2)), dict(mean=at(2) + last), dict(rstd=at(2)), dict(dw=at(2)), dict(db=at(2) + last), dict(dw=at(0)), dict(db=at(1)), dict(dw=at(5)), dict(db=at(3) + 12), dict(dw=at(4)),
               dict(db=at(6) + 28)):
        rc, text = backward(**kw)
        assert rc == INVALID and b"overlaps" in text, kw
    routes = lib().tb_route_forward_workspace(100, 9)
    names = ("index", "gate", "counts", "n", "mean", "losses")

    def route(**kw):
        v = dict(x=at(0), mask=at(1), **{q: at(2 + i) for i, q in enumerate(names)})
        v.update(kw)
        e = err()
        return lib().tb_route_forward(v["x"], 9, 0, 100, 9, 2, 1, v["mask"], *[v[q] for q in names], at(9), routes, None, e, 200), e.value

    ends = {"x": (0, 3596), "mask": (1, 96), "index": (2, 796), "gate": (3, 796), "counts": (4, 32), "n": (5, 0), "mean": (6, 32), "losses": (7, 4)}
    for a in names:
        for b, (i, end) in ends.items():
            if a != b:
                rc, text = route(**{a: at(i) + end})
                assert rc == INVALID and b"overlaps" in text, (a, b)

    def route_back(**kw):
        v = dict(mask=at(1), index=at(2), gate=at(3), counts=at(4), n=at(5), dgate=at(6), dlosses=at(7), d=at(8))
        v.update(kw)
        e = err()
        return lib().tb_route_backward(at(0), 9, 0, 100, 9, 2, 1, v["mask"], v["index"], v["gate"], v["dgate"], v["counts"], v["n"], v["dlosses"], v["d"], 9, None, e, 200), e.value

    for q in ("mask", "index", "gate", "counts", "n", "dgate", "dlosses"):
        for off in (0, 3596):
            rc, text = route_back(**{q: at(8) + off})
            assert rc == INVALID and b"overlaps" in text, (q, off)
    if no_gpu():  # side by side, and in the gaps between the rows of a wider buffer
        gap = dict(stride=3 * n)
        assert forward()[0] == backward()[0] == route()[0] == route_back()[0] == fine
        assert forward(w=at(1) + 4 * rows * n, mean=at(1) - 16, b=at(1) - 48)[0] == fine
        assert forward(w=at(1) + 32, b=at(1) + 96 + 64, mean=at(0) + 32, rstd=at(0) + 48, **gap)[0] == fine
        assert backward(w=at(2) + 32, dw=at(0) + 64, db=at(1) + 96 + 32, mean=at(2) + 192 + 80, **gap)[0] == fine
        assert forward(y=at(0))[0] == backward(dx=at(0))[0] == backward(dx=at(1))[0] == route_back(d=at(0))[0] == fine
