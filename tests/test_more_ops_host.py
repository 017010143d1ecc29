"""The entry points of the root-mean-square norm, of rows by expert and of rows by token without a GPU: refused arguments come back as codes and texts before anything
is launched, accepted ones as "no device" where there is none; sizes of workspaces and lists."""
import ctypes as C
import math

import pytest

import tatara_b200 as tb

INVALID, NO_DEVICE = -1, -6
P = 0x10000  # an address that is never read


def lib():
    return tb.load_library()


def err():
    return C.create_string_buffer(300)


def no_gpu():
    return lib().tb_device_count() <= 0


def at(i):
    return P + (1 << 20) * i


def refused(call, cases):
    for kw, text in cases:
        e = err()
        assert call(e, **kw) == INVALID and text in e.value, (kw, e.value)


def forward(e, x=at(0), xs=8, r=at(1), rs=8, w=at(2), eps=1e-6, t=0, rows=4, n=8, y=at(3), ys=8, h=at(4), hs=8, d=at(5)):
    return lib().tb_rms_norm_forward(x, xs, r, rs, w, eps, t, rows, n, y, ys, h, hs, d, None, e, 300)


def quantised(e, x=at(0), xs=40, r=at(1), rs=40, w=at(2), eps=1e-6, t=0, rows=4, n=40, group=32, q=at(3), qs=40, scale=at(6), h=at(4), hs=40, d=at(5)):
    return lib().tb_rms_norm_quantised(x, xs, r, rs, w, eps, t, rows, n, group, q, qs, scale, h, hs, d, None, e, 300)


def test_rms_norm_arguments():
    common = [(dict(x=None), b"NULL"), (dict(t=3), b"type"), (dict(rows=-1), b"rows"), (dict(rows=1 << 31), b"rows"), (dict(n=0), b"n positive"), (dict(eps=-1.0), b"eps"), (dict(eps=math.nan), b"eps"),
              (dict(xs=7), b"stride"), (dict(rs=7), b"stride"), (dict(hs=7), b"stride"), (dict(r=None), b"residual"), (dict(x=P + 2), b"aligned"), (dict(r=at(1) + 1), b"aligned"), (dict(h=at(4) + 2), b"aligned"),
              (dict(w=at(2) + 2), b"aligned"), (dict(d=at(5) + 1), b"aligned")]
    refused(forward, common + [(dict(y=None), b"NULL"), (dict(ys=7), b"stride"), (dict(y=at(3) + 2), b"aligned")])
    refused(quantised, common + [(dict(q=None), b"NULL"), (dict(qs=39), b"stride"), (dict(scale=None), b"NULL"), (dict(scale=at(6) + 2), b"aligned"), (dict(group=0), b"group"), (dict(group=16), b"group"),
                                 (dict(group=-32), b"group"), (dict(group=256), b"group")])
    assert forward(err(), rows=0, x=None, y=None) == 0 and quantised(err(), rows=0, x=None, q=None, scale=None) == 0


def test_rms_norm_overlaps():
    last = 4 * 31
    refused(forward, [(dict(y=at(0) + 4), b"overlaps"), (dict(y=at(1) + last), b"overlaps"), (dict(h=at(0) + 32), b"overlaps"), (dict(h=at(1) - 4), b"overlaps"), (dict(y=at(4)), b"overlaps"),
                      (dict(y=at(4) + 4), b"overlaps"), (dict(w=at(3)), b"overlaps"), (dict(w=at(4) + last), b"overlaps"), (dict(d=at(0)), b"overlaps"), (dict(d=at(1)), b"overlaps"), (dict(d=at(2) + 28), b"overlaps"),
                      (dict(d=at(3) + last), b"overlaps"), (dict(d=at(4)), b"overlaps"), (dict(y=at(0), h=at(0)), b"overlaps")])
    refused(quantised, [(dict(q=at(0)), b"overlaps"), (dict(q=at(1) + 639), b"overlaps"), (dict(q=at(4)), b"overlaps"), (dict(h=at(0) + 4), b"overlaps"), (dict(scale=at(0)), b"overlaps"),
                        (dict(scale=at(3) + 156), b"overlaps"), (dict(scale=at(5) + 12), b"overlaps"), (dict(d=at(6) + 28), b"overlaps"), (dict(w=at(3) + 156), b"overlaps"), (dict(scale=at(2) + 4), b"overlaps")])
    if no_gpu():
        for kw in (dict(), dict(y=at(0)), dict(y=at(1)), dict(h=at(0)), dict(h=at(1)), dict(y=at(0), h=at(1)), dict(y=at(1), h=at(0)), dict(r=at(0)), dict(r=None, h=None), dict(h=None), dict(d=None), dict(w=None),
                   dict(xs=24, rs=24, ys=24, hs=24, y=at(0) + 32, h=at(0) + 64)):
            e = err()
            assert forward(e, **kw) == NO_DEVICE, (kw, e.value)
        for kw in (dict(), dict(h=at(0)), dict(h=at(1)), dict(r=None, h=None), dict(group=40), dict(group=128), dict(scale=at(6) - 4), dict(q=at(3) + 1)):
            e = err()
            assert quantised(e, **kw) == NO_DEVICE, (kw, e.value)


def test_rms_norm_backward_arguments():
    need = lib().tb_rms_norm_backward_workspace(4, 8)
    assert need > 0 and lib().tb_rms_norm_backward_workspace(0, 8) > 0
    assert lib().tb_rms_norm_backward_workspace(-1, 8) == lib().tb_rms_norm_backward_workspace(4, 0) == lib().tb_rms_norm_backward_workspace(1 << 31, 8) == INVALID

    def call(e, dy=at(0), ds=8, h=at(1), hs=8, rstd=at(2), w=at(3), dres=at(4), rs=8, t=0, rows=4, n=8, dx=at(5), xs=8, dw=at(6), work=at(7), wb=need):
        return lib().tb_rms_norm_backward(dy, ds, h, hs, rstd, w, dres, rs, t, rows, n, dx, xs, dw, work, wb, None, e, 300)

    refused(call, [(dict(dy=None), b"NULL"), (dict(h=None), b"NULL"), (dict(rstd=None), b"NULL"), (dict(dx=None), b"NULL"), (dict(t=-1), b"type"), (dict(rows=-1), b"rows"), (dict(n=0), b"positive"),
                   (dict(ds=7), b"stride"), (dict(hs=7), b"stride"), (dict(rs=7), b"stride"), (dict(xs=7), b"stride"), (dict(wb=need - 1), b"workspace"), (dict(work=None), b"workspace"), (dict(work=at(7) + 4), b"workspace"),
                   (dict(dy=at(0) + 2), b"aligned"), (dict(dres=at(4) + 2), b"aligned"), (dict(rstd=at(2) + 2), b"aligned"), (dict(dw=at(6) + 2), b"aligned"), (dict(dx=at(0) + 4), b"overlaps"),
                   (dict(dx=at(1) + 32), b"overlaps"), (dict(dx=at(4) + 124), b"overlaps"), (dict(dw=at(0)), b"overlaps"), (dict(dw=at(1) + 124), b"overlaps"), (dict(dw=at(4)), b"overlaps"), (dict(dw=at(5)), b"overlaps"),
                   (dict(dw=at(2)), b"overlaps"), (dict(dw=at(3) + 28), b"overlaps"), (dict(dx=at(2)), b"overlaps"), (dict(dx=at(3)), b"overlaps")])
    if no_gpu():
        for kw in (dict(), dict(dx=at(0)), dict(dx=at(1)), dict(dx=at(4)), dict(dres=None), dict(w=None), dict(dw=None, work=None, wb=0)):
            e = err()
            assert call(e, **kw) == NO_DEVICE, (kw, e.value)


def test_sizes_of_orders():
    slots = lib().tb_expert_slots
    assert slots(0, 2, 9, 1) == 0 and slots(10, 2, 9, 1) == 20 and slots(1, 1, 1024, 128) == 128 and slots(10, 2, 9, 16) == (20 + 9 * 15) // 16 * 16
    for bad in ((-1, 2, 9, 1), (10, 0, 9, 1), (10, 17, 9, 1), (10, 2, 0, 1), (10, 2, 1025, 1), (10, 2, 9, 0), (1 << 31, 1, 9, 1), (1 << 30, 2, 9, 1), (10, 2, 9, 1 << 30)):
        assert slots(*bad) == INVALID
    for rows, k, experts in ((1, 1, 1), (100, 2, 9), (65536, 2, 9), (65536, 8, 1024), (1 << 27, 15, 1024)):
        need = lib().tb_expert_order_workspace(rows, k, experts)
        assert 0 <= need < 1 << 26 and need % 4 == 0
    assert lib().tb_expert_order_workspace(10, 17, 9) == INVALID


def test_order_arguments():
    rows, k, experts, align = 3000, 2, 9, 4
    slots, need = lib().tb_expert_slots(rows, k, experts, align), lib().tb_expert_order_workspace(rows, k, experts)
    assert need > 0

    def call(e, ix=at(0), rows=rows, k=k, experts=experts, align=align, po=at(1), so=at(2), slots=slots, of=at(3), work=at(4), wb=need):
        return lib().tb_expert_order(ix, rows, k, experts, align, po, so, slots, of, work, wb, None, e, 300)

    refused(call, [(dict(ix=None), b"NULL"), (dict(po=None), b"NULL"), (dict(so=None), b"NULL"), (dict(of=None), b"NULL"), (dict(k=0), b"k must"), (dict(k=17), b"k must"), (dict(experts=0), b"experts"),
                   (dict(experts=1025), b"experts"), (dict(align=0), b"align"), (dict(rows=-1), b"rows"), (dict(rows=1 << 31), b"rows"), (dict(slots=slots - 1), b"slots"), (dict(wb=need - 1), b"workspace"),
                   (dict(work=None), b"workspace"), (dict(work=at(4) + 2), b"workspace"), (dict(ix=at(0) + 2), b"aligned"), (dict(po=at(1) + 1), b"aligned"), (dict(so=at(2) + 2), b"aligned"), (dict(of=at(3) + 2), b"aligned"),
                   (dict(po=at(0)), b"overlaps"), (dict(so=at(1) - 4), b"overlaps"), (dict(of=at(2) + 4 * (slots - 1)), b"overlaps"), (dict(of=at(0)), b"overlaps")])
    if no_gpu():
        e = err()
        assert call(e) == NO_DEVICE and e.value


def test_row_arguments():
    def dispatch(e, x=at(0), xs=8, t=0, rows=6, n=8, k=2, po=at(1), so=at(2), slots=12, out=at(3), os=8):
        return lib().tb_dispatch_forward(x, xs, t, rows, n, k, po, so, slots, out, os, None, e, 300)

    def combine(e, y=at(0), ys=8, t=0, slots=12, rows=6, n=8, k=2, po=at(1), g=at(2), out=at(3), os=8):
        return lib().tb_combine_forward(y, ys, t, slots, rows, n, k, po, g, out, os, None, e, 300)

    def back(e, d=at(0), ds=8, y=at(4), ys=8, t=0, slots=12, rows=6, n=8, k=2, po=at(1), so=at(2), g=at(5), dy=at(3), dys=8, dg=at(6)):
        return lib().tb_combine_backward(d, ds, y, ys, t, slots, rows, n, k, po, so, g, dy, dys, dg, None, e, 300)

    common = [(dict(t=7), b"type"), (dict(k=0), b"k must"), (dict(k=17), b"k must"), (dict(rows=-1), b"rows"), (dict(rows=1 << 31), b"rows"), (dict(rows=1 << 30), b"rows"), (dict(slots=-1), b"slots"), (dict(slots=1 << 31), b"slots"),
              (dict(n=0), b"n must"), (dict(n=(1 << 30) + 1), b"n must"), (dict(po=None), b"NULL"), (dict(po=at(1) + 2), b"aligned")]
    refused(dispatch, common + [(dict(x=None), b"NULL"), (dict(out=None), b"NULL"), (dict(so=None), b"NULL"), (dict(xs=7), b"stride"), (dict(os=7), b"stride"), (dict(x=at(0) + 2), b"aligned"), (dict(out=at(3) + 1), b"aligned"),
                                (dict(out=at(0)), b"overlaps"), (dict(out=at(0) - 380), b"overlaps"), (dict(out=at(1) + 44), b"overlaps"), (dict(out=at(2)), b"overlaps"), (dict(xs=24, os=24, out=at(0) + 32), b"overlaps")])
    refused(combine, common + [(dict(y=None), b"NULL"), (dict(out=None), b"NULL"), (dict(ys=7), b"stride"), (dict(os=7), b"stride"), (dict(y=at(0) + 2), b"aligned"), (dict(g=at(2) + 2), b"aligned"), (dict(out=at(0)), b"overlaps"),
                               (dict(out=at(1)), b"overlaps"), (dict(out=at(2) + 44), b"overlaps")])
    refused(back, common + [(dict(d=None), b"NULL"), (dict(y=None), b"NULL"), (dict(so=None), b"NULL"), (dict(g=None), b"NULL"), (dict(dy=None), b"NULL"), (dict(dg=None), b"NULL"), (dict(ds=7), b"stride"), (dict(ys=7), b"stride"),
                            (dict(dys=7), b"stride"), (dict(dg=at(6) + 2), b"aligned"), (dict(dy=at(0)), b"overlaps"), (dict(dy=at(4)), b"overlaps"), (dict(dg=at(5)), b"overlaps"), (dict(dg=at(3) + 380), b"overlaps"),
                            (dict(dg=at(0)), b"overlaps")])
    for call in (dispatch, combine, back):
        assert call(err(), rows=0, slots=0, po=None) == 0
    if no_gpu():
        assert dispatch(err()) == combine(err()) == combine(err(), g=None) == back(err()) == NO_DEVICE


def test_embedding_arguments():
    def call(e, to=at(0), tb_=8, count=10, table=at(1), ts=8, t=0, rows=20, n=8, out=at(2), os=8):
        return lib().tb_embedding_forward(to, tb_, count, table, ts, t, rows, n, 1.0, out, os, None, e, 300)

    need = lib().tb_embedding_backward_workspace(5000, 20, 8)
    assert need > 0 and lib().tb_embedding_backward_workspace(10, 20, 8) == 0   # few tokens and a small table need none
    assert lib().tb_embedding_backward_workspace(0, 1, 1) > 0
    for bad in ((-1, 20, 8), (10, 0, 8), (10, 20, 0), (1 << 31, 20, 8), (10, 1 << 31, 8), (10, 20, (1 << 30) + 1), ((1 << 31) - 1, 20, 8)):
        assert lib().tb_embedding_backward_workspace(*bad) == INVALID
    assert lib().tb_embedding_backward_workspace((1 << 31) - 1024, (1 << 31) - 1, 1) > 16 * ((1 << 31) - 1024)

    def back(e, dy=at(1), ds=8, t=0, to=at(0), tb_=8, count=5000, rows=20, n=8, out=at(2), os=8, ot=0, work=at(3), wb=need):
        return lib().tb_embedding_backward(dy, ds, t, to, tb_, count, rows, n, 1.0, out, os, ot, work, wb, None, e, 300)

    common = [(dict(t=5), b"type"), (dict(tb_=2), b"token_bytes"), (dict(count=-1), b"count"), (dict(count=1 << 31), b"count"), (dict(rows=0), b"rows"), (dict(rows=1 << 31), b"rows"), (dict(n=0), b"n must"), (dict(to=None), b"NULL"),
              (dict(to=at(0) + 4), b"aligned"), (dict(out=None), b"NULL"), (dict(os=7), b"stride"), (dict(out=at(2) + 2), b"aligned"), (dict(out=at(0) + 76), b"overlaps"), (dict(out=at(1)), b"overlaps")]
    refused(call, common + [(dict(table=None), b"NULL"), (dict(ts=7), b"stride"), (dict(table=at(1) + 2), b"aligned")])
    refused(back, common + [(dict(dy=None), b"NULL"), (dict(ds=7), b"stride"), (dict(dy=at(1) + 2), b"aligned"), (dict(ot=1), b"dtable_type"), (dict(work=None), b"workspace"), (dict(wb=need - 1), b"workspace"),
                            (dict(work=at(3) + 16), b"workspace")])
    assert call(err(), count=0, to=None, out=None) == 0
    if no_gpu():
        assert call(err()) == call(err(), tb_=4, to=at(0) + 4) == back(err()) == back(err(), t=1, ot=1) == back(err(), t=2, ot=0) == back(err(), count=0, dy=None, to=None) == NO_DEVICE


def test_torch_binding_refuses_host_tensors():
    torch = pytest.importorskip("torch")
    from tatara_b200 import ops
    x, index = torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int32)
    order = ops.Order(index, index.view(-1), index[0])
    for bad in (lambda: ops.rms_norm_forward(x), lambda: ops.rms_norm_quantised(x), lambda: ops.rms_norm_backward(x, x, x[:, 0]), lambda: ops.expert_order(index, 3), lambda: ops.dispatch_forward(x, order),
                lambda: ops.dispatch_backward(x, order), lambda: ops.combine_forward(x, order, x[:, :2]), lambda: ops.combine_backward(x, x, order, x[:, :2]), lambda: ops.embedding_forward(index, x),
                lambda: ops.embedding_backward(x, index[:, 0], 3)):
        with pytest.raises(tb.TrainerError, match="CUDA tensor"):
            bad()
