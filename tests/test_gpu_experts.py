"""Rows by expert and back, on device tensors: the order exactly against a loop, rows against the definition in 64 bits.

Tolerances count roundings of fp32 (u = 2^-24): a sum over k choices runs through k products added in a row, (k + 1) u of the sum of magnitudes; a dot product's thread adds at
most n / 32 + 1 products and ten more sums follow.
"""
import ctypes as C
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


def choices(rows, k, experts, seed, missing=0.0):
    g = torch.Generator().manual_seed(seed)
    index = torch.randint(0, experts, (rows, k), generator=g, dtype=torch.int32)   # an expert may be there twice
    index[torch.rand(rows, k, generator=g) < missing] = -1
    return index


def plain_order(index, experts, align):
    """Entry by entry, as the definition reads."""
    rows, k = index.shape
    lists = [[] for _ in range(experts)]
    for i, e in enumerate(index.flatten().tolist()):
        if 0 <= e < experts:
            lists[e].append(i)
    slots = (rows * k + min(experts, rows * k) * (align - 1)) // align * align
    position, source, offsets = [-1] * (rows * k), [-1] * slots, [0]
    for entries in lists:
        for j, i in enumerate(entries):
            position[i], source[offsets[-1] + j] = offsets[-1] + j, i
        offsets.append(offsets[-1] + -(-len(entries) // align) * align)
    return torch.tensor(position, dtype=torch.int32).view(rows, k), torch.tensor(source, dtype=torch.int32), torch.tensor(offsets, dtype=torch.int32)


# a block's worth and less, more blocks with and without a launch that adds up their counts, every number of keys around the tables' bounds
@pytest.mark.parametrize("rows,k,experts", [(0, 2, 9), (1, 1, 1), (5, 3, 2), (200, 2, 9), (31, 16, 1024), (1024, 4, 64), (4096, 1, 9), (4097, 1, 9), (2049, 2, 65), (3000, 8, 256), (5000, 16, 1000),
                                            (70001, 2, 9), (20000, 8, 512), (60000, 8, 1024), (100000, 1, 1)])
@pytest.mark.parametrize("align", [1, 16, 100])
def test_order(rows, k, experts, align):
    index = choices(rows, k, experts, rows + k, 0.1 if rows % 2 else 0.0)
    if rows > 100:
        index[50:90] = index[50, 0]        # a run of one expert
        index[7, 0], index[8, 0], index[9, 0] = experts, 2 ** 31 - 1, -2 ** 31   # outside
    want = plain_order(index, experts, align)
    got = ops().expert_order(index.cuda(), experts, align=align)
    for a, b in zip(got, want):
        assert a.dtype == torch.int32 and torch.equal(a.cpu(), b)


def test_orders_without_any_choice_and_with_one_expert_of_many():
    for index in (torch.full((300, 4), -1, dtype=torch.int32), torch.full((300, 4), 6, dtype=torch.int32), torch.full((9000, 2), -1, dtype=torch.int32), torch.full((9000, 2), 99, dtype=torch.int32)):
        for align in (1, 128):
            got = ops().expert_order(index.cuda(), 100, align=align)
            assert all(torch.equal(a.cpu(), b) for a, b in zip(got, plain_order(index, 100, align)))


def test_align_of_more_than_all_entries():
    index = choices(10, 2, 5, 3)
    got = ops().expert_order(index.cuda(), 5, align=1 << 20)
    want = plain_order(index, 5, 1 << 20)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want))


@pytest.mark.parametrize("rows,k,experts", [(400_001, 2, 9), (350_000, 4, 1000), (2_500_000, 1, 33)])
def test_orders_of_many_choices(rows, k, experts):
    """Blocks whose entries do not fit their registers; against a stable sort, which is exact."""
    index = torch.randint(-1, experts, (rows, k), generator=torch.Generator("cuda").manual_seed(rows), device="cuda", dtype=torch.int32)
    index[1000:200_000] = experts // 2   # a long run of one expert
    got = ops().expert_order(index, experts, align=64)
    flat = torch.where(index.flatten() < 0, experts, index.flatten())
    by = flat.sort(stable=True)
    counts = torch.bincount(flat, minlength=experts + 1)[:experts]
    begins = torch.cat([counts.new_zeros(1), ((counts + 63) // 64 * 64).cumsum(0)])
    assert torch.equal(got.offsets.long(), begins)
    ok = by.values < experts
    place = begins[by.values[ok].long()] + torch.arange(int(ok.sum()), device="cuda") - torch.cat([counts.new_zeros(1), counts.cumsum(0)])[by.values[ok].long()]
    position = torch.full_like(flat, -1).index_copy_(0, by.indices[ok], place.int())
    source = torch.full_like(got.source, -1).index_copy_(0, place, by.indices[ok].int())
    assert torch.equal(got.position.flatten(), position) and torch.equal(got.source, source)


def rows_of(rows, n, dtype, seed, pad=0, offset=0):
    g = torch.Generator("cuda").manual_seed(seed)
    return torch.randn(rows, n + pad + offset, generator=g, device="cuda").to(dtype)[:, offset:offset + n]


def plain_dispatch(x, order, k):
    source = order.source.long()
    out = x[source.clamp(min=0) // k] if len(x) else torch.zeros(len(source), x.shape[1], dtype=x.dtype, device=x.device)
    return torch.where(source[:, None] >= 0, out, torch.zeros((), dtype=x.dtype, device=x.device))


def check_all(x, index, experts, align, seed, strided=0):
    """Every direction on one order; places without a choice hold NaN, whatever is read there shows."""
    rows, k = index.shape
    n, dtype = x.shape[1], x.dtype
    order = ops().expert_order(index, experts, align=align)
    slots = len(order.source)
    position, source = order.position.long(), order.source.long()
    out = ops().dispatch_forward(x, order)
    assert out.dtype == dtype and torch.equal(out, plain_dispatch(x, order, k))
    y = rows_of(slots, n, dtype, seed, strided, strided)
    y.masked_fill_((source < 0)[:, None], math.nan)
    ok = position >= 0
    gathered = torch.where(ok[:, :, None], y[position.clamp(min=0)].double() if slots else torch.zeros(rows, k, n, device="cuda", dtype=torch.float64), 0.0)
    back = ops().dispatch_backward(y, order)
    assert ((back.double() - gathered.sum(1)).abs() <= U32 * (k + 1) * gathered.abs().sum(1) + HALF[dtype] * gathered.sum(1).abs() * 1.01 + TINY[dtype]).all()
    gate = torch.rand(rows, k, generator=torch.Generator("cuda").manual_seed(seed), device="cuda")
    gate[~ok] = math.nan   # of a choice without a place: not looked at
    g = torch.where(ok, gate, 0.0).double()
    want = (g[:, :, None] * gathered).sum(1)
    got = ops().combine_forward(y, order, gate)
    assert ((got.double() - want).abs() <= U32 * (k + 2) * (g[:, :, None] * gathered).abs().sum(1) + HALF[dtype] * want.abs() * 1.01 + TINY[dtype]).all()
    dout = rows_of(rows, n, dtype, seed + 1, strided, strided)
    dy, dgate = ops().combine_backward(dout, y, order, gate)
    products = gathered * dout.double()[:, None]
    assert ((dgate.double() - products.sum(2)).abs() <= U32 * (n / 32 + 13) * products.abs().sum(2) + 1e-44).all() and (dgate[~ok] == 0).all()
    flat = g.flatten()
    wy = torch.zeros(slots, n, dtype=torch.float64, device="cuda")
    live = source >= 0
    wy[live] = flat[source[live]][:, None] * dout.double()[source[live] // k]
    assert ((dy.double() - wy).abs() <= (U32 + HALF[dtype]) * wy.abs() * 1.01 + TINY[dtype]).all()
    return order


# widths around every change of layout, in 16-byte units of 4 and of 8 elements
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k,experts,n", [(1, 1, 1, 1), (3, 2, 9, 7), (50, 1, 4, 32), (33, 2, 9, 64), (40, 3, 16, 136), (25, 4, 64, 256), (17, 8, 40, 264), (9, 16, 100, 512), (21, 2, 9, 768), (12, 5, 9, 1000),
                                              (7, 2, 3, 1537), (2, 2, 9, 4096), (1300, 2, 9, 600), (1500, 9, 30, 40), (3, 1, 9, 9001)])
def test_rows(rows, k, experts, n, dtype):
    index = choices(rows, k, experts, rows + n, 0.2).cuda()
    for align in (1, 16):
        check_all(rows_of(rows, n, dtype, n), index, experts, align, n + align)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset", [1, 8])
def test_rows_of_a_wider_buffer(dtype, offset):
    index = choices(77, 3, 9, 5, 0.1).cuda()
    check_all(rows_of(77, 96, dtype, 4, 8, offset), index, 9, 4, 9, strided=offset)


def test_rows_without_a_choice():
    for rows in (20, 2000):
        index = choices(rows, 2, 9, 8).cuda()
        index[::3] = -1
        order = check_all(rows_of(rows, 130, torch.bfloat16, 6), index, 9, 8, 3)
        assert (ops().combine_forward(rows_of(len(order.source), 130, torch.bfloat16, 7), order, torch.ones(rows, 2, device="cuda"))[::3] == 0).all()
        index[:] = -1
        check_all(rows_of(rows, 130, torch.bfloat16, 6), index, 9, 8, 3)


def test_no_rows():
    index = torch.empty(0, 2, dtype=torch.int32, device="cuda")
    order = ops().expert_order(index, 9)
    x = torch.empty(0, 16, device="cuda")
    assert ops().dispatch_forward(x, order).shape == (0, 16) and ops().dispatch_backward(x, order).shape == (0, 16)
    assert ops().combine_forward(x, order, torch.empty(0, 2, device="cuda")).shape == (0, 16)
    dy, dgate = ops().combine_backward(x, x, order, torch.empty(0, 2, device="cuda"))
    assert dy.shape == (0, 16) and dgate.shape == (0, 2) and (order.offsets == 0).all()


def test_values_pass_as_they_are():
    x = torch.tensor([[math.inf, -0.0, math.nan, 1e-45] * 8], device="cuda")
    order = ops().expert_order(torch.tensor([[1, 0]], dtype=torch.int32, device="cuda"), 2)
    assert (ops().dispatch_forward(x, order).view(torch.int32) == x.view(torch.int32)).all()


def test_orders_that_are_not_of_this_library_are_safe():
    """Places outside the list are skipped, sources outside the choices are rows of zeros."""
    position = torch.tensor([[0, 7], [-5, 2], [2 ** 31 - 1, 1]], dtype=torch.int32, device="cuda")
    source = torch.tensor([0, 5, 3, 99, -7], dtype=torch.int32, device="cuda")
    order = ops().Order(position, source, None)
    x = rows_of(3, 40, torch.float32, 1)
    out = ops().dispatch_forward(x, order)
    assert torch.equal(out, torch.stack([x[0], x[2], x[1], 0 * x[0], 0 * x[0]]))
    assert torch.equal(ops().dispatch_backward(out, order), x)
    dy, dgate = ops().combine_backward(x, out, order, torch.ones(3, 2, device="cuda"))
    assert torch.equal(dy, out) and dgate[0, 1] == dgate[1, 0] == dgate[2, 0] == 0


def test_gradients_against_differences():
    rows, k, n = 14, 3, 40
    index = choices(rows, k, 5, 2, 0.1).cuda()
    order = ops().expert_order(index, 5, align=4)
    y, dout = rows_of(len(order.source), n, torch.float32, 1), rows_of(rows, n, torch.float32, 2)
    gate = torch.rand(rows, k, device="cuda")
    dy, dgate = ops().combine_backward(dout, y, order, gate)
    ok, at = order.position >= 0, order.position.clamp(min=0).long()
    value = lambda y, g: float(((torch.where(ok, g, 0.0)[:, :, None] * y[at]).sum(1) * dout.double()).sum())  # noqa: E731
    e = 1e-4
    for name, grad in (("y", dy), ("gate", dgate)):
        d = torch.randn(grad.shape, device="cuda", dtype=torch.float64)
        a, b = {"y": y.double(), "g": gate.double()}, {"y": y.double(), "g": gate.double()}
        key = name[0]
        a[key], b[key] = a[key] + e * d, b[key] - e * d
        # bilinear: central differences are exact but for 1e-16 / e
        assert abs(float((grad.double() * d).sum()) - (value(a["y"], a["g"]) - value(b["y"], b["g"])) / (2 * e)) <= U32 * 60 * float((grad.double() * d).abs().sum()) + 1e-9


def test_repeated_calls_agree():
    index = choices(20000, 4, 70, 9, 0.05).cuda()
    first = ops().expert_order(index, 70, align=8)
    y, gate = rows_of(len(first.source), 72, torch.float16, 2), torch.rand(20000, 4, device="cuda")
    dout = rows_of(20000, 72, torch.float16, 3)
    out, (dy, dgate) = ops().combine_forward(y, first, gate), ops().combine_backward(dout, y, first, gate)
    for _ in range(3):
        again = ops().expert_order(index, 70, align=8)
        assert all(torch.equal(a, b) for a, b in zip(again, first))
        got = (ops().combine_forward(y, again, gate), *ops().combine_backward(dout, y, again, gate))
        assert all(torch.equal(a, b) for a, b in zip(got, (out, dy, dgate)))


def test_offsets_beyond_32_bits():
    rows, k, n = 300_000, 2, 8192
    index = choices(rows, k, 9, 1).cuda()
    order = ops().expert_order(index, 9)
    x = torch.empty(rows, n, dtype=torch.float16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(1))
    y = ops().dispatch_forward(x, order)
    for s in (0, 1, rows, rows * k - 2, rows * k - 1):
        assert torch.equal(y[s], x[int(order.source[s]) // k])
    back = ops().combine_forward(y, order, torch.full((rows, k), 0.5, device="cuda"))
    assert torch.equal(back[-7:], x[-7:]) and torch.equal(back[:7], x[:7])
    dy, dgate = ops().combine_backward(x, y, order, torch.full((rows, k), 0.5, device="cuda"))
    assert torch.equal(dy[-3:], (0.5 * y[-3:].float()).half()) and (dgate[-5:] - x[-5:].float().square().sum(1, keepdim=True)).abs().max() <= 1e-3 * n
    del x, y, back, dy


def test_refusals():
    o = ops()
    index = choices(6, 2, 5, 1).cuda()
    order = o.expert_order(index, 5)
    x, y, gate = torch.zeros(6, 8, device="cuda"), torch.zeros(12, 8, device="cuda"), torch.zeros(6, 2, device="cuda")
    for bad in (lambda: o.expert_order(index.cpu(), 5), lambda: o.expert_order(index.long(), 5), lambda: o.expert_order(index[0], 5), lambda: o.expert_order(index.t(), 5), lambda: o.expert_order(index, 0),
                lambda: o.expert_order(index, 1025), lambda: o.expert_order(index, 5, align=0), lambda: o.expert_order(index, 5, align=1 << 31), lambda: o.expert_order(index, 5, align=1 << 30),
                lambda: o.expert_order(index[:, :0].contiguous(), 5), lambda: o.expert_order(torch.zeros(2, 17, dtype=torch.int32, device="cuda"), 5), lambda: o.expert_order(index, "a"),
                lambda: o.dispatch_forward(x[:5], order), lambda: o.dispatch_forward(x.double(), order), lambda: o.dispatch_forward(x[:, :0], order), lambda: o.dispatch_forward(x.cpu(), order),
                lambda: o.dispatch_backward(x, order), lambda: o.combine_forward(y, order, None), lambda: o.combine_forward(y, order, gate[:5]), lambda: o.combine_forward(y, order, gate.half()),
                lambda: o.combine_forward(x, order, gate), lambda: o.combine_backward(x, y, order, None), lambda: o.combine_backward(y, y, order, gate), lambda: o.combine_backward(x.half(), y, order, gate),
                lambda: o.combine_backward(x[:, :4], y, order, gate), lambda: o.dispatch_forward(x, order._replace(source=order.source.long())),
                lambda: o.dispatch_forward(x, order._replace(position=order.position.cpu()))):
        with pytest.raises(tb.TrainerError):
            bad()
    lib, err, p = tb.load_library(), C.create_string_buffer(200), y.data_ptr()
    # a result over what is read
    assert lib.tb_dispatch_forward(p, 8, 0, 6, 8, 2, order.position.data_ptr(), order.source.data_ptr(), 12, p, 8, None, err, 200) == -1 and b"overlaps" in err.value
