"""Routing on device tensors against the definition in 64 bits: the choice and the counts exactly, the rest to counted roundings.

A probability passes an exponential (2 ulp, plus the rounding of l - max: |l - max| u), a sum of `experts` terms and a division; with logits
within +-16 of each other that is (32 + 4 + experts / 4 + 8) u.  The means add chains of rows.
"""
import math

import pytest

import tatara_b200 as tb

torch = pytest.importorskip("torch")
from op_plain import HALF, TINY, U32, route_forward, route_objective  # noqa: E402

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
# experts around every change of layout, odd ones, one expert; rows that leave a block's last groups without one
SIZES = [(1, 1, 1), (5, 2, 2), (300, 9, 1), (513, 9, 2), (77, 16, 16), (64, 17, 3), (130, 64, 8), (33, 65, 4), (40, 128, 16), (50, 129, 2), (61, 256, 8), (20, 300, 5),
         (17, 512, 16), (9, 513, 7), (6, 1024, 16), (4099, 12, 2)]


def ops():
    from tatara_b200 import ops as o
    return o


def make(rows, experts, dtype, seed, forbidden=0.0, ties=False):
    g = torch.Generator("cuda").manual_seed(seed)
    x = (1.5 * torch.randn(rows, experts, generator=g, device="cuda")).clamp(-8, 8)
    if ties:
        x = x.round()
    if forbidden:
        x = x.masked_fill(torch.rand(rows, experts, generator=g, device="cuda") < forbidden, -math.inf)
    return x.to(dtype)


def check(logits, k, renormalise, mask, got):
    want = route_forward(logits, k, renormalise, mask)
    rows, experts = logits.shape
    assert torch.equal(got.index.cpu(), want["index"])
    assert torch.equal(got.counts.cpu(), want["counts"]) and int(got.rows) == want["rows"]
    rel = U32 * (44 + experts / 4)
    gate = got.gate.double().cpu()
    assert ((gate - want["gate"]).abs() <= rel * want["gate"] + 1e-37).all()
    chain = rel + U32 * (rows / 8 + 40)
    assert ((got.prob_mean.double().cpu() - want["prob_mean"]).abs() <= chain * want["prob_mean"] + 1e-37).all()
    losses = got.losses.double().cpu()
    assert abs(float(losses[0] - want["losses"][0])) <= (chain + 4 * U32) * float(want["losses"][0])
    # lse: absolute error of a few u times its parts, at most 8 + log(1024)
    assert abs(float(losses[1] - want["losses"][1])) <= 2 * chain * (float(want["losses"][1]) + 16 * math.sqrt(float(want["losses"][1])))
    return want


@pytest.mark.parametrize("renormalise", [True, False])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,experts,k", SIZES)
def test_forward(rows, experts, k, dtype, renormalise):
    x = make(rows, experts, dtype, rows + experts, ties=k > 1 and rows % 2 == 1)
    check(x, k, renormalise, None, ops().route_forward(x, k, renormalise=renormalise))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,experts,k", [(200, 9, 2), (100, 64, 8), (50, 256, 4), (40, 1000, 16), (30, 3, 3)])
def test_masks_and_forbidden_experts(rows, experts, k, dtype):
    x = make(rows, experts, dtype, 7, forbidden=0.3)
    x[3] = -math.inf                     # nothing to choose
    x[4, 1:] = -math.inf                 # one expert left, or none
    x[5] = torch.finfo(dtype).min        # the type's lowest value is a number: all alike
    x[6] = -math.inf
    x[6, -1] = torch.finfo(dtype).min
    mask = torch.rand(rows, device="cuda") > 0.3
    mask[3:7] = True
    x[0], mask[0] = math.nan, False      # what a masked row holds does not matter
    r = check_rows = ops().route_forward(x, k, mask=mask)
    lowest = torch.zeros(rows, dtype=torch.bool, device="cuda")
    lowest[5:7] = True
    # the z loss of rows at the lowest value overflows, as the definition's does in fp32: the rest is checked without them
    want = route_forward(x, k, True, mask.cpu())
    assert torch.equal(r.index.cpu(), want["index"]) and torch.equal(r.counts.cpu(), want["counts"]) and int(r.rows) == want["rows"]
    assert (r.index[3] == -1).all() and (r.gate[3] == 0).all() and (r.gate[0] == 0).all()
    assert (r.index[4, 1:] == -1).all() and r.gate[4, 0] == (r.index[4, 0] == 0)
    assert (r.index[5].cpu() == torch.arange(k)).all() and (r.gate[5] - 1 / k).abs().max() <= 4 * U32
    assert r.index[6, 0] == experts - 1 and r.gate[6, 0] == 1
    m2 = mask & ~lowest
    check(x, k, False, m2.cpu(), ops().route_forward(x, k, renormalise=False, mask=m2))
    assert check_rows.prob_mean.isfinite().all()


def test_nothing_left_and_no_rows():
    for x, mask in ((torch.full((6, 5), -math.inf, device="cuda"), None), (torch.zeros(6, 5, device="cuda"), torch.zeros(6, dtype=torch.bool, device="cuda")),
                    (torch.zeros(0, 5, device="cuda"), None)):
        r = ops().route_forward(x, 2, mask=mask)
        assert (r.index == -1).all() and (r.gate == 0).all() and (r.counts == 0).all() and int(r.rows) == 0
        assert (r.prob_mean == 0).all() and (r.losses == 0).all()
        d = ops().route_backward(x, r, torch.ones_like(r.gate), torch.ones(2, device="cuda"), mask=mask)
        assert d.shape == x.shape and (d == 0).all()


def test_values_that_are_not_numbers_are_seen():
    x = make(40, 9, torch.float32, 3)
    x[7, 4], x[9, 2] = math.nan, math.inf
    r = ops().route_forward(x, 2)
    assert r.index[7, 0] == 4 and r.gate[7].isnan().all() and r.index[9, 0] == 2 and r.gate[9].isnan().any()
    assert r.losses.isnan().all()
    keep = [i for i in range(40) if i not in (7, 9)]
    want = route_forward(x[keep], 2, True)
    assert torch.equal(r.index[keep].cpu(), want["index"])


def test_one_expert_left():
    for dtype in TYPES:
        x = make(30, 70, dtype, 13)
        x[11, :69] = -math.inf
        r = ops().route_forward(x, 4)
        assert r.index[11].tolist() == [69, -1, -1, -1] and r.gate[11].tolist() == [1, 0, 0, 0]
        check(x, 4, True, None, r)


def test_both_zeros_tie():
    x = torch.tensor([[-0.0, 0.0, -0.0], [0.0, -0.0, 0.0]], device="cuda")
    assert ops().route_forward(x, 3).index.tolist() == [[0, 1, 2], [0, 1, 2]]


@pytest.mark.parametrize("renormalise", [True, False])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,experts,k,forbidden", [(1, 1, 1, 0.0), (7, 2, 1, 0.0), (300, 9, 2, 0.2), (65, 16, 16, 0.0), (90, 40, 4, 0.3), (33, 100, 8, 0.0), (40, 256, 8, 0.1),
                                                       (12, 500, 3, 0.0), (6, 1024, 16, 0.5)])
def test_backward(rows, experts, k, forbidden, dtype, renormalise):
    x = make(rows, experts, dtype, experts, forbidden)
    mask = torch.rand(rows, device="cuda") > 0.2 if rows > 8 else None
    r = ops().route_forward(x, k, renormalise=renormalise, mask=mask)
    dgate, dl = torch.randn(rows, k, device="cuda"), torch.tensor([0.7, 0.3], device="cuda")
    got = ops().route_backward(x, r, dgate, dl, renormalise=renormalise, mask=mask)
    live = (x > -math.inf).any(1)
    if mask is not None:
        live = live & mask
    z = torch.where(x == -math.inf, torch.full_like(x, -1e4, dtype=torch.float32).double(), x.double()).requires_grad_()
    route_objective(z, r.index, r.counts, int(r.rows), k, renormalise, live, dgate.double(), dl.double()).backward()
    want = z.grad
    # every part of the sum is off by (44 + experts / 4) u and the sums over the row and the chosen add their lengths
    p = torch.softmax(z.detach(), 1)
    n = max(int(r.rows), 1)
    h = 0.7 * experts * r.counts.double() / (n * k) / n
    g = r.gate.double()
    dot = (g * dgate.double()).abs().sum(1, keepdim=True)
    lse = torch.logsumexp(z.detach(), 1).abs()
    parts = p * (h + (p * h).sum(1, keepdim=True) + 0.6 / n * (lse[:, None] + 16) + (0 if renormalise else dot))
    part = torch.zeros_like(parts).scatter_add_(1, r.index.clamp(min=0).long(), g * (dgate.double().abs() + dot))
    tol = U32 * (60 + experts / 2 + k) * (parts + part) + HALF[dtype] * want.abs() * 1.01 + TINY[dtype]
    assert ((got.double() - want).abs() <= tol)[live].all(), float(((got.double() - want).abs() / tol)[live].max())
    assert (got[~live] == 0).all()
    assert (got[x == -math.inf] == 0).all()


@pytest.mark.parametrize("renormalise", [True, False])
def test_gradient_against_differences(renormalise):
    rows, experts, k = 23, 9, 3
    x = make(rows, experts, torch.float32, 5)
    r = ops().route_forward(x, k, renormalise=renormalise)
    dgate, dl = torch.randn(rows, k, device="cuda"), torch.tensor([2.0, 0.5], device="cuda")
    got = ops().route_backward(x, r, dgate, dl, renormalise=renormalise).double()
    live = torch.ones(rows, dtype=torch.bool, device="cuda")
    value = lambda z: float(route_objective(z, r.index, r.counts, rows, k, renormalise, live, dgate.double(), dl.double()))  # noqa: E731
    h = 1e-5
    for seed in range(4):
        d = torch.randn(x.shape, device="cuda", dtype=torch.float64, generator=torch.Generator("cuda").manual_seed(seed))
        want = (value(x.double() + h * d) - value(x.double() - h * d)) / (2 * h)
        assert abs(float((got * d).sum()) - want) <= 200 * U32 * float((got * d).abs().sum() + d.abs().sum() / rows) + 1e-7


def test_either_gradient_alone_and_strides():
    x = make(200, 20, torch.float32, 5)
    wide = torch.full((200, 29), math.nan, device="cuda")
    wide[:, 3:23] = x
    r, s = ops().route_forward(x, 2), ops().route_forward(wide[:, 3:23], 2)
    check(x, 2, True, None, s)   # rows that do not start on 16-byte boundaries are added in another order
    dgate, dl = torch.randn(200, 2, device="cuda"), torch.tensor([1.0, 0.25], device="cuda")
    both, a, b = ops().route_backward(x, r, dgate, dl), ops().route_backward(x, r, dgate), ops().route_backward(x, r, None, dl)
    assert ((a + b - both).abs() <= 16 * U32 * (a.abs() + b.abs() + 1)).all()
    assert ((ops().route_backward(wide[:, 3:23], r, dgate, dl) - both).abs() <= 16 * U32 * (a.abs() + b.abs() + 1)).all()
    again = ops().route_forward(x, 2)
    assert all(torch.equal(p, q) for p, q in zip(r, again))


def test_offsets_beyond_32_bits():
    far = (1 << 30) + 16
    wide = torch.zeros(3 * far, dtype=torch.float16, device="cuda")
    x = wide.as_strided((3, 12), (far, 1))
    x.copy_(make(3, 12, torch.float16, 4))
    check(x, 2, True, None, ops().route_forward(x, 2))


def test_uint8_mask_and_another_stream():
    x = make(3000, 9, torch.float32, 8)
    mask = torch.rand(3000, device="cuda") > 0.5
    want = ops().route_forward(x, 1, mask=mask)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        y = x * 1.0
        got = ops().route_forward(y, 1, mask=mask.to(torch.uint8))
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals():
    o = ops()
    x = torch.zeros(4, 8, device="cuda")
    r = o.route_forward(x, 2)
    for bad in (lambda: o.route_forward(x, 0), lambda: o.route_forward(x, 9), lambda: o.route_forward(torch.zeros(4, 40, device="cuda"), 17), lambda: o.route_forward(x.double(), 1),
                lambda: o.route_forward(x.cpu(), 1), lambda: o.route_forward(x.t(), 1), lambda: o.route_forward(torch.zeros(2, 1025, device="cuda"), 1),
                lambda: o.route_forward(x, 1, mask=torch.ones(3, dtype=torch.bool, device="cuda")), lambda: o.route_forward(x, 1, mask=torch.ones(4, device="cuda")),
                lambda: o.route_backward(x, r, torch.zeros(4, 3, device="cuda")), lambda: o.route_backward(x[:3], r), lambda: o.route_backward(x, r, None, torch.zeros(3, device="cuda")),
                lambda: o.route_forward(x[:, :0], 1)):
        with pytest.raises(tb.TrainerError):
            bad()
    lib = tb.load_library()
    p = x.data_ptr()
    assert lib.tb_route_forward(p, 8, 0, 4, 8, 2, 1, None, p, p, p, p, p, p, p, 0, None, None, 0) == -1
    assert lib.tb_route_forward_workspace(4, 0) == -1 and lib.tb_route_forward_workspace(-1, 8) == -1


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,experts,k,offset", [(20001, 9, 2, 0), (20001, 12, 4, 0), (9001, 48, 8, 0), (9001, 47, 8, 1), (5003, 128, 4, 0), (5003, 256, 8, 0), (3001, 255, 8, 3), (777, 1024, 16, 0)])
def test_gradient_over_the_logits(rows, experts, k, offset, dtype):
    """dlogits in the logits' memory, through the C entry point: the bits of a result of its own."""
    wide = torch.full((rows, experts + offset), 3.0, dtype=dtype, device="cuda")
    x = wide[:, offset:]
    x.copy_(make(rows, experts, dtype, 3, forbidden=0.1))
    mask = torch.rand(rows, device="cuda") > 0.2
    r = ops().route_forward(x, k, mask=mask)
    dgate, dl = torch.randn(rows, k, device="cuda"), torch.tensor([0.7, 0.3], device="cuda")
    want = ops().route_backward(x, r, dgate, dl, mask=mask)
    kind = TYPES.index(dtype)
    rc = tb.load_library().tb_route_backward(x.data_ptr(), x.stride(0), kind, rows, experts, k, 1, mask.data_ptr(), r.index.data_ptr(), r.gate.data_ptr(), dgate.data_ptr(),
                                             r.counts.data_ptr(), r.rows.data_ptr(), dl.data_ptr(), x.data_ptr(), x.stride(0), torch.cuda.current_stream().cuda_stream, None, 0)
    assert rc == 0
    assert torch.equal(x, want) and (wide[:, :offset] == 3).all()


@pytest.mark.parametrize("dtype,bits", [(torch.float16, (0x7e00, 0xfe00, 0x7c01, 0xffff)), (torch.bfloat16, (0x7fc0, 0xffc0, 0x7f81, 0xffff))])
@pytest.mark.parametrize("experts,k", [(9, 2), (9, 1), (48, 8), (256, 8), (300, 4)])
def test_values_that_are_not_numbers_in_16_bits(experts, k, dtype, bits):
    """A NaN of either sign, quiet or not, is the largest; two of them tie, and +inf comes behind them."""
    x = make(40, experts, dtype, 3)
    raw = x.view(torch.int16)
    for row, pattern in enumerate(bits):
        raw[row, 5] = pattern - (1 << 16) if pattern >= 1 << 15 else pattern
    x[4, 7], x[4, 2] = math.nan, math.nan
    x[5, 6], x[5, 8] = math.inf, math.nan
    x[6, 3] = math.inf
    x[7] = -math.inf
    x[7, 1] = math.nan
    r = ops().route_forward(x, k)
    assert r.index[:8, 0].tolist() == [5, 5, 5, 5, 2, 8, 3, 1]
    if k > 1:
        assert r.index[4, 1] == 7 and r.index[5, 1] == 6 and r.index[7, 1] == -1
    assert r.gate[:6, 0].isnan().all() and r.gate[7, 0].isnan() and r.losses.isnan().all()
    keep = list(range(8, 40))
    want = route_forward(x[keep], k, True)
    assert torch.equal(r.index[keep].cpu(), want["index"])
    # the gradient: NaN in those rows, the others as without them
    dgate, dl = torch.randn(40, k, device="cuda"), torch.tensor([0.0, 0.0], device="cuda")
    d = ops().route_backward(x, r, dgate, dl)
    mask = torch.zeros(40, dtype=torch.bool, device="cuda")
    mask[8:] = True
    clean = ops().route_backward(x, ops().route_forward(x, k, mask=mask), dgate, dl, mask=mask)
    assert d[:8].isnan().any(1).all() and torch.equal(d[8:], clean[8:]) and (clean[:8] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_order_of_the_smallest_numbers_in_16_bits(dtype):
    """Subnormal logits are told apart, of either sign."""
    bits = torch.tensor([[0x0001, 0x0003, 0x8001, 0x0002, 0x8002, 0x0000, 0x8000, 0x0010]], dtype=torch.int32)
    x = bits.to(torch.int16).view(dtype).cuda()
    assert ops().route_forward(x, 8).index.tolist() == [[7, 1, 3, 0, 5, 6, 2, 4]]
