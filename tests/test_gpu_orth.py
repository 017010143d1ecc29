"""Orthogonalisation and the Muon step on device tensors against the definition in 64 bits.

Tolerances, as the norm of the difference over the norm of the result.  A step makes three products of operands rounded to u (2^-12 of an
element with one limb, 2^-22 with two): sqrt(3) sqrt(2 / 3) u = 1.4 u of its result, which the plateau of the polynomial (slope up to 3.9 where
the value is 0.7 of the argument) may raise by 5.5; over five steps 1.4 * 5.5 * sqrt(5) = 17 u.  fp32 accumulation adds 2^-24 times the root of the 3 K / 16
partial sums, raised alike: 1e-5 at K = 1000.  A short side of up to 64 is computed in 64 bits: only the result is rounded.
"""
import math

import pytest

import tatara_b200 as tb

torch = pytest.importorskip("torch")
from op_plain import HALF, muon_step, orthogonalise  # noqa: E402

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
SMALL = [(1, 1, 1), (2, 1, 5), (3, 7, 3), (9, 16, 1536), (1, 1024, 32), (2, 33, 64), (4, 64, 64), (1, 64, 65), (2, 300, 64), (1, 5, 20011), (1, 3000, 17), (70, 13, 9), (9, 32, 30)]
LARGE = [(1, 65, 65), (2, 65, 200), (1, 128, 128), (3, 129, 257), (1, 200, 130), (2, 384, 1000), (1, 777, 1000), (1, 1000, 65), (1, 70, 2500),
         (64, 70, 300), (22, 300, 400), (5, 1100, 1300), (1, 2600, 2700), (70, 130, 67)]
UNIT = {torch.float32: 2.0 ** -22, torch.float16: 2.0 ** -22, torch.bfloat16: 2.0 ** -12}


def ops():
    from tatara_b200 import ops as o
    return o


def make(batch, rows, cols, seed, dtype=torch.float32):
    """Gradients: some strong directions over noise, of ordinary small size."""
    g = torch.Generator("cuda").manual_seed(seed)
    rank = min(rows, cols, 8)
    x = torch.randn(batch, rows, rank, generator=g, device="cuda") @ torch.randn(batch, rank, cols, generator=g, device="cuda")
    return ((0.3 * x + torch.randn(batch, rows, cols, generator=g, device="cuda")) * 1e-2).to(dtype)


def tolerance(dtype, rows, cols):
    if min(rows, cols) <= 64:
        return 2 * HALF[dtype]
    return 17 * UNIT[dtype] + 1.1e-5 + HALF[dtype]


def far(got, want):
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,rows,cols", SMALL + LARGE)
def test_orthogonalise(batch, rows, cols, dtype):
    x = make(batch, rows, cols, rows + cols, dtype)
    got = ops().orthogonalise(x)
    want = orthogonalise(x)
    assert got.dtype == dtype and got.shape == x.shape
    for b in range(batch):
        assert far(got[b], want[b]) <= tolerance(dtype, rows, cols)


@pytest.mark.parametrize("rows,cols", [(12, 40), (150, 90)])
@pytest.mark.parametrize("steps", [1, 2, 3, 8])
def test_steps_and_coefficients(rows, cols, steps):
    x = make(2, rows, cols, steps)
    got = ops().orthogonalise(x, steps=steps)
    assert far(got, orthogonalise(x, steps)) <= tolerance(torch.float32, rows, cols) * max(1, steps / 5)
    c = (1.875, -1.25, 0.375)  # the convergent quintic
    got = ops().orthogonalise(x, steps=steps, coefficients=c)
    assert far(got, orthogonalise(x, steps, c)) <= tolerance(torch.float32, rows, cols) * max(1, steps / 5)


@pytest.mark.parametrize("rows,cols", [(16, 600), (96, 300), (300, 96)])
def test_strided_batches_and_in_place(rows, cols):
    wide = torch.full((3, rows + 2, cols + 7), math.nan, device="cuda")
    x = make(3, rows, cols, 5)
    view = wide[:, 1:1 + rows, 3:3 + cols]
    view.copy_(x)
    want = ops().orthogonalise(x)
    assert torch.equal(ops().orthogonalise(view), want)
    assert torch.equal(ops().orthogonalise(x), want)       # again: the same bits
    out = torch.full((3, rows + 1, cols + 5), 2.0, device="cuda")
    ops().orthogonalise(view, out=out[:, :rows, 2:2 + cols])
    assert torch.equal(out[:, :rows, 2:2 + cols], want) and (out[:, rows:] == 2).all() and (out[:, :, :2] == 2).all() and (out[:, :, 2 + cols:] == 2).all()
    assert torch.equal(ops().orthogonalise(view, out=view), want)
    assert wide[:, 0].isnan().all() and wide[:, :, :3].isnan().all()
    assert torch.equal(ops().orthogonalise(x[0]), want[0])


@pytest.mark.parametrize("rows,cols", [(16, 200), (64, 64), (120, 256), (256, 120)])
def test_few_directions(rows, cols):
    """Rank one: the other singular values are zero, and what roundings put there grows like 3.4445^5 = 485."""
    g = torch.Generator("cuda").manual_seed(1)
    x = torch.randn(rows, 1, generator=g, device="cuda") * torch.randn(1, cols, generator=g, device="cuda")
    assert far(ops().orthogonalise(x), orthogonalise(x)) <= (2.0 ** -23 if min(rows, cols) <= 64 else 2 * 485 * 2.0 ** -22)


@pytest.mark.parametrize("rows,cols", [(16, 200), (120, 256)])
def test_zeros_sizes_and_values_that_are_not_numbers(rows, cols):
    x = make(4, rows, cols, 3)
    want = ops().orthogonalise(x)
    y = x.clone()
    y[1] = 0
    y[2, 3, 5] = math.nan
    got = ops().orthogonalise(y)
    assert (got[1] == 0).all() and got[2].isnan().all() and torch.equal(got[0], want[0]) and torch.equal(got[3], want[3])
    y[2, 3, 5] = math.inf
    assert ops().orthogonalise(y)[2].isnan().all()
    # the norm neither overflows nor vanishes: squares would, in 32 bits
    for size in (2.0 ** 90, 2.0 ** -90):
        got = ops().orthogonalise(x * size, eps=0.0)
        assert far(got, orthogonalise(x.double(), eps=0.0)) <= tolerance(torch.float32, rows, cols)


@pytest.mark.parametrize("g_type", TYPES)
@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("batch,rows,cols", [(9, 16, 256), (1, 512, 32), (1, 1, 1), (2, 130, 300), (1, 300, 130)])
def test_muon_step(batch, rows, cols, nesterov, g_type):
    w, m = 0.05 * torch.randn(batch, rows, cols, device="cuda"), make(batch, rows, cols, 1)
    g = make(batch, rows, cols, 2, g_type)
    args = dict(lr=0.05, beta=0.9, nesterov=nesterov, weight_decay=0.1, scale=1.5, clip=0.12)
    w2, m2 = torch.empty_like(w), torch.empty_like(m)
    keep = w.clone(), m.clone()
    ops().muon_step(w, m, g, weight_out=w2, momentum_out=m2, **args)
    want_w, want_m = muon_step(w, m, g, **args)
    assert torch.equal(w, keep[0]) and torch.equal(m, keep[1])
    assert ((m2.double() - want_m).abs() <= 2.0 ** -23 * (0.9 * m.double().abs() + g.double().abs())).all()
    # the weights: their own roundings and the orthogonalised update's (u itself is rounded: 2^-23 of its parts)
    o = (want_w - w.double()).norm() / 1.0
    err = float((w2.double() - want_w).norm())
    size = 0.05 * 1.5 * math.sqrt(batch * min(rows, cols)) * 1.2
    assert err <= 3 * 2.0 ** -24 * float(w.double().norm()) + size * (tolerance(torch.float32, rows, cols) + 100 * 2.0 ** -23), (err, float(o))
    assert (w2.abs() <= torch.tensor(0.12, device="cuda")).all()
    # in place, and the same bits
    ops().muon_step(w, m, g, **args)
    assert torch.equal(w, w2) and torch.equal(m, m2)


def test_muon_defaults_and_two_dimensions():
    w, m, g = 0.1 * torch.randn(200, 50, device="cuda"), torch.zeros(200, 50, device="cuda"), make(1, 200, 50, 4)[0]
    want, _ = muon_step(w, m, g, 0.02, 0.95, True, 0.0, 2.0, math.inf)
    got, m1 = ops().muon_step(w.clone(), m, g, lr=0.02)
    assert far(got, want) <= 2.0 ** -23 and torch.equal(m1, g)


def test_another_stream():
    x = make(1, 400, 500, 6)
    want = ops().orthogonalise(x)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        y = ops().orthogonalise(x * 1.0)
    s.synchronize()
    assert torch.equal(y, want)


@pytest.mark.parametrize("rows,cols", [(8, 40), (70, 130)])
def test_matrices_far_apart(rows, cols):
    """Offsets beyond 32 bits."""
    far = (1 << 31) + 64
    wide = torch.zeros(far + rows * cols, dtype=torch.bfloat16, device="cuda")
    x = wide.as_strided((2, rows, cols), (far, cols, 1))
    x.copy_(make(2, rows, cols, 9, torch.bfloat16))
    want = ops().orthogonalise(x.contiguous())
    assert torch.equal(ops().orthogonalise(x), want)
    assert torch.equal(ops().orthogonalise(x, out=x), want) and (wide[rows * cols:far] == 0).all()


@pytest.mark.parametrize("rows,cols", [(12, 40), (70, 90)])
def test_outputs_that_overlap_the_input_in_part(rows, cols):
    x = make(3, rows, cols, 5)
    flat = torch.cat([x.flatten(), torch.zeros(rows * cols, device="cuda")])
    want = ops().orthogonalise(x)
    with pytest.raises(tb.TrainerError, match="overlaps"):
        ops().orthogonalise(flat[:x.numel()].view_as(x), out=flat[rows * cols:].view_as(x))
    wide = torch.zeros(3, rows, 2 * cols, device="cuda")
    wide[:, :, :cols] = x
    with pytest.raises(tb.TrainerError, match="overlaps"):
        ops().orthogonalise(wide[:, :, :cols], out=wide[:, :, 3:3 + cols])
    # other columns of the same rows
    assert torch.equal(ops().orthogonalise(wide[:, :, :cols], out=wide[:, :, cols:]), ops().orthogonalise(wide[:, :, :cols]))
    assert float((wide[:, :, cols:] - want).abs().max()) <= 1e-4


# tiles of 64, 128 and 256 columns, K in parts and whole, several matrices; every layout of the result
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,rows,cols", [(1, 130, 4096), (2, 130, 1500), (1, 359, 785), (1, 785, 360), (3, 500, 304), (7, 66, 128), (1, 1024, 1024), (20, 65, 129), (1, 1500, 1100)])
def test_orthogonalise_in_every_tile_shape(batch, rows, cols, dtype):
    x = make(batch, rows, cols, batch + rows + cols, dtype)
    assert far(ops().orthogonalise(x), orthogonalise(x)) <= tolerance(dtype, rows, cols)


def test_refusals():
    o = ops()
    x = make(2, 70, 80, 0)
    w = x.clone()
    both = torch.zeros(3, 70, 80, device="cuda")
    for bad in (lambda: o.orthogonalise(x.double()), lambda: o.orthogonalise(x.cpu()), lambda: o.orthogonalise(x[0, 0]), lambda: o.orthogonalise(x.transpose(1, 2)),
                lambda: o.orthogonalise(x, steps=0), lambda: o.orthogonalise(x, steps=33), lambda: o.orthogonalise(x, eps=-1.0), lambda: o.orthogonalise(x, coefficients=(8.0, 0.0, 0.0)),
                lambda: o.orthogonalise(x, coefficients=(1.0, 2.0)), lambda: o.orthogonalise(x, coefficients=(math.nan, 0.0, 0.0)), lambda: o.orthogonalise(x, out=x.half()),
                lambda: o.orthogonalise(x, out=x[0]), lambda: o.orthogonalise(x[:, :0]), lambda: o.orthogonalise(x[:1].expand(2, 70, 80)),
                lambda: o.muon_step(w, x[:1], x, lr=0.1), lambda: o.muon_step(w, w, x.double(), lr=0.1), lambda: o.muon_step(w.half(), w, x, lr=0.1),
                lambda: o.muon_step(w, w, x.cpu(), lr=0.1), lambda: o.muon_step(w, w, x, lr=0.1, clip=0.0), lambda: o.muon_step(w, w, x, lr=0.1, clip=math.nan),
                lambda: o.muon_step(w.transpose(1, 2), w, x, lr=0.1), lambda: o.muon_step(w, w, x, lr=0.1), lambda: o.muon_step(w, x, x, lr=0.1),
                lambda: o.muon_step(both[:2], x, w, lr=0.1, weight_out=both[1:]), lambda: o.muon_step(both[0], both[1], both[2], lr=0.1, momentum_out=both[2]),
                lambda: o.muon_step(both[0], both[1], both[2], lr=0.1, weight_out=both[1])):
        with pytest.raises(tb.TrainerError):
            bad()
    lib = tb.load_library()
    import ctypes as C
    p, c = x.data_ptr(), (C.c_float * 3)(3.4445, -4.7750, 2.0315)
    assert lib.tb_orthogonalise(p, 5600, 80, 0, 2, 70, 80, 5, c, 1e-7, p, 5600, 80, None, 0, None, None, 0) == -1      # no workspace
    assert lib.tb_orthogonalise(p, 5600, 80, 0, 2, 70, 80, 5, None, 1e-7, p, 5600, 80, p, 1 << 30, None, None, 0) == -1
    assert lib.tb_orthogonalise_workspace(0, 1, 0, 5) == -1 and lib.tb_orthogonalise_workspace(7, 1, 5, 5) == -1 and lib.tb_muon_step_workspace(-1, 5, 5) == -1
    assert lib.tb_orthogonalise(None, 0, 80, 0, 0, 70, 80, 5, c, 1e-7, None, 0, 80, None, 0, None, None, 0) == 0        # an empty batch
    assert lib.tb_muon_step(None, p, p, p, 0, 2, 70, 80, p, p, None, 0, None, None, 0) == -1


# Blocks far below the others keep their digits: nothing of one block's rounding reaches another, so each is as near as a whole matrix is.  (Entries of
# the last block are about 1e-8 of the norm: two limbs are off by at most 2^-47 of it there, which is less than 2^-20 of such an entry.)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(200, 200), (60, 230), (230, 70), (600, 800), (1100, 1000)])
def test_blocks_of_different_scale(rows, cols, dtype):
    scales = (1.0, 0.03, 1e-2) if dtype == torch.float16 else (1.0, 1e-3, 1e-5)  # results of fp16 stay in the range of their type
    x = torch.zeros(3 * rows, 3 * cols, device="cuda")
    blocks = [(slice(i * rows, (i + 1) * rows), slice(i * cols, (i + 1) * cols)) for i in range(3)]
    for i, b in enumerate(blocks):
        x[b] = make(1, rows, cols, 7 + i)[0] * (scales[i] * 30)
    x = x.to(dtype)
    got, want = ops().orthogonalise(x), orthogonalise(x)
    for b in blocks:
        assert far(got[b], want[b]) <= tolerance(dtype, 3 * rows, 3 * cols), far(got[b], want[b])
    out = torch.ones(3 * rows, 3 * cols, dtype=torch.bool, device="cuda")
    for b in blocks:
        out[b] = False
    assert (got[out] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,cols", [(16, 200), (120, 256), (256, 120), (301, 97)])
def test_norms_at_the_ends_of_the_range(rows, cols, dtype):
    """eps = 0: what the norm divides is the type's smallest and largest numbers, and its reciprocal beyond them."""
    for size in (2.0 ** -136, 2.0 ** -125, 2.0 ** -110, 2.0 ** 110, 2.0 ** 126):
        x = (make(2, rows, cols, 4, torch.float32).clamp_(-1, 1).double() * size).to(dtype)
        got = ops().orthogonalise(x, eps=0.0)
        if (x == 0).all():  # below the type's smallest number: 0 / 0
            assert got.isnan().all()
        else:
            assert far(got, orthogonalise(x, eps=0.0)) <= tolerance(dtype, rows, cols), size


# Products of tiles of 256 columns by pairs of blocks that take several tiles each (all three kinds at 4096 x 4096, and in 16 bits from 3072 on), results that
# are stored straight from registers (rows on 16-byte boundaries, or tall) and through shared memory.  fp32 sums of K terms: the tolerance's 1.1e-5 is of K = 1000 and
# grows with its root.
LARGEST = [(1, 4096, 4096), (1, 3072, 3200), (1, 3200, 3072), (1, 2600, 4096), (1, 3073, 3001), (1, 4097, 4100), (6, 1024, 1024)]


def large_tolerance(dtype, rows, cols):
    return 17 * UNIT[dtype] + 1.1e-5 * math.sqrt(max(1.0, max(rows, cols) / 1000)) + HALF[dtype]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,rows,cols", LARGEST)
def test_largest(batch, rows, cols, dtype):
    x = make(batch, rows, cols, rows + 2 * cols, dtype)
    assert far(ops().orthogonalise(x), orthogonalise(x)) <= large_tolerance(dtype, rows, cols)


@pytest.mark.parametrize("g_type", TYPES)
@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("batch,rows,cols", [(1, 4096, 4096), (1, 3200, 3072), (1, 2600, 2700), (2, 136, 304), (2, 304, 136), (4, 72, 1000), (1, 100, 2048), (3, 520, 520), (12, 200, 264)])
def test_muon_step_of_every_layout(batch, rows, cols, nesterov, g_type):
    """Rows on 16-byte boundaries with gradients of every type, tall ones, one and several tiles per block."""
    w, m = 0.05 * torch.randn(batch, rows, cols, device="cuda"), make(batch, rows, cols, 1)
    g = make(batch, rows, cols, 2, g_type)
    args = dict(lr=0.05, beta=0.9, nesterov=nesterov, weight_decay=0.1, scale=1.5, clip=0.12)
    want_w, want_m = muon_step(w, m, g, **args)
    w2, m2 = ops().muon_step(w, m, g, weight_out=torch.empty_like(w), momentum_out=torch.empty_like(m), **args)
    assert ((m2.double() - want_m).abs() <= 2.0 ** -23 * (0.9 * m.double().abs() + g.double().abs())).all()
    size = 0.05 * 1.5 * math.sqrt(batch * min(rows, cols)) * 1.2
    off = float((w2.double() - want_w).norm())
    assert off <= 3 * 2.0 ** -24 * float(w.double().norm()) + size * (large_tolerance(torch.float32, rows, cols) + 100 * 2.0 ** -23), off
    # every weight by itself: an update's element is off by no more than the whole update's root mean square times 1e-3
    each = 1e-3 * 0.05 * 1.5 / math.sqrt(max(rows, cols)) + 2.0 ** -22 * w.double().abs()
    assert ((w2.double() - want_w).abs() <= each).all()
    w3, m3 = ops().muon_step(w, m, g, **args)
    assert torch.equal(w3, w2) and torch.equal(m3, m2)
