"""The root-mean-square norm in 8 bits where weights, results or squares leave the usual range."""
import math

import pytest

torch = pytest.importorskip("torch")
from test_gpu_rms import EPS, check_backward, check_quantised, make, ops, plain, vector  # noqa: E402

pytestmark = pytest.mark.gpu
# rows, columns, type, first column in a wider buffer: lanes that share a warp, a warp per row, walking down, several warps, few rows with more, rows read again; and rows that start anywhere
LAYOUTS = [(37, 40, torch.float32, 0), (129, 256, torch.float16, 0), (20000, 1000, torch.bfloat16, 0), (400, 1000, torch.float32, 0), (9, 1000, torch.float32, 0), (70, 2048, torch.float16, 0),
           (3, 33000, torch.float32, 0), (37, 41, torch.float32, 1), (300, 1001, torch.bfloat16, 1), (5, 4000, torch.float32, 3)]


@pytest.mark.parametrize("rows,n,dtype,offset", LAYOUTS)
@pytest.mark.parametrize("group", [None, 32, 64, 128])
def test_weights_far_from_one(rows, n, dtype, offset, group):
    """h * weight leaves fp32, or has fewer bits there, while h * rstd * weight does not."""
    x = make(rows, n, dtype, 3, offset, offset)
    half = dtype == torch.float16
    for size, weight in ((1.0 if half else 1e17, 1e36), (1.0, 1e37), (1e-4 if half else 1e-10, 1e-33), (1.0, 1e-34)):
        v = (x.float() * size).to(dtype)
        w = vector(n, 4) * weight
        check_quantised(v, w, None, group, ops().rms_norm_quantised(v, w, eps=0.0, group=group), eps=0.0)


@pytest.mark.parametrize("n,offset", [(8, 0), (100, 1), (256, 0), (1000, 0), (1536, 1), (9000, 0), (33000, 0)])
def test_scales_and_gradients_of_rows_whose_squares_leave_fp32(n, offset):
    factor = torch.tensor([1.0, 1e25, 1e-25, 1e30, 1.0, 1e-30, 1e37, 1e19, 1e-19], device="cuda")
    x = make(9, n, torch.float32, n, offset, offset).abs() + 0.5
    for dtype in (torch.float32, torch.bfloat16):
        v = torch.cat([torch.zeros(9, offset, device="cuda"), x * factor[:, None]], 1).to(dtype)[:, offset:]
        w, dy = vector(n, 4), make(9, n, dtype, 6)
        for group in (None, 32, 64, 128):
            check_quantised(v, w, None, group, ops().rms_norm_quantised(v, w, eps=0.0, group=group), eps=0.0)
        h, rstd = ops().rms_norm_forward(v, w, eps=0.0)[1:]
        check_backward(dy, h, rstd, w, None, ops().rms_norm_backward(dy, h, rstd, w))


def groups_of(n, group):
    return torch.arange(n, device="cuda") // (n if group is None else group)


@pytest.mark.parametrize("rows,n,dtype,offset", LAYOUTS)
@pytest.mark.parametrize("group", [None, 32, 128])
def test_a_group_with_an_infinity_from_the_weight(rows, n, dtype, offset, group):
    x = make(rows, n, dtype, 1, offset, offset)
    for odd in (math.inf, -math.inf, math.nan, 3e38):   # the last one makes y infinite wherever |h| / rms is above 1.2
        w = vector(n, 2)
        w[n // 2] = odd
        q, scale, _, _ = ops().rms_norm_quantised(x, w, eps=EPS, group=group)
        y = plain(x, w, None, EPS)[0].float()
        column = groups_of(n, group)
        most = torch.zeros(scale.shape, device="cuda").index_reduce_(1, column, y.abs(), "amax")
        near = (plain(x, w, None, EPS)[0].abs() / torch.finfo(torch.float32).max - 1).abs().amin(1, keepdim=True) < 1e-3   # y may round to either side
        bad = ~most.isfinite()
        assert bad.any() and ((scale == math.inf) | scale.isnan() | ~bad | near).all()
        assert (q.float().isnan() | ~bad[:, column] | near).all()
        assert (q.float().isfinite() | bad[:, column] | near).all() and (scale.isfinite() | bad | near).all()
