"""Results of one call that lie in one allocation: each has its own memory there, whatever its type."""
import itertools

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,n", [(1, 1), (3, 7), (33, 1000)])
def test_results_do_not_overlap(rows, n, dtype):
    from tatara_b200 import ops
    x = torch.randn(rows, n, device="cuda").to(dtype)
    order = ops.expert_order(torch.zeros(rows, 2, dtype=torch.int32, device="cuda"), 3, align=16)
    for results in (ops.rms_norm_forward(x, residual=x), ops.rms_norm_quantised(x, residual=x, group=32), ops.layer_norm_forward(x), order, ops.route_forward(x[:, :9], 1)):
        spans = []
        for t in results:
            assert t.is_contiguous()
            base = t.untyped_storage()
            assert t.data_ptr() == base.data_ptr() + t.storage_offset() * t.element_size()
            assert t.data_ptr() + t.numel() * t.element_size() <= base.data_ptr() + base.nbytes()
            spans.append((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()))
        for (a0, a1), (b0, b1) in itertools.combinations(spans, 2):
            assert a1 <= b0 or b1 <= a0
    h = ops.rms_norm_forward(x, residual=x)[1]
    assert torch.equal(h, (x.float() + x.float()).to(dtype))
