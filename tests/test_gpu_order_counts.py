"""The places of a sort over many blocks: their counts are added up a batch at a time, or by a launch of their own."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


# entries for one block to a few hundred of them, around whole batches of 16 blocks per thread; keys from one per thread to four, with and without the launch between
@pytest.mark.parametrize("experts", [1, 3, 9, 33, 64, 128, 200, 256, 300, 1024])
@pytest.mark.parametrize("entries", [2048, 2049, 3 * 1024 + 1, 15 * 1024, 16 * 1024, 16 * 1024 + 7, 17 * 1024, 33 * 1024 - 5, 63 * 1024, 65 * 1024, 128 * 1024, 129 * 1024 + 3, 148 * 1024, 160 * 2048, 700000])
def test_order_of_many_blocks(entries, experts):
    from tatara_b200 import ops
    g = torch.Generator("cuda").manual_seed(entries + experts)
    index = torch.randint(-1, experts, (entries, 1), generator=g, device="cuda", dtype=torch.int32)
    index[::3] = experts // 2   # one in demand
    position, source, offsets = ops.expert_order(index, experts)
    key = torch.where(index[:, 0] < 0, experts, index[:, 0].long())
    by = torch.sort(key, stable=True).indices
    used = int((key < experts).sum())
    assert torch.equal(source[:used], by[:used].int()) and (source[used:] == -1).all()
    want = torch.full((entries,), -1, dtype=torch.int32, device="cuda")
    want[by[:used]] = torch.arange(used, dtype=torch.int32, device="cuda")
    assert torch.equal(position[:, 0], want)
    assert torch.equal(offsets, torch.cat([torch.zeros(1, device="cuda", dtype=torch.long), torch.bincount(key, minlength=experts + 1)[:experts].cumsum(0)]).int())
