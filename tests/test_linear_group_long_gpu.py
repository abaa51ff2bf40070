"""group_rows of lists beyond one LDS map (131072 rows) over hundreds of groups: sizes at which every workgroup walks the list map by map."""
import pytest
import torch

from pixelbox_amd import linear

pytestmark = pytest.mark.gpu


def check(group, groups, offsets, order):
    key = torch.where((group >= 0) & (group < groups), group, torch.full_like(group, groups)).cpu()
    assert torch.equal(order.cpu().long(), torch.argsort(key, stable=True))
    counts = torch.bincount(key.long(), minlength=groups + 1)
    assert offsets.cpu().tolist() == [0] + counts[:groups].cumsum(0).tolist()


@pytest.mark.parametrize("m,groups", [(131072 + 1, 256), (262144, 300), (300_001, 1024), (1_000_003, 513), (4_000_000, 700)])
@pytest.mark.parametrize("kind", ["even", "uneven", "runs"])
def test_long_lists_of_many_groups(m, groups, kind):
    g = torch.Generator(device="cuda").manual_seed(m + groups)
    if kind == "even":
        group = torch.randint(-1, groups + 1, (m,), generator=g, device="cuda", dtype=torch.int32)
    elif kind == "uneven":  # most rows in a few groups, a tenth without one, many groups empty
        group = (torch.rand(m, generator=g, device="cuda") ** 8 * groups * 0.9).to(torch.int32)
        group[torch.rand(m, generator=g, device="cuda") < 0.1] = -1
    else:  # one group after the other, in falling order
        group = (groups - 1 - torch.arange(m, device="cuda") * groups // m).to(torch.int32)
    offsets, order = linear.group_rows(group, groups)
    check(group, groups, offsets, order)
    # into the caller's buffers, from an address off 16 bytes
    odd = torch.empty(m + 1, dtype=torch.int32, device="cuda")[1:]
    odd.copy_(group)
    o2, r2 = torch.full((groups + 1,), -7, dtype=torch.int32, device="cuda"), torch.full((m,), -7, dtype=torch.int32, device="cuda")
    linear.group_rows(odd, groups, offsets=o2, order=r2)
    assert torch.equal(o2, offsets) and torch.equal(r2, order)
