"""Table entries outside the pool in the rows that fork_pages reads."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tail", [0, 5])
@pytest.mark.parametrize("bad", [-1, -7, 12, 1 << 30])
@pytest.mark.parametrize("at", [0, 2])
def test_full_pages_of_a_parent_are_checked(bad, at, tail):
    """An entry outside the pool is skipped (-1 in the child) and recorded; the others are shared as they are."""
    from paged import fork_pages, pages_status
    page, g = 16, torch.Generator().manual_seed(1)
    pools = [torch.randn(12, 2, page, 16, generator=g).half().cuda() for _ in range(2)]
    table = torch.full((5, 6), -1, dtype=torch.int32)
    table[0, :4] = torch.tensor([3, 1, 7, 4])
    table[1, :4] = torch.tensor([2, 5, 6, 8])
    table[2:] = 9
    table[0, at] = bad
    assert pages_status() == 0
    dev = table.cuda()
    n = 3 * page + tail
    new = [10, 11, 0] if tail else [-1] * 3
    fork_pages(dev, *pools, [0, 1, 0], [2, 3, 4], [n, n, n], new)
    assert pages_status() == 3 and pages_status() == 0
    want = table.clone()
    for child, parent, x in zip((2, 3, 4), (0, 1, 0), new):
        want[child] = -1
        want[child, :3] = table[parent, :3]
        if parent == 0:
            want[child, at] = -1
        if tail:
            want[child, 3] = x
            for p in pools:
                assert torch.equal(p[x, :, :tail], p[int(table[parent, 3]), :, :tail])
    assert torch.equal(dev.cpu(), want)


def test_entries_behind_the_copied_positions_may_be_anything():
    from paged import fork_pages, pages_status
    pools = [torch.zeros(4, 1, 16, 16).half().cuda() for _ in range(2)]
    dev = torch.tensor([[2, -1, 99], [0, 0, 0]], dtype=torch.int32).cuda()
    fork_pages(dev, *pools, [0], [1], [16], [-1])
    assert dev.cpu().tolist() == [[2, -1, 99], [2, -1, -1]] and pages_status() == 0
