"""Tensors that share memory, as the paged operators take or refuse them."""
import pytest
import torch

from paged_helpers import Case

pytestmark = pytest.mark.gpu


def test_outputs_over_other_rows_or_the_pools_are_refused():
    c = Case(torch.float16, 128, 2, 2, 32, [6], [96], [20, 4], seed=60)
    plan = c.plan()
    want, lse = c.run(plan)
    n = c.q.numel()
    both = torch.zeros(n + 512, dtype=c.q.dtype, device="cuda")
    c.q, kept = both[:n].view_as(c.q).copy_(c.q), c.q.clone()
    for bad in (both[512:].view_as(c.q), both[8:n + 8].view_as(c.q)):
        with pytest.raises(ValueError, match="overlaps q"):
            c.run(plan, out=bad)
    pool = c.k_pool = c.k_pool.contiguous()
    c.v_pool = c.v_pool.contiguous()
    with pytest.raises(ValueError, match="overlaps the pools"):
        c.run(plan, out=pool.view(-1)[:n].view_as(c.q))
    assert torch.equal(c.q, kept)
    out, again = c.run(plan, out=c.q)                   # q itself
    assert torch.equal(out, want) and torch.equal(again, lse)


def test_pools_of_one_tensor():
    from paged import copy_pages
    base = torch.randn(12, 1, 2, 16, 64, device="cuda").half()
    with pytest.raises(ValueError, match="overlap"):
        copy_pages(base[:8], base[4:], [0], [1])
    want = base.clone()
    want[1], want[7] = want[0], want[6]
    copy_pages(base[:6], base[6:], [0], [1])
    assert torch.equal(base, want)
