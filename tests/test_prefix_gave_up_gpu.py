"""Rows of shared_prefix_attention after a wait of the prefix kernel gave up:
its partial results are not what the workspace holds, and the rows that need
them say so.  No wait runs out here: the code that it would have recorded is
written into the plan's status word."""
import pytest
import torch

from paged_helpers import Case

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
PW_ERR = 12                                             # the plan's word that holds the place of its status


def _plant(plan, code):
    at = int(plan.header[PW_ERR])
    plan.words[at:at + 2] = torch.tensor([7, code], dtype=torch.int32)   # the code is the upper half


@pytest.mark.parametrize("dtype,dim,kv,ratio,page,rows,prefix,own,longest", [
    (F16, 128, 2, 2, 128, 5, 640, [40, 3], None),          # joined by the own kernel
    (BF16, 64, 8, 2, 32, 130, 640, [40, 3, 70], None),     # one-warp own CTAs
    (F16, 128, 1, 2, 128, 5, 3000, [700, 40], 6000),       # joined by the join kernel
])
def test_rows_that_share_a_prefix_are_nan(dtype, dim, kv, ratio, page, rows, prefix, own, longest):
    c = Case(dtype, dim, kv, ratio, page, [rows], [prefix], own, seed=40)
    c.lengths[1] = prefix - 1
    c.lengths[3] = 0
    plan = c.plan() if longest is None else c.plan(max_length=longest)
    good, lse0 = c.run(plan)
    c.check(good, lse0)
    # A plan shares whole blocks of 16 tokens: shorter rows run on their own pages.
    alone = [r for r in range(rows) if int(c.lengths[r]) < prefix // 16 * 16]
    assert 3 in alone
    rest = [r for r in range(rows) if r not in alone]
    _plant(plan, 1)
    for _ in range(2):                                  # until the status is read
        out, lse = c.run(plan)
        assert bool(torch.isnan(out[rest]).all()) and bool(torch.isnan(lse[rest]).all())
        assert torch.equal(out[alone], good[alone]) and torch.equal(lse[alone], lse0[alone])
    assert plan.status() == 1 and plan.status() == 0
    out, lse = c.run(plan)
    assert torch.equal(out, good) and torch.equal(lse, lse0)
    _plant(plan, 3)                                     # a skipped page loses nothing else
    out, lse = c.run(plan)
    assert torch.equal(out, good) and torch.equal(lse, lse0) and plan.status() == 3
