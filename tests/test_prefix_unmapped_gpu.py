"""Rows of shared_prefix_attention that see nothing but unmapped pages: the
same result whichever kernel the plan gives them to."""
import math

import pytest
import torch

from paged_helpers import Case

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.parametrize("missing", [-1, 10_000])
@pytest.mark.parametrize("dtype,dim,ratio,page,rows,prefix,longest", [
    (F16, 128, 2, 32, 4, 128, 200),        # short rows: the own kernel alone
    (F16, 128, 2, 32, 4, 128, 4000),       # the prefix kernel, one tile
    (F16, 128, 2, 128, 4, 768, 800),       # a CTA per tile
    (BF16, 64, 4, 16, 40, 1008, 1100),     # parts of two tiles, whose streams are joined
    (BF16, 128, 8, 64, 30, 1600, 1700),    # pairs of query tiles
    (F16, 128, 2, 128, 3, 0, 900),         # nothing shared, own splits
])
def test_rows_without_a_mapped_page(dtype, dim, ratio, page, rows, prefix, longest, missing):
    """Skipped and recorded, so nothing is seen: 0 and -inf."""
    own = 0 if prefix else 700
    c = Case(dtype, dim, 2, ratio, page, [rows], [prefix], [own], seed=30)
    plan = c.plan(max_length=longest)
    good, good_lse = c.run(plan)
    c.check(good, good_lse)
    table = c.table.clone()
    c.table.fill_(missing)
    out, lse = c.run(plan)
    assert plan.status() == 3
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    # One page left: its tokens alone are seen.
    keep = min(2, table.shape[1] - 2)
    c.table[:, keep] = table[:, keep]
    out, lse = c.run(plan)
    assert plan.status() == 3
    only = Case.__new__(Case)
    only.__dict__.update(c.__dict__)
    only.table = table[:, keep:keep + 1].contiguous()
    only.lengths = torch.full_like(c.lengths, min(page, int(c.lengths[0]) - keep * page))
    only.check(out, lse)
    c.table.copy_(table)
    out, lse = c.run(plan)
    assert plan.status() == 0 and torch.equal(out, good) and torch.equal(lse, good_lse)


def test_scores_of_minus_infinity_beside_unmapped_pages():
    """A page that is seen and gives only scores of -inf makes NaN, one that is not mapped nothing."""
    c = Case(F16, 128, 1, 2, 32, [3], [640], [0], seed=31)
    plan = c.plan(max_length=4000)
    c.q.abs_()
    page = int(c.table[0, 7])
    c.table.fill_(-1)
    c.table[:, 7] = page
    c.k_pool[page] = -math.inf
    out, lse = c.run(plan)
    assert plan.status() == 3 and bool(torch.isnan(out).all()) and bool((lse == -math.inf).all())
