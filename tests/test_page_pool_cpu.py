"""PagePool.claim (batched.py) as a step loop calls it: what it looks at, and
that its result is that of reserve and unshare."""
import copy
import random

import pytest

from batched import PAGE, PagePool


class _Row(list):
    """A table row that counts the entries read from it."""
    read = 0

    def __getitem__(self, i):
        got = super().__getitem__(i)
        _Row.read += len(got) if isinstance(i, slice) else 1
        return got


@pytest.mark.parametrize("pages", [1, 8, 64])
def test_a_call_that_changes_nothing_looks_at_each_page_once(pages):
    """256 sequences call it before every step: one look at the pages up to the
    position, one at those that are written."""
    pp = PagePool(num_pages=70, num_seqs=2, max_pages=64)
    pp.reserve(0, pages * PAGE - 1)
    pp.table[0] = _Row(pp.table[0])
    _Row.read = 0
    assert pp.claim(0, pages * PAGE - 1, pages * PAGE - 1) == (False, [])
    assert _Row.read <= pages + 2


@pytest.mark.parametrize("seed", range(30))
def test_claim_is_reserve_and_unshare(seed):
    r = random.Random(seed)
    pp = PagePool(num_pages=r.randint(8, 24), num_seqs=5, max_pages=6)
    pp.reserve(0, r.randint(0, 6 * PAGE - 1))
    n = r.randint(0, sum(p >= 0 for p in pp.table[0]) * PAGE)
    try:
        pp.fork(0, [1, 2, 3], n)
    except RuntimeError:
        pp.fork(0, [1], n // PAGE * PAGE)
    for _ in range(8):
        seq, last = r.randrange(5), r.randint(0, 6 * PAGE - 1)
        first = r.randint(0, last)
        other = copy.deepcopy(pp)
        try:
            got = pp.claim(seq, first, last)
        except RuntimeError:
            assert pp.table == other.table and pp.free == other.free and pp.refs == other.refs
            continue
        assert got == (other.reserve(seq, last), other.unshare(seq, first, last))
        assert pp.table == other.table and pp.free == other.free and pp.refs == other.refs
        assert all(pp.refs[p] == 1 for p in pp.table[seq][first // PAGE:last // PAGE + 1])
    for bad in ((5, 0, 0), (0, 0, -1), (0, 0, 6 * PAGE)):
        with pytest.raises(ValueError, match="outside the page table"):
            pp.claim(*bad)


@pytest.mark.parametrize("kind", ["list", "numpy", "tensor"])
def test_fork_takes_integers_of_any_type(kind):
    """The same child twice is the same child, also as two numbers that are not the same object."""
    import numpy as np
    import torch
    make = {"list": list, "numpy": np.array, "tensor": torch.tensor}[kind]
    pp = PagePool(num_pages=8, num_seqs=4, max_pages=3)
    pp.reserve(0, PAGE + 5)
    before = copy.deepcopy(pp.__dict__)
    for children in ([1, 1], [1, 0], [2, 4]):
        with pytest.raises(ValueError):
            pp.fork(make([0])[0], make(children), make([PAGE + 6])[0])
        assert pp.__dict__ == before
    assert pp.fork(make([0])[0], make([3, 1]), make([PAGE + 6])[0]) == [2, 3]
    assert pp.table == [[0, 1, -1], [0, 3, -1], [-1] * 3, [0, 2, -1]] and pp.refs[:4] == [3, 1, 1, 1]
    assert all(type(x) is int for row in pp.table for x in row)


@pytest.mark.parametrize("args", [(0.0, [1], 5), (0, [1.0], 5), (0, [1], 5.0), (0, [None], 5), (0, 1, 5)])
def test_fork_refuses_what_is_no_integer(args):
    pp = PagePool(num_pages=8, num_seqs=4, max_pages=3)
    pp.reserve(0, PAGE + 5)
    before = copy.deepcopy(pp.__dict__)
    with pytest.raises(ValueError):
        pp.fork(*args)
    assert pp.__dict__ == before
