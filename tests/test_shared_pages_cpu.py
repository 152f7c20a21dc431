"""Host bookkeeping of shared pages (batched.py PagePool): fork, copy on write,
release by reference count, compaction."""
import random

import pytest

from batched import PAGE, PagePool


def _consistent(pp):
    held = [p for row in pp.table for p in row if p >= 0]
    for page in range(pp.num_pages):
        assert pp.refs[page] == held.count(page)
    assert sorted(pp.free) == [p for p in range(pp.num_pages) if pp.refs[p] == 0]


def test_fork_shares_full_pages_and_gives_a_tail_page():
    pp = PagePool(num_pages=10, num_seqs=4, max_pages=4)
    pp.reserve(0, 2 * PAGE + 9)
    assert pp.fork(0, [1, 3], 2 * PAGE + 10) == [3, 4]
    assert pp.table[1] == [0, 1, 3, -1] and pp.table[3] == [0, 1, 4, -1]
    assert pp.refs[:5] == [3, 3, 1, 1, 1] and pp.in_use == 5
    _consistent(pp)


@pytest.mark.parametrize("length,tables", [(0, [-1, -1]), (PAGE, [0, -1]), (1, [2, -1])])
def test_fork_lengths(length, tables):
    pp = PagePool(num_pages=4, num_seqs=2, max_pages=2)
    pp.reserve(0, 2 * PAGE - 1)
    new = pp.fork(0, [1], length)
    assert pp.table[1] == tables and new == [2 if length == 1 else -1]
    _consistent(pp)


def test_fork_refusals_change_nothing():
    pp = PagePool(num_pages=4, num_seqs=4, max_pages=3)
    pp.reserve(0, PAGE + 5)
    pp.reserve(3, 0)
    for args, err in [((0, [1], 2 * PAGE + 1), ValueError),      # positions without a page
                      ((0, [0], 5), ValueError), ((0, [1, 1], 5), ValueError), ((0, [3], 5), ValueError),
                      ((0, [4], 5), ValueError), ((5, [1], 5), ValueError), ((0, [1], -1), ValueError),
                      ((0, [1, 2], PAGE + 5), RuntimeError)]:    # one free page, two tails
        with pytest.raises(err):
            pp.fork(*args)
        assert pp.in_use == 3 and pp.table[1] == [-1] * 3 and pp.table[2] == [-1] * 3
        _consistent(pp)


def test_unshare_before_a_write():
    pp = PagePool(num_pages=8, num_seqs=3, max_pages=3)
    pp.reserve(0, 2 * PAGE - 1)
    pp.fork(0, [1, 2], 2 * PAGE)
    assert pp.unshare(1, 40, 2 * PAGE - 1) == [(0, 2, 40), (1, 3, 0)]
    assert pp.unshare(1, 0, 2 * PAGE - 1) == []                  # now its own
    assert pp.unshare(0, PAGE + 3, PAGE + 3) == [(1, 4, 3)]
    assert pp.unshare(2, PAGE + 3, PAGE + 3) == []               # the last holder writes in place
    _consistent(pp)


def test_claim_changes_nothing_when_the_pool_is_exhausted():
    pp = PagePool(num_pages=3, num_seqs=2, max_pages=3)
    pp.reserve(0, 2 * PAGE - 1)
    pp.fork(0, [1], 2 * PAGE)
    with pytest.raises(RuntimeError, match="exhausted"):
        pp.claim(1, 2 * PAGE - 1, 2 * PAGE)                      # a page of its own and a new one; one is free
    assert pp.table[1] == [0, 1, -1] and pp.in_use == 2
    _consistent(pp)
    assert pp.claim(1, 2 * PAGE, 2 * PAGE) == (True, []) and pp.table[1] == [0, 1, 2]
    _consistent(pp)


def test_shared_pages_are_freed_with_their_last_holder():
    pp = PagePool(num_pages=4, num_seqs=3, max_pages=2)
    pp.reserve(0, PAGE - 1)
    pp.fork(0, [1, 2], PAGE)
    pp.release(0)
    pp.release(1)
    assert pp.in_use == 1
    pp.release(2)
    assert pp.in_use == 0
    _consistent(pp)


@pytest.mark.parametrize("seed", range(20))
def test_random_sequences_of_calls(seed):
    """Every sequence keeps seeing its own pages' contents through any order of
    calls: page contents are simulated by the labels written into them."""
    r = random.Random(seed)
    pp = PagePool(num_pages=40, num_seqs=8, max_pages=6)
    content = [dict() for _ in range(40)]                        # page -> {offset: label}
    want = [dict() for _ in range(8)]                            # sequence -> {position: label}
    length = [0] * 8
    for step in range(120):
        s = r.randrange(8)
        op = r.choice(["write", "write", "fork", "release", "compact", "rewind"])
        try:
            if op == "write":
                n = r.randint(1, 90)
                lo, hi = length[s], length[s] + n - 1
                if hi >= 6 * PAGE:
                    continue
                pp.reserve(s, hi)
                for a, b, t in pp.unshare(s, lo, hi):
                    content[b] = {k: v for k, v in content[a].items() if k < t}
                for p in range(lo, hi + 1):
                    content[pp.table[s][p // PAGE]][p % PAGE] = want[s][p] = (step, p)
                length[s] = hi + 1
            elif op == "rewind":
                length[s] = r.randint(0, length[s])
                want[s] = {p: v for p, v in want[s].items() if p < length[s]}
            elif op == "fork":
                kids = [k for k in range(8) if k != s and length[k] == 0 and pp.table[k] == [-1] * 6][:2]
                n = r.randint(0, length[s])
                for k, page in zip(kids, pp.fork(s, kids, n)):
                    if page >= 0:
                        src = pp.table[s][n // PAGE]
                        content[page] = {o: v for o, v in content[src].items() if o < n % PAGE}
                    length[k], want[k] = n, {p: v for p, v in want[s].items() if p < n}
            elif op == "release":
                pp.release(s)
                length[s], want[s] = 0, {}
            else:
                src, dst = pp.compact()
                assert not set(src) & set(dst)
                for a, b in zip(src, dst):
                    content[b] = dict(content[a])
                assert all(p < pp.in_use for row in pp.table for p in row)
        except RuntimeError as e:
            assert "exhausted" in str(e)
        _consistent(pp)
        for q in range(8):
            for p, v in want[q].items():
                assert content[pp.table[q][p // PAGE]][p % PAGE] == v
