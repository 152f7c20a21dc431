"""copy_pages, fork_pages, compact_pages and free_pages (paged.py,
include/qwen_b200_paged.h): every byte of the pools and every table entry
against plain indexing on the host."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

# pages, layers, kv heads, tokens of a page, dim, dtype
GEOMETRIES = [
    (40, 2, 8, 128, 128, torch.float16),
    (300, 1, 2, 16, 64, torch.bfloat16),
    (64, 3, 1, 48, 8, torch.float16),        # rows of 16 bytes
    (50, 1, 3, 7, 24, torch.float16),        # odd page, 48-byte tokens
    (30, 2, 2, 32, 64, torch.float8_e4m3fn),
    (20, 28, 8, 16, 128, torch.float32),
]
IDS = [str(i) for i in range(len(GEOMETRIES))]


def _pools(geo, seed):
    g = torch.Generator().manual_seed(seed)
    shape, dtype = geo[:5], geo[5]
    size = torch.empty(0, dtype=dtype).element_size()
    raw = [torch.randint(0, 256, (*shape[:4], shape[4] * size), dtype=torch.uint8, generator=g) for _ in range(2)]
    return raw, [r.cuda().view(dtype) for r in raw]


def _same(raw, pools):
    for r, p in zip(raw, pools):
        assert torch.equal(p.view(torch.uint8).cpu(), r)


@pytest.mark.parametrize("geo", GEOMETRIES, ids=IDS)
@pytest.mark.parametrize("partial", [False, True])
def test_copy(geo, partial):
    from paged import copy_pages
    r = random.Random(1)
    raw, pools = _pools(geo, 1)
    n = geo[0] // 3
    order = r.sample(range(geo[0]), 2 * n)
    src, dst = order[:n], order[n:]
    src[1] = src[0]                                       # one source to two places
    tokens = [r.randint(0, geo[3]) for _ in src] if partial else None
    copy_pages(*pools, src, dst, tokens)
    for x in raw:
        for i, (a, b) in enumerate(zip(src, dst)):
            t = tokens[i] if partial else geo[3]
            x[b, :, :, :t] = x[a, :, :, :t]
    _same(raw, pools)


@pytest.mark.parametrize("geo", GEOMETRIES, ids=IDS)
def test_fork(geo):
    from paged import fork_pages, pages_status
    r = random.Random(2)
    raw, pools = _pools(geo, 2)
    page, wide = geo[3], 5
    lens = [0, 1, page, 2 * page, 2 * page + 3, 3 * page - 1]
    free = list(range(geo[0]))
    r.shuffle(free)
    table = torch.full((20, wide), -1, dtype=torch.int32)
    for p, n in enumerate(lens):
        for i in range(-(-n // page)):
            table[p, i] = free.pop()
    table[6:] = 3                                         # stale rows of the children
    parents = [4, 0, 1, 2, 3, 4, 5, 4, 5]
    children = [7, 6, 9, 10, 8, 15, 12, 13, 19]
    cut = [lens[p] for p in parents]
    cut[5] = page + 1                                     # fewer positions than the parent has
    new = [free.pop() if n % page else -1 for n in cut]
    dev = table.cuda()
    fork_pages(dev, *pools, parents, children, cut, new)
    for p, c, n, x in zip(parents, children, cut, new):
        full, tail = divmod(n, page)
        src = int(table[p, full]) if tail else -1
        row = table[p].clone()
        row[full:] = -1
        if tail:
            row[full] = x
            for y in raw:
                y[x, :, :, :tail] = y[src, :, :, :tail]
        table[c] = row
    assert torch.equal(dev.cpu(), table)
    _same(raw, pools)
    assert pages_status() == 0


@pytest.mark.parametrize("geo", GEOMETRIES, ids=IDS)
def test_free_and_compact(geo):
    from paged import compact_pages, free_pages
    r = random.Random(3)
    raw, pools = _pools(geo, 3)
    order = r.sample(range(geo[0]), geo[0] - 2)
    table = torch.full((6, geo[0]), -1, dtype=torch.int32)
    for i, x in enumerate(order):
        table[i % 6, i // 6] = x
    table[5, :3] = table[4, :3]                           # shared pages
    dev = torch.full((6, geo[0] + 3), -9, dtype=torch.int32, device="cuda")[:, :geo[0]]
    dev.copy_(table)
    free_pages(dev, [1, 3, 1])
    table[1], table[3] = -1, -1
    assert torch.equal(dev.cpu(), table)
    used = sorted({x for x in table.flatten().tolist() if x >= 0})
    src = [x for x in used if x >= len(used)]
    dst = [x for x in range(len(used)) if x not in used]
    r.shuffle(dst)
    compact_pages(dev, *pools, src, dst)
    for a, b in zip(src, dst):
        table[table == a] = b
        for x in raw:
            x[b] = x[a]
    assert torch.equal(dev.cpu(), table)
    assert bool((dev._base[:, geo[0]:] == -9).all())
    _same(raw, pools)


def test_lists_longer_than_one_launch():
    from paged import compact_pages, copy_pages, fork_pages, free_pages
    geo = (6000, 1, 1, 2, 16, torch.float16)
    raw, pools = _pools(geo, 4)
    order = torch.randperm(6000, generator=torch.Generator().manual_seed(4)).tolist()
    copy_pages(*pools, order[:2500], order[2500:5000], torch.ones(2500, dtype=torch.int64))
    for x in raw:
        x[order[2500:5000], :, :, :1] = x[order[:2500], :, :, :1]
    _same(raw, pools)
    table = torch.full((3001, 2), -1, dtype=torch.int32)
    table[0, 0], table[0, 1] = order[0], order[1]
    dev = table.cuda()
    children = list(range(1, 3001))
    fork_pages(dev, *pools, [0] * 3000, children, [3] * 3000, order[2:3002])
    table[1:, 0] = order[0]
    table[1:, 1] = torch.tensor(order[2:3002], dtype=torch.int32)
    for x in raw:
        x[order[2:3002], :, :, :1] = x[order[1], :, :, :1]
    assert torch.equal(dev.cpu(), table)
    _same(raw, pools)
    compact_pages(dev, *pools, order[2:2002], order[3500:5500])
    table[1:2001, 1] = torch.tensor(order[3500:5500], dtype=torch.int32)
    for x in raw:
        x[order[3500:5500]] = x[order[2:2002]]
    assert torch.equal(dev.cpu(), table)
    _same(raw, pools)
    free_pages(dev, children[:2000])
    table[1:2001] = -1
    assert torch.equal(dev.cpu(), table)


def test_bad_parent_page_is_skipped_and_recorded():
    from paged import fork_pages, pages_status
    geo = (10, 1, 2, 16, 64, torch.float16)
    raw, pools = _pools(geo, 5)
    dev = torch.tensor([[0, -1, -1], [1, 400, -1], [7, 7, 7], [7, 7, 7]], dtype=torch.int32, device="cuda")
    fork_pages(dev, *pools, [0, 1], [2, 3], [20, 20], [4, 5])
    assert pages_status() == 3 and pages_status() == 0
    assert dev.cpu().tolist()[2:] == [[0, 4, -1], [1, 5, -1]]
    _same(raw, pools)


def test_captured_calls_replay():
    from paged import compact_pages, copy_pages, free_pages
    geo = (12, 2, 2, 16, 64, torch.float16)
    raw, pools = _pools(geo, 6)
    dev = torch.tensor([[9, 3], [2, 8]], dtype=torch.int32, device="cuda")
    start = dev.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        copy_pages(*pools, [9], [4], [5])
        free_pages(dev, [1])
        compact_pages(dev, *pools, [9], [0])
    for _ in range(2):
        dev.copy_(start)
        g.replay()
    for x in raw:
        x[4, :, :, :5] = x[9, :, :, :5]
        x[0] = x[9]
    assert dev.cpu().tolist() == [[0, 3], [-1, -1]]
    _same(raw, pools)


def test_offsets_past_32_bits():
    from paged import copy_pages
    shape = (70, 8, 8, 128, 512)                          # 2.3e9 elements
    k = torch.zeros(shape, dtype=torch.float16, device="cuda")
    v = torch.zeros(shape, dtype=torch.float16, device="cuda")
    k[69] = 1.0
    v[69] = 2.0
    copy_pages(k, v, [69], [68], [100])
    assert bool((k[68, :, :, :100] == 1).all()) and bool((v[68, :, :, :100] == 2).all())
    assert not bool(k[68, :, :, 100:].any()) and not bool(k[:68].any())


def test_lists_of_every_kind():
    """Lists, tuples, ranges, generators, arrays and tensors of integers."""
    import numpy as np
    from paged import copy_pages
    geo = (12, 1, 2, 16, 64, torch.float16)
    raw, (k, v) = _pools(geo, 8)
    kinds = [list, tuple, iter, np.array, torch.tensor, lambda x: torch.tensor(x, dtype=torch.int32)[::1],
             lambda x: torch.tensor([y for z in x for y in (z, 99)])[::2]]
    for i, kind in enumerate(kinds):
        copy_pages(k, v, kind([0, 1]), kind([4 + i % 4, 8 + i % 4]), kind([16, 9]))
        for pool, r in zip((k, v), raw):
            r[4 + i % 4], r[8 + i % 4, :, :, :9] = r[0], r[1, :, :, :9]
        _same(raw, (k, v))
    copy_pages(k, v, range(0), [], ())


def test_refusals_leave_the_pools_alone():
    from paged import compact_pages, copy_pages, fork_pages, free_pages
    geo = (10, 1, 2, 16, 64, torch.float16)
    raw, (k, v) = _pools(geo, 7)
    table = torch.tensor([[0, 1], [-1, -1]], dtype=torch.int32, device="cuda")
    for call, what in [
            (lambda: copy_pages(k, v, [0], [1, 2]), "entries"),
            (lambda: copy_pages(k, v, [0, 1], [1, 2]), "also a source"),
            (lambda: copy_pages(k, v, [0], [10]), "outside the pool"),
            (lambda: copy_pages(k, v, [0], [1 << 40]), "32 bits"),
            (lambda: copy_pages(k, v, torch.tensor([0]), torch.tensor([1 << 40])), "32 bits"),
            (lambda: copy_pages(k, v, torch.tensor([0.0]), [1]), "list of integers"),
            (lambda: copy_pages(k, v, torch.tensor([0], device="cuda"), [1]), "list of integers"),
            (lambda: copy_pages(k, v, torch.tensor([[0]]), [1]), "list of integers"),
            (lambda: copy_pages(k, v, [0.0], [1]), "list of integers"),
            (lambda: copy_pages(k, v, [[0]], [1]), "list of integers"),
            (lambda: copy_pages(k, v, ["0"], [1]), "list of integers"),
            (lambda: copy_pages(k, v, 0, [1]), "list of integers"),
            (lambda: copy_pages(k, v, [0], [1], 5), "list of integers"),
            (lambda: copy_pages(k, v, [-(1 << 70)], [1]), "32 bits"),
            (lambda: copy_pages(k[:, :, :, :8], v[:, :, :, :8], [0], [1]), "contiguous"),
            (lambda: copy_pages(k, v[:5], [0], [1]), "same shape"),
            (lambda: copy_pages(k, k, [0], [1]), "same pool"),
            (lambda: copy_pages(k[..., :4].contiguous(), v[..., :4].contiguous(), [0], [1]), "multiple of 16"),
            (lambda: fork_pages(table, k, v, [0], [0], [20], [5]), "also a parent"),
            (lambda: fork_pages(table.long(), k, v, [0], [1], [20], [5]), "int32"),
            (lambda: fork_pages(table.cpu(), k, v, [0], [1], [20], [5]), "CUDA"),
            (lambda: compact_pages(table, k, v, [5, 5], [2, 3]), "moves twice"),
            (lambda: free_pages(table, [2]), "outside the table")]:
        with pytest.raises(ValueError, match=what):
            call()
    assert table.cpu().tolist() == [[0, 1], [-1, -1]]
    _same(raw, (k, v))
