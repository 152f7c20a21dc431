"""The softmax weights of shared_prefix_attention: a long tail behind one
dominant token, and tokens that alone decide a row's result, one at each place
where the work is cut (tiles of 128 tokens, parts of the plan, splits of the own
part, the border of the prefix, blocks of 16 tokens, pages)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16

# fp16 weights are held to 11 bits, or to 2^-32 of their row's largest weight
# where that is more (half of fp16's smallest step, 2^-25, of weights kept 2^7
# times larger).
FLOOR = {F16: 2.0 ** -32, BF16: 0.0}


def _pools(k, v, page, seed):
    """k, v [kv heads, n, dim] as pages in no order: pools, and the page of each `page` tokens."""
    kv, n, d = k.shape
    pages = -(-n // page)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))
    pools = []
    for x in (k, v):
        pool = torch.full((pages, kv, page, d), math.nan, dtype=x.dtype)
        for i in range(pages):
            part = x[:, i * page:(i + 1) * page]
            pool[order[i], :, :part.shape[1]] = part
        pools.append(pool.cuda())
    return pools, order.int()


def _run(q, pools, order, n, plan):
    """Rows of n tokens with a table row each, all of them over the same pages."""
    from paged import shared_prefix_attention
    rows = q.shape[0]
    ids = torch.arange(rows, dtype=torch.int32, device="cuda")
    out, lse = shared_prefix_attention(q.cuda(), *pools, order.repeat(rows, 1).cuda(), ids, torch.full_like(ids, n),
                                       plan, return_lse=True)
    assert plan.status() == 0
    return out.double().cpu(), lse.double().cpu()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n,prefix,longest", [
    (30000, 29952, 30000),      # the prefix kernel
    (30000, 0, 30000),          # the own kernel, split over many CTAs
    (900, 896, 1000), (900, 0, 900)])
@pytest.mark.parametrize("gap", [14.0, 17.0, 18.0])
@pytest.mark.parametrize("at", [0, -1])
def test_a_tail_behind_a_dominant_token(dtype, n, prefix, longest, gap, at):
    """The dominant token's value is 0: what the row gives is its tail, of
    weight e^-gap each and n e^-gap together.

    Bounds: a score is off by e (products exact in fp32, each of 128 additions
    by 2^-23 of what was added at most), so a normalised weight by w (2 e +
    2^-19) and its rounding: u w, or FLOOR of the largest one."""
    from paged import PrefixPlan
    g = torch.Generator().manual_seed(3)
    d, rows = 128, 2
    k = 0.02 * torch.randn(1, n, d, generator=g)
    k[..., 0] = 0.0
    k[0, at, 0] = gap / 1.4142135
    v = 1.0 + 0.25 * torch.randn(1, n, d, generator=g)
    v[0, at] = 0.0
    q = 0.1 * torch.randn(rows, 1, d, generator=g)
    q[..., 0] = 16.0                                    # x dim^-0.5 = 1.414
    q, k, v = (x.to(dtype) for x in (q, k, v))
    pools, order = _pools(k, v, 128, 1)
    out, lse = _run(q, pools, order, n, PrefixPlan([rows], [prefix], 1, 1, d, max_length=longest))
    qd, kd, vd = q.double()[:, 0], k.double()[0], v.double()[0]
    s = qd @ kd.T * d ** -0.5
    w = torch.softmax(s, -1)
    ref = w @ vd
    e = d * 2.0 ** -23 * d ** -0.5 * (qd.abs() @ kd.abs().T)
    u = torch.finfo(dtype).eps / 2
    # The largest error of a score bounds that of the sum, each weight has its own.
    off = w * (u + e + e.amax(-1, keepdim=True) + 2.0 ** -19) + FLOOR[dtype] * w.amax(-1, keepdim=True)
    tiny = 2.0 ** -25 if dtype == F16 else 0.0          # the smallest step of the output
    bound = off @ vd.abs() + u * ref.abs() + tiny
    err = (out[:, 0] - ref).abs()
    assert bool((err <= bound).all()), f"{float((err / bound).max())} times the bound, {float((err / ref.abs()).max())} of the result"
    want = torch.logsumexp(s, -1)
    assert bool(((lse[:, 0] - want).abs() <= 2 * e.amax(-1) + 2.0 ** -19 + 2.0 ** -22 * want.abs()).all())


def _needles(n, prefix, own_from):
    """Every border of 16 tokens and its two neighbours, thinned to about 1,500 of them, and the ends."""
    at = {0, 1, n - 2, n - 1, prefix - 1, prefix, own_from - 1, own_from}
    for b in range(16, n, 16 if n < 8000 else 128):
        at |= {b - 1, b}
    return sorted(x for x in at if 0 <= x < n)


@pytest.mark.parametrize("dtype,dim,ratio,page,n,prefix,rows,longest", [
    (F16, 128, 2, 128, 2200, 1920, 4, 2300),            # a prefix in parts of two tiles, an own part of 280
    (F16, 128, 2, 128, 2200, 1900, 4, 6000),            # cut inside a block of 16; own part split
    (BF16, 64, 4, 16, 1100, 1000, 3, 1100),             # small pages
    (F16, 128, 8, 64, 700, 640, 40, 700),               # 320 queries: a pair of tiles and a single one
    (BF16, 128, 2, 128, 1300, 0, 2, 1300),              # nothing shared: own splits
    (F16, 64, 2, 32, 9000, 8000, 2, 9000),
    (BF16, 128, 1, 48, 30000, 29000, 3, 30000),
    (F16, 128, 2, 128, 250, 128, 2, 250),               # one CTA alone
])
def test_a_token_that_decides_is_counted_once(dtype, dim, ratio, page, n, prefix, rows, longest):
    """Query j points along dimension j and one token's key does too, far
    enough that its weight is all but 1: the result is that token's value and
    the logarithm is its score.  A token left out would give the mean of the
    others, one counted twice ln 2 more.  One call asks for dim tokens."""
    from paged import PrefixPlan
    plan = PrefixPlan([rows], [prefix], ratio, 1, dim, max_length=longest)
    g = torch.Generator().manual_seed(4)
    at = _needles(n, prefix, prefix // 16 * 16)
    v = torch.randn(1, n, dim, generator=g).to(dtype)
    base = (0.02 * torch.randn(1, n, dim, generator=g)).to(dtype)
    heads = ratio
    scale = dim ** -0.5
    u = torch.finfo(dtype).eps / 2
    for i in range(0, len(at), dim):
        some = at[i:i + dim]
        k = base.clone()
        k[0, some, :] = 0.0
        k[0, some, range(len(some))] = 20.0
        pools, order = _pools(k, v, page, 1)
        for first in range(0, len(some), rows * heads):
            mine = some[first:first + rows * heads]
            q = torch.zeros(rows * heads, dim)
            q[range(len(mine)), range(first, first + len(mine))] = 32.0
            q = q.reshape(rows, heads, dim).to(dtype)
            out, lse = _run(q, pools, order, n, plan)
            out, lse = out.reshape(-1, dim)[:len(mine)], lse.reshape(-1)[:len(mine)]
            s = q.double().reshape(-1, dim)[:len(mine)] @ k.double()[0].T * scale
            ref = torch.softmax(s, -1) @ v.double()[0]
            e = dim * 2.0 ** -23 * scale * 640.0
            rest = n * math.exp(-40.0)                  # what the other tokens weigh: 640 scale - 3 > 40
            bound = (2 * u + 4 * e + 2.0 ** -18) * ref.abs() + 8.0 * rest + 2.0 ** -24
            assert bool(((out - ref).abs() <= bound).all())
            assert bool(((lse - torch.logsumexp(s, -1)).abs() <= 2 * e + 2.0 ** -19 + 2.0 ** -22 * 80).all())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("prefix", [0, 1920])
@pytest.mark.parametrize("size", [100.0, 700.0, 3000.0])
def test_large_finite_scores_stay_finite(dtype, prefix, size):
    """Scores up to 1e7: one step of a score in fp32 is then more than the
    distance between the largest fp16 number and the largest weight."""
    from paged import PrefixPlan
    g = torch.Generator().manual_seed(5)
    n, d = 2000, 128
    q, k = (size * torch.randn(*s, d, generator=g) for s in ((20, 2), (1, n)))
    v = torch.randn(1, n, d, generator=g)
    q, k, v = (x.to(dtype) for x in (q, k, v))
    pools, order = _pools(k, v, 64, 2)
    out, lse = _run(q, pools, order, n, PrefixPlan([20], [prefix], 2, 1, d, max_length=n))
    top = (q.double().reshape(40, d) @ k.double()[0].T * d ** -0.5).amax(-1)
    assert bool(torch.isfinite(out).all()) and float(out.abs().max()) <= 1.01 * float(v.abs().max())
    e = d * 2.0 ** -23 * d ** -0.5 * (q.double().reshape(40, d).abs() @ k.double()[0].abs().T).amax(-1)
    assert bool(((lse.reshape(-1) - top).abs() <= 2 * e + math.log(n) + 2.0 ** -22 * top.abs()).all())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,kv,n,prefix,longest", [
    (128, 8, 8000, 7936, 8000),    # the prefix kernel, several tiles to a part
    (64, 8, 12000, 11904, 12000),
    (128, 1, 450, 0, 450),         # the own kernel alone
    (64, 2, 3000, 0, 3000),        # its splits
    (64, 2, 1900, 640, 4000),      # all three kernels
])
@pytest.mark.parametrize("at", [300, 449, 1500, 4000, 6677, -1])
@pytest.mark.parametrize("rows", [3, 90])
def test_a_dominant_token_is_not_rounded(dtype, dim, kv, n, prefix, longest, at, rows):
    """One token has most of the weight, between two steps of the input type as
    seen from the largest scores before it, which lie 2.2 to 5.2 lower.  The
    result may be off by the roundings of the other weights, u w each, and its
    own (and by 2^-23 of what has been added at each of n / 16 steps of the
    products)."""
    from paged import PrefixPlan
    g = torch.Generator().manual_seed(6)
    at = at % n
    before = [at - x for x in (16, 32, 64, 128, 256, 384) if x <= at]
    k = 0.01 * torch.randn(kv, n, dim, generator=g)
    k[..., :2] = 0.0
    k[:, before + [at]] = 0.0
    k[:, at, 0], k[:, before, 1] = 8.0, 8.0
    v = torch.randn(kv, n, dim, generator=g)
    q = 0.05 * torch.randn(rows, 2 * kv, dim, generator=g)
    q[..., 0] = 14.0 / 8.0 * dim ** 0.5
    q[..., 1] = ((14.0 - torch.linspace(2.2, 5.2, 2 * kv * rows)) / 8.0 * dim ** 0.5).view(rows, 2 * kv)
    q, k, v = (x.to(dtype) for x in (q, k, v))
    pools, order = _pools(k, v, 128, 3)
    out, _ = _run(q, pools, order, n, PrefixPlan([rows], [prefix], 2 * kv, kv, dim, max_length=longest))
    qd, kd, vd = (x.double().cuda() for x in (q.view(rows, kv, 2, dim).transpose(0, 1).reshape(kv, -1, dim), k, v))
    w = torch.softmax(qd @ kd.mT * dim ** -0.5, -1)
    ref = w @ vd
    e = dim * 2.0 ** -23 * dim ** -0.5 * (qd.abs() @ kd.abs().mT)
    u = torch.finfo(dtype).eps / 2
    others = w.clone()
    others[..., at] = 0.0
    off = u * others + w * (e + e.amax(-1, keepdim=True) + 2.0 ** -19 + n / 16 * 2.0 ** -23)
    off += FLOOR[dtype] * w.amax(-1, keepdim=True)
    bound = off @ vd.abs() + u * ref.abs() + 2.0 ** -25
    err = (out.view(rows, kv, 2, dim).transpose(0, 1).reshape(kv, -1, dim).cuda() - ref).abs()
    heavy = w[..., at] > 0.5
    assert bool(heavy.any())
    assert bool((err <= bound)[heavy].all()), f"{float((err / bound)[heavy].max())} times the bound"
