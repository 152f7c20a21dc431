"""shared_prefix_attention (paged.py, include/qwen_b200_paged.h) against the
64-bit definition, elementwise within bounds that count its roundings
(paged_helpers.attention_reference).  Every unused place of the pools is NaN."""
import math

import pytest
import torch

from paged_helpers import Case

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16

# dtype, dim, kv heads, ratio, page, sequences per group, prefix per group, own lengths, tokens per sequence
CASES = [
    (F16, 128, 8, 2, 128, [2], [128], [1, 8], 1),              # smallest: one tile, one own token
    (F16, 128, 8, 2, 128, [4], [16], [1], 1),                  # one step of the products
    (F16, 128, 2, 2, 128, [3], [15], [1, 2], 1),               # below a step: all own
    (F16, 128, 2, 2, 128, [3], [129], [5, 300, 64], 1),        # one token behind a tile
    (BF16, 128, 2, 2, 128, [3], [255], [1, 17], 1),
    (F16, 64, 2, 4, 16, [5], [1000], [3, 70, 16, 15, 17], 1),  # small pages, prefix inside a page
    (BF16, 64, 4, 1, 32, [33], [700], [1, 40], 1),             # one head per kv head, odd rows
    (BF16, 128, 1, 8, 64, [40], [1300], [9, 130], 1),          # 320 queries: a full pair and a single tile
    (F16, 128, 1, 16, 48, [9], [500], [31, 1, 200], 1),        # two head tiles, pages of 48
    (F16, 128, 2, 5, 128, [60], [640], [3, 50], 1),            # 300 queries, heads of a row in two tiles
    (F16, 64, 1, 2, 16, [200], [333], [1], 1),                 # many rows, one own token
    (F16, 128, 2, 2, 128, [1, 3, 1, 2], [500, 260, 0, 128], [4, 90, 1], 1),   # groups of one, no prefix
    (BF16, 64, 2, 3, 32, [2, 70, 5, 1], [96, 2000, 33, 64], [1, 33, 500], 1),
    (F16, 128, 2, 2, 64, [6], [400], [8, 30], 8),              # draft tokens: rows of one sequence
    (F16, 128, 2, 2, 128, [4], [0], [1, 700, 2000, 128], 1),   # nothing shared: paged attention
    (F16, 128, 1, 2, 128, [3], [9000], [2100, 1, 77], 1),      # long, few rows: split over many CTAs
    (F16, 64, 1, 1, 256, [2], [512], [256, 1], 1),             # pages of two tiles
    # Batches of over 1480 (row, kv head) pairs: one-warp CTAs for the own parts.
    (F16, 128, 8, 2, 128, [190], [256], [1, 130, 33, 32, 64, 257], 1),
    (BF16, 64, 8, 4, 16, [100, 90], [48, 160], [1, 95, 16, 63, 64, 65, 300], 1),
    (F16, 128, 8, 2, 64, [25], [200], [9, 40, 70, 128], 8),    # runs of four rows
    (BF16, 128, 4, 3, 32, [60, 1, 20], [128, 100, 64], [6, 41, 12], 5),  # runs of two, an odd row left
    (F16, 64, 8, 16, 16, [95], [32], [3, 80], 1),              # two head tiles
    (F16, 128, 8, 1, 128, [200], [0], [1, 2, 100], 1),         # nothing shared
    (F16, 128, 1, 2, 128, [1, 2, 1], [5000, 300, 1500], [20, 3], 1),     # long prefixes of single rows
    (BF16, 128, 1, 4, 64, [40], [3000], [5, 60], 8),           # many partial results: a join of its own
    (F16, 128, 2, 2, 16, [1, 1, 1], [4000, 30, 1500], [20, 3, 700], 1),  # single rows alone
    (F16, 64, 1, 2, 32, [1, 3], [0, 64], [9500, 30, 200], 1),  # one row far longer than the others
]


@pytest.mark.parametrize("longest", [None, 4000])           # as it is; told to be long (other plans, other splits)
@pytest.mark.parametrize("i", range(len(CASES)))
def test_matches_the_definition(i, longest):
    c = Case(*CASES[i], seed=100 + i)
    plan = c.plan() if longest is None else c.plan(max_length=longest)
    c.check(*c.run(plan))
    assert plan.status() == 0


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("layout", ["hnd", "nhd"])
def test_layouts_and_strides(dtype, layout):
    c = Case(dtype, 128, 4, 2, 32, [6], [200], [1, 60], layout=layout, layers=3, seed=5)
    qkv = torch.zeros(c.q.shape[0], 40, 128, dtype=dtype, device="cuda")
    qkv[:, 8:16] = c.q
    c.q = qkv[:, 8:16]                                  # rows of a fused projection
    big = torch.full((c.q.shape[0], 12, 136), 7.0, dtype=dtype, device="cuda")
    out, lse = c.run(c.plan(), out=big[:, 2:10, :128])
    c.check(out, lse)
    big[:, 2:10, :128] = 7.0
    assert bool((big == 7.0).all())                     # nothing else was written
    assert out.data_ptr() == big[:, 2:10].data_ptr()


def test_tables_with_wider_rows_and_sequences_in_any_order():
    """A window of a larger table, rows of sequences in no order, some twice."""
    c = Case(F16, 128, 2, 2, 32, [7], [300], [20, 90, 1], seed=20)
    n, w = c.table.shape
    wide = torch.full((n + 3, w + 5), 12345, dtype=torch.int32, device="cuda")
    wide[2:2 + n, 3:3 + w] = c.table
    c.table = wide[2:2 + n, 3:3 + w]
    order = torch.tensor([4, 0, 6, 4, 2, 1, 5], device="cuda")
    c.seq_ids, c.lengths = c.seq_ids[order].contiguous(), c.lengths[order].contiguous()
    for longest in (400, 4000):
        plan = c.plan(max_length=longest)
        c.check(*c.run(plan))
        assert plan.status() == 0


def test_calls_of_two_threads():
    """Host threads with a stream and a plan each, at the same time."""
    import threading
    cases = [Case(F16, 128, 2, 2, 32, [9], [700], [20, 90], seed=21), Case(BF16, 64, 4, 1, 16, [3, 30], [100, 900], [7], seed=22)]
    plans = [c.plan() for c in cases]
    want = [c.run(p) for c, p in zip(cases, plans)]
    torch.cuda.synchronize()
    bad = []

    def work(c, p, ref):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                out, lse = c.run(p)
                if not (torch.equal(out, ref[0]) and torch.equal(lse, ref[1])):
                    bad.append(c)
    threads = [threading.Thread(target=work, args=x) for x in zip(cases, plans, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad and all(p.status() == 0 for p in plans)


def test_empty_and_short_rows():
    """Length 0 gives 0 and -inf; a row shorter than its group's prefix is right on its own pages."""
    c = Case(F16, 128, 2, 2, 64, [6], [640], [40, 3], seed=6)
    c.lengths[1], c.lengths[2], c.lengths[3], c.lengths[4] = 0, 1, 639, 640
    plan = c.plan()
    out, lse = c.run(plan)
    c.check(out, lse)
    assert bool((out[1] == 0).all()) and bool((lse[1] == -math.inf).all())
    c.lengths.zero_()
    out, lse = c.run(plan)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    assert plan.status() == 0


def test_lengths_change_under_one_plan():
    c = Case(BF16, 128, 2, 4, 128, [7], [384], [300], seed=7)
    plan = c.plan(max_length=400)                       # longer rows than it was told are still right
    for n in (385, 684, 500, 1, 384):
        c.lengths.fill_(n)
        c.check(*c.run(plan))


def test_large_scores_and_far_maxima():
    """Scores that grow along the sequence move the running maximum many times."""
    c = Case(F16, 128, 1, 2, 128, [70], [1024], [30], seed=8, q_scale=0.5)
    ramp = torch.linspace(0.0, 6.0, 1024, device="cuda").half()
    for s in range(1024 // 128):
        c.k_pool[c.table[0, s].long()] = c.k_pool[c.table[0, s].long()] * 0.1 + ramp[128 * s:128 * s + 128, None]
    c.q += 1.0
    c.check(*c.run(c.plan()))


def test_infinities_and_nan_stay_in_their_rows():
    c = Case(F16, 128, 2, 2, 32, [5], [96], [20], seed=9)
    plan = c.plan()
    before, lse0 = c.run(plan)
    own = c.table[2, 3].long()                          # an own page of sequence 2
    c.v_pool[own, :, 4] = math.nan
    c.k_pool[own, :, 5] = math.inf
    out, lse = c.run(plan)
    keep = [0, 1, 3, 4]
    assert torch.equal(out[keep], before[keep]) and torch.equal(lse[keep], lse0[keep])
    assert bool(torch.isnan(out[2]).all())
    # A NaN in the shared part reaches every row that sees it, and no other.
    c.v_pool[c.table[0, 1].long(), :, 0] = math.nan
    c.lengths[4] = 32                                   # sees page 0 alone
    out, _ = c.run(plan)
    assert bool(torch.isnan(out[:4]).all()) and not bool(torch.isnan(out[4]).any())


@pytest.mark.parametrize("seqs", [3, 60])                   # two-warp and one-warp CTAs
def test_nan_of_a_later_token_stays_out_of_earlier_rows(seqs):
    """Rows of one sequence run together; a token that only the later ones see
    may hold anything."""
    c = Case(BF16, 128, 8, 2, 32, [seqs], [64], [45, 60], tokens=6, seed=14)
    plan = c.plan()
    before, lse0 = c.run(plan)
    last = int(c.lengths[5]) - 1                        # only row 5 of sequence 0 sees it
    page, at = int(c.table[0, last // 32]), last % 32
    c.v_pool[page, :, at] = math.nan
    c.v_pool[page, :, at - 1] = math.inf
    c.k_pool[page, :, at] = math.inf
    out, lse = c.run(plan)
    assert torch.equal(out[:4], before[:4]) and torch.equal(out[6:], before[6:])
    assert torch.equal(lse[:5], lse0[:5]) and torch.equal(lse[6:], lse0[6:])
    assert not bool(torch.isfinite(out[4]).any()) and bool(torch.isnan(out[5]).all())


def test_scores_of_minus_infinity():
    """All visible scores -inf: NaN, as the softmax of nothing else; some: weight 0."""
    c = Case(BF16, 64, 1, 1, 16, [3], [32], [4], seed=10)
    c.q.abs_()
    c.k_pool[c.table[0, 0].long()] = -math.inf          # half of the shared part
    c.check(*c.run(c.plan()))
    for x in c.table[:, :3].flatten().tolist():
        c.k_pool[x] = -math.inf
    out, _ = c.run(c.plan())
    assert bool(torch.isnan(out).all())


@pytest.mark.parametrize("dtype,own", [(F16, [1, 70, 1]), (BF16, [300, 1, 30])])
def test_a_visible_nan_reaches_its_row(dtype, own):
    """Also where it is the only token of a part, whose other parts are finite."""
    c = Case(dtype, 128, 2, 2, 32, [3], [160], own, seed=15)
    plan = c.plan()
    good, lse0 = c.run(plan)
    r = own.index(1)
    at = int(c.lengths[r]) - 1
    page, at = int(c.table[r, at // 32]), at % 32
    k = c.k_pool[page, :, at].clone()
    c.k_pool[page, :, at] = math.nan                    # the row's one own token
    out, lse = c.run(plan)
    keep = [i for i in range(3) if i != r]
    assert torch.equal(out[keep], good[keep]) and torch.equal(lse[keep], lse0[keep])
    assert bool(torch.isnan(out[r]).all()) and bool(torch.isnan(lse[r]).all())
    c.k_pool[page, :, at] = k
    for x in c.table[0, :4].long().tolist():            # the first tile of the shared part
        c.k_pool[x] = math.nan
    out, lse = c.run(plan)
    assert bool(torch.isnan(out).all()) and bool(torch.isnan(lse).all())


@pytest.mark.parametrize("ahead", [1, 40])
def test_padding_ahead_of_a_group(ahead):
    """Rows of length 0, of no sequence or too short to hold the prefix, in
    front of the rows whose pages are the group's."""
    c = Case(F16, 128, 2, 2, 32, [ahead + 3], [300], [20, 70], seed=16)
    plan = c.plan()
    want, lse0 = c.run(plan)
    c.lengths[:ahead] = torch.tensor([0, 5, 299], dtype=torch.int32, device="cuda").repeat(ahead)[:ahead]
    c.table[0] = -1                                     # released
    c.lengths[0] = 0
    out, lse = c.run(plan)
    assert torch.equal(out[ahead:], want[ahead:]) and torch.equal(lse[ahead:], lse0[ahead:])
    assert bool((out[0] == 0).all()) and plan.status() == 0
    c.check(out, lse)
    c.seq_ids[0] = -1
    again, _ = c.run(plan)
    assert plan.status() == 3 and torch.equal(again, out)


def test_rows_of_the_output_that_overlap_are_refused():
    c = Case(F16, 128, 2, 2, 32, [3], [64], [5], seed=17)
    plan = c.plan()
    flat = torch.empty(3 * 4 * 128, dtype=F16, device="cuda")
    for strides in [(128, 128, 1), (384, 128, 1), (128, 256, 1), (64, 192, 1), (512, 0, 1), (0, 128, 1)]:
        with pytest.raises(ValueError, match="overlap"):
            c.run(plan, out=flat.as_strided((3, 4, 128), strides))
    c.check(*c.run(plan, out=flat.as_strided((3, 4, 128), (128, 384, 1))))   # heads outermost
    c.check(*c.run(plan, out=c.q.clone()))


def test_output_in_place_of_the_queries():
    c = Case(BF16, 128, 4, 2, 64, [30, 5], [300, 64], [5, 90], seed=18)
    plan = c.plan()
    want, lse0 = c.run(plan)
    out, lse = c.run(plan, out=c.q)
    assert out.data_ptr() == c.q.data_ptr() and torch.equal(out, want) and torch.equal(lse, lse0)


def test_bad_table_entries_are_skipped_and_recorded():
    c = Case(F16, 128, 2, 2, 32, [4], [128], [40], seed=11)
    plan = c.plan()
    good, _ = c.run(plan)
    c.table[1, 4] = -1                                  # an own page of sequence 1
    c.table[2, 4] = 10_000
    out, _ = c.run(plan)
    assert plan.status() == 3 and plan.status() == 0
    assert torch.equal(out[[0, 3]], good[[0, 3]]) and bool(torch.isfinite(out).all())
    c.seq_ids[3] = 99
    out, lse = c.run(plan)
    assert plan.status() == 3 and bool((out[3] == 0).all()) and bool((lse[3] == -math.inf).all())
    c.seq_ids[3] = 3
    c.lengths[0] = 1 << 30
    c.run(plan)
    assert plan.status() == 3
    c.lengths[0] = 168
    c.table[0, 1] = -1                                  # a shared page, read through row 0: masked for all
    out, lse = c.run(plan)
    assert plan.status() == 3 and bool(torch.isfinite(out).all())


def test_same_bits_again_other_stream_and_graph():
    c = Case(F16, 128, 8, 2, 128, [40], [600], [1, 130, 64], seed=12)
    plan = c.plan()
    out, lse = c.run(plan)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        a, la = c.run(plan)
    b, lb = c.run(plan)                                 # at the same time as the other stream's call
    torch.cuda.synchronize()
    for x, y in ((a, la), (b, lb)):
        assert torch.equal(x, out) and torch.equal(y, lse)
    graphs, outs = [], []
    for _ in range(2):                                  # two graphs of one plan
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(c.run(plan))
        graphs.append(g)
    c.q.copy_(torch.flip(c.q, [0]))
    for _ in range(3):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    want = c.run(plan)
    for o in outs:
        assert torch.equal(o[0], want[0]) and torch.equal(o[1], want[1])
    c.check(*want)


def test_tiles_that_land_out_of_order():
    """Many CTAs that start on new rows, their pages not cached and in no order:
    the copies of a segment's first tiles return late and out of order."""
    c = Case(F16, 128, 4, 2, 128, [1] * 39 + [2], [2048] * 40, [5, 70], seed=19)
    plan = c.plan()
    want = c.run(plan)
    c.check(*want)
    flush = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
    for i in range(100):
        flush.fill_(i)                                  # larger than the L2
        out, lse = c.run(plan)
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    assert plan.status() == 0


def test_offsets_past_32_bits():
    """A pool of over 2^31 elements: pages at its far end."""
    page, d, kv = 128, 128, 8
    n = (1 << 31) // (page * d * kv) + 8
    c = Case(F16, d, kv, 2, page, [3], [256], [10], seed=13)
    used = c.k_pool.shape[0]
    for name in ("k_pool", "v_pool"):
        big = torch.empty(n, kv, page, d, dtype=F16, device="cuda")
        big[n - used:] = getattr(c, name)
        setattr(c, name, big)
    c.table = torch.where(c.table >= 0, c.table + (n - used), c.table)
    c.check(*c.run(c.plan()))
