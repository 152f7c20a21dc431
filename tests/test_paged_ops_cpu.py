"""Arguments that the paged operators refuse, and the plans of the
shared-prefix attention: host code alone, no GPU (the C ABI checks everything
that the host knows before any CUDA call)."""
import ctypes
import random

import pytest
import torch

import paged


class Pools(ctypes.Structure):
    _fields_ = [("k_pool", ctypes.c_void_p), ("v_pool", ctypes.c_void_p), ("num_pages", ctypes.c_int),
                ("inner", ctypes.c_int), ("page_tokens", ctypes.c_int), ("token_bytes", ctypes.c_int)]


class Table(ctypes.Structure):
    _fields_ = [("entries", ctypes.c_void_p), ("num_seqs", ctypes.c_int), ("max_pages", ctypes.c_int),
                ("pitch", ctypes.c_longlong)]


class Attention(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in ("q", "out", "lse", "k_pool", "v_pool", "page_table", "seq_ids",
                                                "lengths", "plan_header", "plan", "workspace")]
                + [(n, ctypes.c_longlong) for n in ("workspace_bytes", "q_row_stride", "q_head_stride",
                                                    "out_row_stride", "out_head_stride", "page_stride",
                                                    "head_stride", "token_stride", "table_pitch")]
                + [(n, ctypes.c_int) for n in ("rows", "heads", "kv_heads", "dim", "dtype", "num_pages",
                                               "page_tokens", "num_seqs", "max_pages", "max_length", "length_bias")]
                + [("scale", ctypes.c_float)])


def _lib():
    L = paged.lib()
    vp, i = ctypes.c_void_p, ctypes.c_int
    pools, table = ctypes.POINTER(Pools), ctypes.POINTER(Table)
    for name, args in [("pages_copy", [pools, vp, vp, vp, i, vp]), ("pages_fork", [pools, table, vp, vp, vp, vp, i, vp]),
                       ("pages_compact", [pools, table, vp, vp, i, vp]), ("pages_free", [table, vp, i, vp]),
                       ("prefix_attention", [ctypes.POINTER(Attention), vp])]:
        f = getattr(L, "qwen_b200_" + name)
        f.restype, f.argtypes = i, args
    return L


def _err():
    return paged._last_error()


POOLS = dict(k_pool=1 << 20, v_pool=1 << 21, num_pages=8, inner=4, page_tokens=16, token_bytes=128)
TABLE = dict(entries=1 << 22, num_seqs=4, max_pages=3, pitch=3)


def _ints(v):
    return (ctypes.c_int * max(1, len(v)))(*v) if v is not None else None


def _call(name, pools=None, table=None, lists=(), n=None):
    p = Pools(**{**POOLS, **(pools or {})})
    t = Table(**{**TABLE, **(table or {})})
    arrays = [_ints(v) for v in lists]
    n = len(lists[0]) if n is None else n
    f = getattr(_lib(), "qwen_b200_pages_" + name)
    head = {"copy": [ctypes.byref(p)], "free": [ctypes.byref(t)]}.get(name, [ctypes.byref(p), ctypes.byref(t)])
    return f(*head, *arrays, n, None)


@pytest.mark.parametrize("name,kw,what", [
    ("copy", dict(lists=([8], [1], None)), "outside the pool"),
    ("copy", dict(lists=([0], [-1], None)), "outside the pool"),
    ("copy", dict(lists=([0, 1], [2, 2], None)), "destination twice"),
    ("copy", dict(lists=([0, 1], [1, 2], None)), "also a source"),
    ("copy", dict(lists=([3], [3], None)), "also a source"),
    ("copy", dict(lists=([0], [1], [17])), "17 tokens of a page of 16"),
    ("copy", dict(lists=([0], [1], [-1])), "tokens of a page"),
    ("copy", dict(lists=([0], [1], None), n=-1), "n=-1"),
    ("copy", dict(lists=([0], None, None)), "null list"),
    ("copy", dict(lists=([0], [1], None), pools=dict(k_pool=None)), "null pool"),
    ("copy", dict(lists=([0], [1], None), pools=dict(k_pool=(1 << 20) + 8)), "16-byte aligned"),
    ("copy", dict(lists=([0], [1], None), pools=dict(v_pool=1 << 20)), "same pool"),
    ("copy", dict(lists=([0], [1], None), pools=dict(token_bytes=24)), "multiple of 16"),
    ("copy", dict(lists=([0], [1], None), pools=dict(num_pages=0)), "must be positive"),
    ("copy", dict(lists=([0], [1], None), pools=dict(inner=1 << 30)), "over 16 GB"),
    ("fork", dict(lists=([4], [1], [5], [0])), "outside the table"),
    ("fork", dict(lists=([0], [-1], [5], [0])), "outside the table"),
    ("fork", dict(lists=([0], [1], [49], [0])), "outside a table row"),
    ("fork", dict(lists=([0], [1], [-1], [0])), "outside a table row"),
    ("fork", dict(lists=([0], [1], [5], [8])), "new page 8"),
    ("fork", dict(lists=([0], [1], [5], [-1])), "new page -1"),
    ("fork", dict(lists=([0, 0], [1, 2], [5, 5], [3, 3])), "two children"),
    ("fork", dict(lists=([0, 0], [1, 1], [5, 5], [3, 4])), "named twice"),
    ("fork", dict(lists=([0, 1], [1, 2], [5, 5], [3, 4])), "also a parent"),
    ("fork", dict(lists=([0], [1], [5], [0]), table=dict(entries=None)), "null page table"),
    ("fork", dict(lists=([0], [1], [5], [0]), table=dict(pitch=2)), "pitch=2"),
    ("compact", dict(lists=([5, 5], [0, 1])), "moves twice"),
    ("compact", dict(lists=([5, 6], [0, 0])), "destination twice"),
    ("compact", dict(lists=([5, 6], [0, 5])), "also a source"),
    ("compact", dict(lists=([9], [0])), "outside the pool"),
    ("free", dict(lists=([4],)), "outside the table"),
    ("free", dict(lists=([-1],)), "outside the table"),
])
def test_page_lists_are_refused(name, kw, what):
    assert _call(name, **kw) != 0
    assert what in _err()


@pytest.mark.parametrize("name,k", [("copy", 3), ("fork", 4), ("compact", 2), ("free", 1)])
def test_empty_lists_are_no_calls(name, k):
    assert _call(name, lists=([],) * k) == 0


def _attention(**kw):
    words = paged.plan_words(torch.tensor([4], dtype=torch.int32), torch.tensor([256], dtype=torch.int32), 4, 2, 128, 512, 148)
    header = words[:16].clone()
    kw = dict(kw)
    if kw.pop("bad_plan", False):
        header[0] = 0
    base = dict(q=1 << 20, out=1 << 21, lse=None, k_pool=1 << 22, v_pool=1 << 23, page_table=1 << 24, seq_ids=1 << 25,
                lengths=1 << 26, plan_header=header.data_ptr(), plan=1 << 27, workspace=1 << 28,
                workspace_bytes=1 << 40, q_row_stride=512, q_head_stride=128, out_row_stride=512, out_head_stride=128,
                page_stride=2 * 64 * 128, head_stride=64 * 128, token_stride=128, table_pitch=8, rows=4, heads=4,
                kv_heads=2, dim=128, dtype=0, num_pages=64, page_tokens=64, num_seqs=4, max_pages=8, max_length=512,
                length_bias=0, scale=0.1)
    a = Attention(**{**base, **kw})
    return _lib().qwen_b200_prefix_attention(ctypes.byref(a), None)


@pytest.mark.parametrize("kw,what", [
    (dict(bad_plan=True), "plan"),
    (dict(rows=5), "plan is for 4 rows"),
    (dict(heads=8), "plan is for"),
    (dict(dim=96), "dim=96"),
    (dict(dtype=2), "dtype=2"),
    (dict(page_tokens=24), "multiple of 16 tokens"),
    (dict(page_tokens=0), "multiple of 16 tokens"),
    (dict(num_pages=0), "num_pages=0"),
    (dict(table_pitch=7), "pitch=7"),
    (dict(max_pages=1 << 28, table_pitch=1 << 28), "2^31 tokens"),
    (dict(scale=0.0), "scale"),
    (dict(scale=-1.0), "scale"),
    (dict(scale=float("nan")), "scale"),
    (dict(q=None), "null"),
    (dict(workspace=None), "null"),
    (dict(q=(1 << 20) + 4), "16-byte aligned"),
    (dict(v_pool=(1 << 23) + 8), "16-byte aligned"),
    (dict(q_head_stride=132), "multiple of 8"),
    (dict(token_stride=64), "overlap"),
    (dict(workspace_bytes=1024), "workspace of 1024"),
    (dict(max_length=-1), "max_length"),
])
def test_attention_arguments_are_refused(kw, what):
    assert _attention(**kw) != 0
    assert what in _err()


@pytest.mark.parametrize("rows,lens,heads,kv,ctas", [
    ([], [], 4, 2, 8), ([0], [16], 4, 2, 8), ([-1, 3], [16, 16], 4, 2, 8), ([3], [-1], 4, 2, 8), ([3], [16], 5, 2, 8),
    ([3], [16], 1, 2, 8), ([3], [16], 4, 0, 8), ([3], [16], 4, 2, 0), ([70000], [16], 4, 2, 8), ([3], [16], 258, 2, 8),
])
def test_plan_arguments_are_refused(rows, lens, heads, kv, ctas):
    with pytest.raises(ValueError, match="plan"):
        paged.plan_words(torch.tensor(rows, dtype=torch.int32), torch.tensor(lens, dtype=torch.int32), heads, kv, 64, 512, ctas)


def test_python_refusals_without_a_gpu():
    z = torch.zeros(4, 2, 16, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        paged.copy_pages(z, z, [0], [1])
    with pytest.raises(ValueError, match="CUDA"):
        paged.free_pages(torch.zeros(2, 2, dtype=torch.int32), [0])
    with pytest.raises(ValueError, match="PrefixPlan"):
        paged.shared_prefix_attention(torch.zeros(2, 4, 64, dtype=torch.float16), z, z, z, z, z, None)
    with pytest.raises(ValueError, match="CUDA device"):
        paged.PrefixPlan([2], [16], 4, 2, 64, max_length=32, device="cpu")
    with pytest.raises(ValueError, match="head_dim"):
        paged.PrefixPlan([2], [16], 4, 2, 96, max_length=32)
    with pytest.raises(ValueError, match="entries"):
        paged.PrefixPlan([2, 1], [16], 4, 2, 64, max_length=32)
    with pytest.raises(ValueError, match="32 bits"):
        paged._host_list([1 << 40], "x")
    for bad in ([1.5], [[1, 2]], [torch.tensor([1, 2])]):
        with pytest.raises(ValueError, match="list of integers"):
            paged._host_list(bad, "x")
    with pytest.raises(ValueError, match="32 bits"):
        paged.PrefixPlan([2], torch.tensor([(1 << 32) + 16]), 4, 2, 64, max_length=32)
    with pytest.raises(ValueError, match="list of integers"):
        paged.PrefixPlan(torch.tensor([2.5]), [16], 4, 2, 64, max_length=32)
    assert paged._host_list((), "x").numel() == 0


def _plan(rows, lens, heads, kv, longest, ctas):
    w = paged.plan_words(torch.tensor(rows, dtype=torch.int32), torch.tensor(lens, dtype=torch.int32), heads, kv,
                         128, longest, ctas).tolist()
    h = w[:16]
    cta = [w[h[8] + 16 * i:h[8] + 16 * i + 16] for i in range(h[3])]  # what each CTA reads first
    return dict(rows=h[1], cta=cta,
                segs=[tuple(w[h[9] + 8 * i:h[9] + 8 * i + 8]) for i in range(h[4])],
                tiles=w[h[10]:h[10] + h[5] + 1], row=[tuple(w[h[11] + 4 * i:h[11] + 4 * i + 4]) for i in range(h[1])])


@pytest.mark.parametrize("seed", range(40))
def test_plans_cover_every_tile_once(seed):
    """Every (query tile, kv head, token tile) of the shared parts belongs to
    one CTA, and each row finds the partial results of all its heads."""
    r = random.Random(seed)
    n, kv = r.randint(1, 8), r.choice([1, 2, 4, 8])
    ratio = r.choice([1, 2, 3, 5, 8, 16])
    rows = [r.choice([0, 1, 2, 3, 17, 64, 100]) for _ in range(n)] + [3]
    lens = [r.choice([0, 1, 15, 16, 127, 128, 129, 1000, 5000]) for _ in rows]
    ctas = r.choice([1, 3, 148])
    longest = r.choice([0, 200, 6000, 60000])
    p = _plan(rows, lens, kv * ratio, kv, longest, ctas)
    assert p["rows"] == sum(rows) and len(p["cta"]) <= ctas
    assert [c[0] for c in p["cta"]] + [len(p["segs"])] == [0] + [c[1] for c in p["cta"]]
    for first, last, *_, in p["cta"]:
        assert first <= last
    for c in p["cta"]:
        assert c[0] == c[1] or tuple(c[8:]) == p["segs"][c[0]]
    assert p["tiles"] == sorted(p["tiles"])
    seen = set()
    for row0, nq, q0, h, t0, t1, prefix, dual in p["segs"]:
        assert t0 < t1 and dual == (nq - q0 > 128)
        for t in range(t0, t1):
            assert (row0, q0, h, t) not in seen
            seen.add((row0, q0, h, t))
    want, row0 = 0, 0
    any_shared = any(m > 1 and q >= 16 for m, q in zip(rows, lens))
    if max([longest] + lens) <= 256 and sum(rows) * kv * -(-ratio // 8) <= 296:
        lens = [0] * len(lens)                           # a small batch of short rows: all their own
    for m, q in zip(rows, lens):
        q = q // 16 * 16 if m > 1 or (m == 1 and q >= 1024 and any_shared) else 0
        want += -(-q // 128) * kv * -(-m * ratio // 256) if q else 0
        for j in range(m):
            prefix, tile0, query, queries = p["row"][row0 + j]
            assert prefix == q and query == j * ratio and queries == m * ratio
            for h in range(kv * ratio if q else 0):
                qi = query + h % ratio
                tile = tile0 + qi // 256 * kv + h // ratio
                mine = p["segs"][p["tiles"][tile]:p["tiles"][tile + 1]]
                assert mine and all(s[0] == row0 and s[3] == h // ratio and s[2] <= qi < s[2] + 256 and s[6] == q
                                    for s in mine)
                assert [s[4] for s in mine[1:]] == [s[5] for s in mine[:-1]]
                assert mine[0][4] == 0 and mine[-1][5] == -(-q // 128)
        row0 += m
    assert len(seen) == want
