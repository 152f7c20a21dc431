"""Cases of the shared-prefix attention and of the page operators of a paged KV cache.

Four operators, each in a plain form (elementary torch operations, 32 bits)
and as the calls that a program makes of the package:

``attention``  shared_prefix_attention: rows of a batch whose sequences share
               their first pages (completions of one prompt, requests under
               one system prompt, draft tokens being verified)
``copy``       copy_pages: private copies of pages, whole or their first tokens
``fork``       fork_pages: children that share their parent's full pages and
               get a copy of its last, partly filled one
``compact``    free_pages + compact_pages: the rows of finished sequences
               cleared, the pages in use moved to the front of the pool
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
_DEV = "cuda"


def _package():
    """The package's module of these operators."""
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen0.6b_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import paged
    return paged


# ------------------------------------------------------------------- cases
def listed():
    attention = dict(op="attention", dtype="fp16", layers=1, groups=1, tokens=1, heads=16, kv_heads=8, dim=128,
                     page=128, mix=0)
    pages = dict(layers=28, kv_heads=8, page=128, dim=128, dtype="fp16", mix=0)
    return [
        # Two completions of a short question, first steps: a decode step in which latency is all.
        dict(attention, name="attention: 2 rows, 128 shared", seqs=2, prefix=128, own=8),
        # 32 completions of one prompt of the decode benchmark's length, its 128 new tokens under way.
        dict(attention, name="attention: 32 rows, 1920 shared", layers=2, seqs=32, prefix=1920, own=128, mix=1),
        # The batched benchmark's 256 sequences as samples of one prompt, up to 256 tokens into their answers.
        dict(attention, name="attention: 256 rows, 2048 shared", seqs=256, prefix=2048, own=256, mix=2),
        # Several system prompts of different lengths, small pages, narrow heads, an odd count of sequences.
        dict(attention, name="attention: 7 ragged groups, small pages", dtype="bf16", groups=7, seqs=93, prefix=3000,
             own=500, heads=32, kv_heads=8, dim=64, page=16, mix=3),
        # A few agents over one long document, a thousand own tokens each.
        dict(attention, name="attention: 13 rows over 60000 shared", dtype="bf16", seqs=13, prefix=60000, own=1000,
             heads=32, kv_heads=4, page=64, mix=4),
        # 64 sequences verifying 8 draft tokens each behind a long common context: the products' rate counts.
        dict(attention, name="attention: 64 x 8 rows over 30000 shared", seqs=64, tokens=8, prefix=30000, own=200,
             mix=5),
        # One page of a two-layer model becomes private before a write: a call in the loop of a small program.
        dict(pages, name="copy: one page, 2 layers", op="copy", layers=2, pool=8, pairs=1, tokens=37),
        # Many sequences become private at once (a rollback of a forked batch), each with its own fill.
        dict(pages, name="copy: 90 pages, 28 layers", op="copy", pool=200, pairs=90, tokens=0, mix=6),
        # Beams of a small program: four children of one sequence.
        dict(pages, name="fork: 1 to 4, 2 layers", op="fork", layers=2, parents=1, children=4, length=178),
        # 255 more completions of a prompt of 1997 tokens: every child gets its copy of the 77 tokens behind page 15.
        dict(pages, name="fork: 1 to 255, 28 layers", op="fork", parents=1, children=255, length=1997),
        # A pool of small pages after a third of its sequences finished: many short moves.
        dict(pages, name="compact: small pages", op="compact", dtype="bf16", layers=4, kv_heads=4, page=16, dim=64,
             pool=6000, seqs=160, finished=53, mix=7),
        # The full model's pool after a quarter of its sequences finished.
        dict(pages, name="compact: 28 layers", op="compact", pool=256, seqs=48, finished=12, mix=8),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "copy", "fork", "compact"])
    mix = rng.randrange(1 << 20)
    if op == "attention":
        kv_heads = rng.choice([1, 2, 4, 8, 8])
        c = dict(op=op, dtype=rng.choice(["fp16", "bf16"]), layers=rng.choice([1, 1, 2]), groups=_log(rng, 1, 9),
                 tokens=rng.choice([1, 1, 1, 2, 5, 8]), kv_heads=kv_heads,
                 heads=kv_heads * rng.choice([1, 2, 2, 4, 5, 8]), dim=rng.choice([64, 128, 128]),
                 page=rng.choice([16, 32, 64, 128, 128]), prefix=_log(rng, 16, 60000), own=_log(rng, 8, 1200), mix=mix)
        c["seqs"] = max(c["groups"], _log(rng, 1, 300))
        # No more rows, products or bytes than the largest listed case.
        while (c["seqs"] * c["tokens"] > 512 or c["seqs"] * c["own"] * c["kv_heads"] * c["dim"] > 1 << 27
               or c["seqs"] * c["tokens"] * c["heads"] * c["dim"] * (c["prefix"] + c["own"]) > 30e9):
            k = "seqs" if c["seqs"] > 1 and rng.random() < 0.5 else "prefix" if c["prefix"] > 64 else "own"
            c[k] = max(1 if k == "seqs" else 8, int(c[k] * 0.7))
            c["groups"] = min(c["groups"], c["seqs"])
        while c["groups"] * c["prefix"] * c["kv_heads"] * c["dim"] > 1 << 28:
            c["prefix"] = int(c["prefix"] * 0.7)
        return c
    c = dict(op=op, dtype=rng.choice(["fp16", "bf16"]), layers=_log(rng, 1, 28), kv_heads=rng.choice([2, 4, 8]),
             page=rng.choice([16, 32, 64, 128]), dim=rng.choice([64, 128]), mix=mix)
    page_bytes = 4 * c["layers"] * c["kv_heads"] * c["page"] * c["dim"]  # K and V
    most = max(8, min(6000, int(2.4e9 / page_bytes)))  # pages of a pool
    if op == "copy":
        pairs = _log(rng, 1, max(1, min(1200, most // 3)))
        return dict(c, pool=2 * pairs + rng.randint(2, 20), pairs=pairs, tokens=rng.choice([0, 0, rng.randint(1, c["page"])]))
    if op == "fork":
        parents = _log(rng, 1, 8)
        children = _log(rng, 1, max(1, min(255, most // (2 * parents))))
        return dict(c, parents=parents, children=children, length=_log(rng, 3, 15 * c["page"]))
    seqs = _log(rng, 3, 200)
    return dict(c, pool=max(4 * seqs, _log(rng, 16, most)) if 4 * seqs < most else most, seqs=min(seqs, most // 3),
                finished=max(1, min(seqs, most // 3) // rng.randint(2, 5)))


# ---------------------------------------------- layouts (from the case alone)
def _groups(c):
    """Sequences and shared tokens (whole pages) of each group, and each sequence's own tokens."""
    r = random.Random(c["mix"])
    n, g = c["seqs"], c["groups"]
    if g == 1:
        sizes, shared = [n], [c["prefix"] // c["page"] * c["page"]]
    else:
        cuts = sorted(r.sample(range(1, n), g - 1)) if n > g else list(range(1, g))
        sizes = [b - a for a, b in zip([0] + cuts, cuts + [n])]
        shared = [max(c["page"], int(c["prefix"] * r.uniform(0.1, 1.0)) // c["page"] * c["page"]) for _ in range(g - 1)]
        shared.append(c["prefix"] // c["page"] * c["page"])
    return sizes, shared, [c["tokens"] + r.randrange(c["own"]) for _ in range(n)]


def _rows(c):
    """Per row: its group, its sequence and how many positions it sees."""
    sizes, shared, extra = _groups(c)
    group, seq, length = [], [], []
    s = 0
    for g, n in enumerate(sizes):
        for _ in range(n):
            for j in range(c["tokens"]):
                group.append(g)
                seq.append(s)
                length.append(shared[g] + extra[s] - (c["tokens"] - 1 - j))
            s += 1
    return group, seq, length


def _copy_lists(c):
    r = random.Random(c["mix"])
    order = r.sample(range(c["pool"]), 2 * c["pairs"])
    src, dst = order[:c["pairs"]], order[c["pairs"]:]
    return src, dst, [c["tokens"] or r.randint(1, c["page"]) for _ in src]


def _fork_lists(c):
    """(parents, children, lengths, new pages) and the parents' own tables: parent p is sequence p."""
    r = random.Random(c["mix"])
    n = c["parents"] * c["children"]
    length = [c["length"] if p == 0 else r.randint(1, c["length"]) for p in range(c["parents"])]
    held = [-(-t // c["page"]) for t in length]
    order = list(range(sum(held) + n))
    r.shuffle(order)
    table, at = [], 0
    for h in held:
        table.append(order[at:at + h])
        at += h
    parents = [i // c["children"] for i in range(n)]
    return parents, [c["parents"] + i for i in range(n)], [length[p] for p in parents], order[at:], table


def _compact_lists(c):
    """The table before, the finished sequences, and the moves (source, destination) that follow."""
    r = random.Random(c["mix"])
    order = list(range(c["pool"]))
    r.shuffle(order)
    order = order[:int(c["pool"] * 0.9)]
    cuts = sorted(r.sample(range(1, len(order)), c["seqs"] - 1))
    table = [order[a:b] for a, b in zip([0] + cuts, cuts + [len(order)])]
    finished = sorted(r.sample(range(c["seqs"]), c["finished"]))
    gone = set(finished)
    used = {p for s, row in enumerate(table) if s not in gone for p in row}
    src = sorted(p for p in used if p >= len(used))
    dst = [p for p in range(len(used)) if p not in used]
    return table, finished, src, dst


def _int32(values, device="cpu"):
    return torch.tensor(values, dtype=torch.int32, device=device)


def _table(rows, max_pages):
    return _int32([row + [-1] * (max_pages - len(row)) for row in rows], _DEV)


# ------------------------------------------------------------------ inputs
def _normal(shape, dtype, g):
    return torch.randn(shape, dtype=dtype, device=_DEV, generator=g)


def prepare(case, seed):
    c = case
    g = torch.Generator(device=_DEV).manual_seed(seed)
    dtype = _DTYPES[c["dtype"]]
    s = {"case": c, "op": c["op"]}
    if c["op"] == "attention":
        sizes, shared, extra = _groups(c)
        group, seq, length = _rows(c)
        page = c["page"]
        rows, at = [], 0
        need = [[sh // page] * n for sh, n in zip(shared, sizes)]
        total = sum(sh // page for sh in shared) + sum(-(-e // page) for e in extra)
        # A pool in use for a while: pages in no order.
        order = torch.randperm(total, device=_DEV, generator=g).tolist()
        i = 0
        for sh, n in zip(shared, sizes):
            first = order[at:at + sh // page]
            at += sh // page
            for _ in range(n):
                mine = -(-extra[i] // page)
                rows.append(first + order[at:at + mine])
                at += mine
                i += 1
        widest = max(len(r) for r in rows)
        shape = (total, c["layers"], c["kv_heads"], page, c["dim"])
        k, v = _normal(shape, dtype, g), _normal(shape, dtype, g)
        s.update(q=_normal((len(seq), c["heads"], c["dim"]), dtype, g) * 2, k_pool=k[:, -1], v_pool=v[:, -1],
                 page_table=_table(rows, widest), seq_ids=_int32(seq, _DEV), lengths=_int32(length, _DEV),
                 scale=c["dim"] ** -0.5, group_rows=[n * c["tokens"] for n in sizes], prefix_lens=shared,
                 max_length=max(length))
        # What the plain form indexes with.
        firsts = [sum(s["group_rows"][:j]) for j in range(len(sizes))]
        s.update(group=torch.tensor(group, device=_DEV), first=torch.tensor([seq[f] for f in firsts], device=_DEV),
                 place=torch.tensor([j - firsts[gr] for j, gr in enumerate(group)], device=_DEV),
                 shared=torch.tensor(shared, device=_DEV), widest_own=max(-(-e // page) for e in extra))
        if own:  # the handle that a serving loop makes when it forks and keeps for its steps
            s["plan"] = _package().PrefixPlan(s["group_rows"], s["prefix_lens"], c["heads"], c["kv_heads"], c["dim"],
                                              max_length=s["max_length"], device=_DEV)
        return s
    if c["op"] == "copy":
        src, dst, tokens = _copy_lists(c)
        pool = c["pool"]
        s.update(src=_int32(src), dst=_int32(dst), tokens=_int32(tokens))
    elif c["op"] == "fork":
        parents, children, lengths, new, table = _fork_lists(c)
        pool = sum(map(len, table)) + len(new)
        s.update(parents=_int32(parents), children=_int32(children), lengths=_int32(lengths), new_pages=_int32(new),
                 page_table=_table(table + [[] for _ in children], 1 + max(map(len, table))))
    else:
        table, finished, src, dst = _compact_lists(c)
        pool = c["pool"]
        s.update(finished=_int32(finished), src=_int32(src), dst=_int32(dst),
                 page_table=_table(table, max(map(len, table))))
    shape = (pool, c["layers"], c["kv_heads"], c["page"], c["dim"])
    s.update(k_pool=_normal(shape, dtype, g), v_pool=_normal(shape, dtype, g))
    return s


# ------------------------------------------------------------- plain forms
def _softmax_parts(scores, values):
    """(largest, sum of exponentials, weighted values) over the last axis of `scores`; all masked: (-inf, 0, 0)."""
    m = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(m == -math.inf, torch.zeros_like(m), m))
    return m.squeeze(-1), p.sum(-1), p @ values


def _plain_attention(s):
    c = s["case"]
    rows, ratio, hkv, d, page = s["q"].shape[0], c["heads"] // c["kv_heads"], c["kv_heads"], c["dim"], c["page"]
    q = s["q"].float().view(rows, hkv, ratio, d) * s["scale"]
    # The shared part, once for each group: its queries side by side.
    most = max(s["group_rows"])
    n_pages = max(1, max(s["prefix_lens"]) // page)
    qg = q.new_zeros(len(s["prefix_lens"]), most, hkv, ratio, d)
    qg[s["group"], s["place"]] = q
    qg = qg.transpose(1, 2).reshape(-1, hkv, most * ratio, d)
    ids = s["page_table"][s["first"], :n_pages].long().clamp(min=0)
    k = s["k_pool"][ids].float().transpose(1, 2).reshape(-1, hkv, n_pages * page, d)
    v = s["v_pool"][ids].float().transpose(1, 2).reshape(-1, hkv, n_pages * page, d)
    scores = qg @ k.transpose(2, 3)
    at = torch.arange(n_pages * page, device=q.device)
    scores.masked_fill_((at >= s["shared"][:, None])[:, None, None], -math.inf)
    parts = [t.reshape(-1, hkv, most, ratio, *t.shape[3:])[s["group"], :, s["place"]] for t in _softmax_parts(scores, v)]
    del scores, k, v
    # Each row's own part.
    start = s["shared"][s["group"]]
    ids = (start // page)[:, None] + torch.arange(s["widest_own"], device=q.device)
    ids = s["page_table"].long()[s["seq_ids"].long()[:, None], ids.clamp(max=s["page_table"].shape[1] - 1)].clamp(min=0)
    k = s["k_pool"][ids].float().transpose(1, 2).reshape(rows, hkv, -1, d)
    v = s["v_pool"][ids].float().transpose(1, 2).reshape(rows, hkv, -1, d)
    scores = q @ k.transpose(2, 3)
    at = start[:, None] + torch.arange(s["widest_own"] * page, device=q.device)
    scores.masked_fill_((at >= s["lengths"][:, None])[:, None, None], -math.inf)
    own_parts = _softmax_parts(scores, v)
    # The two joined.
    m = torch.maximum(parts[0], own_parts[0])
    f, h = torch.exp(parts[0] - m), torch.exp(own_parts[0] - m)
    total = parts[1] * f + own_parts[1] * h
    o = (parts[2] * f[..., None] + own_parts[2] * h[..., None]) / total[..., None]
    return {"out": o.reshape(rows, -1, d).to(s["q"].dtype), "lse": (m + torch.log(total)).reshape(rows, -1)}


def _plain_copy(pool, src, dst, tokens):
    """The first tokens[i] tokens of page src[i] into page dst[i]."""
    inside = torch.arange(pool.shape[3], device=pool.device) < tokens[:, None]
    pool[dst] = torch.where(inside[:, None, None, :, None], pool[src], pool[dst])


def _plain(s):
    c = s["case"]
    if s["op"] == "attention":
        return _plain_attention(s)
    on = lambda t: t.to(_DEV).long()  # noqa: E731
    if s["op"] == "copy":
        src, dst, tokens = on(s["src"]), on(s["dst"]), on(s["tokens"])
        _plain_copy(s["k_pool"], src, dst, tokens)
        _plain_copy(s["v_pool"], src, dst, tokens)
        return {"k_pool": s["k_pool"], "v_pool": s["v_pool"]}
    table = s["page_table"]
    if s["op"] == "fork":
        parents, children, lengths, new = on(s["parents"]), on(s["children"]), on(s["lengths"]), on(s["new_pages"])
        full, tail = lengths // c["page"], lengths % c["page"]
        at = torch.arange(table.shape[1], device=_DEV)
        rows = torch.where(at < full[:, None], table[parents], -1)
        rows = torch.where((at == full[:, None]) & (tail > 0)[:, None], new[:, None].int(), rows)
        src = table[parents, full.clamp(max=table.shape[1] - 1)].long().clamp(min=0)
        table[children] = rows.int()
        _plain_copy(s["k_pool"], src, new, tail)
        _plain_copy(s["v_pool"], src, new, tail)
    else:
        src, dst = on(s["src"]), on(s["dst"])
        table[on(s["finished"])] = -1
        names = torch.arange(c["pool"], device=_DEV)
        names[src] = dst
        table.copy_(torch.where(table >= 0, names[table.long().clamp(min=0)].int(), table))
        s["k_pool"][dst] = s["k_pool"][src]
        s["v_pool"][dst] = s["v_pool"][src]
    return {"page_table": table, "k_pool": s["k_pool"], "v_pool": s["v_pool"]}


def run(state):
    s = state
    if not own:
        return _plain(s)
    p = _package()
    if s["op"] == "attention":
        out, lse = p.shared_prefix_attention(s["q"], s["k_pool"], s["v_pool"], s["page_table"], s["seq_ids"],
                                             s["lengths"], s["plan"], scale=s["scale"], return_lse=True)
        return {"out": out, "lse": lse}
    if s["op"] == "copy":
        p.copy_pages(s["k_pool"], s["v_pool"], s["src"], s["dst"], s["tokens"])
        return {"k_pool": s["k_pool"], "v_pool": s["v_pool"]}
    if s["op"] == "fork":
        p.fork_pages(s["page_table"], s["k_pool"], s["v_pool"], s["parents"], s["children"], s["lengths"],
                     s["new_pages"])
    else:
        p.free_pages(s["page_table"], s["finished"])
        p.compact_pages(s["page_table"], s["k_pool"], s["v_pool"], s["src"], s["dst"])
    return {"page_table": s["page_table"], "k_pool": s["k_pool"], "v_pool": s["v_pool"]}


# ------------------------------------------------------------------- work
def work(case):
    c = case
    if c["op"] == "attention":
        sizes, shared, extra = _groups(c)
        _, _, length = _rows(c)
        token = 2 * 2 * c["kv_heads"] * c["dim"]  # K and V of a token
        rows = len(length) * c["heads"]
        return {"bytes": token * (sum(shared) + sum(extra)) + rows * (2 * 2 * c["dim"] + 4) + 8 * len(length),
                "flops": 4 * c["dim"] * c["heads"] * sum(length)}
    token = 2 * 2 * c["layers"] * c["kv_heads"] * c["dim"]
    if c["op"] == "copy":
        src, dst, tokens = _copy_lists(c)
        return {"bytes": token * 2 * sum(tokens), "flops": 0}
    if c["op"] == "fork":
        parents, _, lengths, _, table = _fork_lists(c)
        tail = {p: n % c["page"] for p, n in zip(parents, lengths)}
        return {"bytes": token * (sum(tail.values()) + sum(n % c["page"] for n in lengths))
                + 4 * len(parents) * (1 + max(map(len, table))), "flops": 0}
    table, finished, src, dst = _compact_lists(c)
    return {"bytes": token * 2 * c["page"] * len(src) + 8 * len(table) * max(map(len, table)), "flops": 0}


# ------------------------------------------------------- the definition
def exact(case, seed):
    """Attention in 64 bits, one softmax over all that a row sees; the page operators compute no numbers."""
    if case["op"] != "attention":
        return None
    s = prepare(case, seed)
    c = case
    rows, d, hkv, page = s["q"].shape[0], c["dim"], c["kv_heads"], c["page"]
    out = torch.empty(rows, c["heads"], d, dtype=torch.float64, device=_DEV)
    lse = torch.empty(rows, c["heads"], dtype=torch.float64, device=_DEV)
    ids, lens = s["seq_ids"].tolist(), s["lengths"].tolist()

    def tokens(pool, seq, lo, hi):
        got = pool[s["page_table"][seq, lo // page:-(-hi // page)].long()].double()
        return got.permute(1, 0, 2, 3).reshape(hkv, -1, d)[:, lo % page:lo % page + hi - lo]

    r = 0
    for n, shared in zip(s["group_rows"], s["prefix_lens"]):
        kp, vp = tokens(s["k_pool"], ids[r], 0, shared), tokens(s["v_pool"], ids[r], 0, shared)
        for j in range(r, r + n):
            q = s["q"][j].double().view(hkv, -1, d)
            ko = tokens(s["k_pool"], ids[j], shared, lens[j])
            vo = tokens(s["v_pool"], ids[j], shared, lens[j])
            z = torch.cat([q @ kp.mT, q @ ko.mT], -1) / math.sqrt(d)
            w = torch.softmax(z, -1)
            out[j] = (w[..., :shared] @ vp + w[..., shared:] @ vo).reshape(-1, d)
            lse[j] = torch.logsumexp(z, -1).reshape(-1)
        r += n
    return {"out": out, "lse": lse}
