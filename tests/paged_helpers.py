"""Plain 64-bit forms of the paged operators, for their tests."""
import math

import torch


def tokens_of(pool, table_row, n):
    """[kv heads, n, dim] in 64 bits: positions 0 .. n - 1 of a sequence."""
    page = pool.shape[2]
    ids = table_row[: -(-n // page)].long()
    return pool[ids].double().permute(1, 0, 2, 3).reshape(pool.shape[1], -1, pool.shape[3])[:, :n]


def attention_reference(q, k_pool, v_pool, table, seq_ids, lengths, scale):
    """(out, lse, bound, lse_bound) in 64 bits, one softmax per row and head.

    The bounds count the roundings of a computation that keeps scores, sums
    and statistics in fp32 and rounds only the weights (relative u = eps / 2)
    and the result.  A score is a sum of dim products that are exact in fp32,
    each addition off by 2^-23 of what has been added at most (the tensor
    cores truncate), so it is off by e = dim 2^-23 scale sum |q k|; 2^x adds a
    few 2^-22.  A weight relative to the sum is then off by w (u + 2 e + 2^-19)
    at most, the result by that times sum w |v|, plus its own rounding u |o|.
    fp16 weights below 2^-14 are off by 2^-25 absolutely instead."""
    rows, heads, d = q.shape
    kv = k_pool.shape[1]
    u = torch.finfo(q.dtype).eps / 2
    out = torch.zeros(rows, heads, d, dtype=torch.float64)
    bound = torch.zeros_like(out)
    lse = torch.full((rows, heads), -math.inf, dtype=torch.float64)
    lse_bound = torch.zeros_like(lse)
    for r in range(rows):
        n = int(lengths[r])
        if n == 0:
            continue
        k = tokens_of(k_pool, table[int(seq_ids[r])], n)
        v = tokens_of(v_pool, table[int(seq_ids[r])], n)
        qr = q[r].double().reshape(kv, -1, d)
        s = scale * (qr @ k.mT)
        e = d * 2.0 ** -23 * scale * (qr.abs() @ k.abs().mT).amax(-1, keepdim=True)
        w = torch.softmax(s, -1)
        o = w @ v
        b = (w @ v.abs()) * (u + 2 * e + 2.0 ** -19) + u * o.abs() + 2.0 ** -24
        if q.dtype == torch.float16:
            b = b + n * 2.0 ** -25 * v.abs().amax()
        out[r], bound[r] = o.reshape(heads, d).cpu(), b.reshape(heads, d).cpu()
        lse[r] = torch.logsumexp(s, -1).reshape(heads).cpu()
        lse_bound[r] = (2 * e.squeeze(-1) + 2.0 ** -19).reshape(heads).cpu() + 2.0 ** -22 * lse[r].abs()
    return out, lse, bound, lse_bound


class Case:
    """A batch over paged pools whose every unused place holds NaN: groups of
    rows (one sequence each unless `tokens` > 1), each group's sequences
    sharing the full pages of their first prefix[g] positions and holding equal
    copies of the tokens of the page behind them."""

    def __init__(self, dtype, dim, kv_heads, ratio, page, group_seqs, prefix, own, tokens=1, layout="hnd", layers=1,
                 seed=0, device="cuda", q_scale=1.5):
        g = torch.Generator().manual_seed(seed)
        self.dim, self.kv_heads, self.heads, self.page = dim, kv_heads, kv_heads * ratio, page
        rows_table, lengths, seq_ids, self.group_rows = [], [], [], []
        fill = []  # (page, tokens filled, copy of (page, tokens) or None)
        total, s = 0, 0
        for n, p in zip(group_seqs, prefix):
            shared = list(range(total, total + p // page))
            total += len(shared)
            fill += [(x, page, None) for x in shared]
            first_tail = None
            self.group_rows.append(n * tokens)
            for _ in range(n):
                o = own[s % len(own)]
                length = p + o
                mine = list(range(total, total + -(-length // page) - len(shared)))
                total += len(mine)
                for i, x in enumerate(mine):
                    t = min(page, length - (len(shared) + i) * page)
                    fill.append((x, t, first_tail if i == 0 else None))
                if first_tail is None and p % page and mine:
                    first_tail = (mine[0], p % page)
                rows_table.append(shared + mine)
                for j in range(tokens):
                    seq_ids.append(s)
                    lengths.append(max(0, length - (tokens - 1 - j)))
                s += 1
        order = torch.randperm(total + 3, generator=g)  # pages in no order, three never used
        shape = (total + 3, layers, kv_heads, page, dim)
        pools = []
        for _ in range(2):
            pool = torch.full(shape, math.nan, dtype=dtype)
            for x, t, copy in fill:
                pool[order[x], :, :, :t] = torch.randn(layers, kv_heads, t, dim, generator=g).to(dtype)
                if copy is not None:
                    y, c = copy
                    c = min(c, t)
                    pool[order[x], :, :, :c] = pool[order[y], :, :, :c]
            if layout == "nhd":  # tokens outermost within a page
                pool = pool.permute(0, 1, 3, 2, 4).contiguous().to(device).permute(0, 1, 3, 2, 4)
            pools.append(pool.to(device)[:, -1])
        self.k_pool, self.v_pool = pools
        widest = max(1, max(len(r) for r in rows_table))
        self.table = torch.full((len(rows_table), widest + 1), -1, dtype=torch.int32)
        for i, r in enumerate(rows_table):
            self.table[i, : len(r)] = order[torch.tensor(r, dtype=torch.long)].int() if r else self.table[i, :0]
        self.table = self.table.to(device)
        self.seq_ids = torch.tensor(seq_ids, dtype=torch.int32, device=device)
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device=device)
        self.q = (q_scale * torch.randn(len(seq_ids), self.heads, dim, generator=g)).to(dtype).to(device)
        self.prefix = list(prefix)
        self.scale = dim ** -0.5

    def plan(self, **kw):
        from paged import PrefixPlan
        kw.setdefault("max_length", int(self.lengths.max()))
        return PrefixPlan(self.group_rows, self.prefix, self.heads, self.kv_heads, self.dim, **kw)

    def run(self, plan, **kw):
        from paged import shared_prefix_attention
        return shared_prefix_attention(self.q, self.k_pool, self.v_pool, self.table, self.seq_ids, self.lengths, plan,
                                       return_lse=True, **kw)

    def reference(self):
        return attention_reference(self.q, self.k_pool, self.v_pool, self.table, self.seq_ids, self.lengths, self.scale)

    def check(self, out, lse):
        ref, ref_lse, bound, lse_bound = self.reference()
        err = (out.cpu().double() - ref).abs()
        assert bool((err <= bound).all()), f"out: {float((err / bound.clamp(min=1e-30)).max())} times the bound"
        lse = lse.cpu().double()
        empty = ref_lse == -math.inf
        assert torch.equal(lse == -math.inf, empty)
        err = (lse - ref_lse)[~empty].abs()
        assert bool((err <= lse_bound[~empty]).all()), f"lse off by {float(err.max())}"
