"""Batched greedy decode of many independent sequences per GPU (B200).

No upstream counterpart: upstream decodes one sequence at a time through
``Decoder`` (``Model/Qwen06B_architecture.py:205-382``).  Each sequence keeps
the upstream per-sequence fp16 KV-cache layout ``[layers, 8, max_seq, 128]``
(``:233-237``); the caches of all sequences are stacked into one K and one V
pool.  A step advances up to ``max_rows`` sequences by one token each through
the C ABI of ``include/qwen_b200_batched.h`` (tcgen05 GEMMs for the
projections and the lm_head, split-KV attention over each sequence's cache).

torch only allocates device memory here; every kernel lives in
``libqwen_b200.so``, and the class refuses to run without it.

Multi-GPU: sequences are independent, so a job shards them across GPUs (one
process per GPU, each with a full weight replica and its own sequences); no
collective is involved.  ``shard_sequences`` gives the split.
"""
from __future__ import annotations

import ctypes
import math
import os

import torch

from paged import PrefixPlan, _host_list, _int, compact_pages, copy_pages, fork_pages, free_pages

_PKG = os.path.dirname(os.path.abspath(__file__))
_lib = None

H, IM, NQ, NKV, HD = 1024, 3072, 16, 8, 128
VOCAB = 151936


class _Layer(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in
                ("input_norm", "w_qkv", "q_norm", "k_norm", "w_o", "post_norm", "w_gu", "w_down")]


def lib() -> ctypes.CDLL:
    global _lib
    if _lib is None:
        path = os.path.join(_PKG, "libqwen_b200.so")
        if not os.path.exists(path):
            raise RuntimeError(f"{path} is missing: build it with qwen0.6b_b200/build.py")
        L = ctypes.CDLL(path)
        vp, i, ll = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong
        L.qwen_b200_batched_workspace.restype = ll
        L.qwen_b200_batched_workspace.argtypes = [i, i]
        L.qwen_b200_batched_create.restype = i
        L.qwen_b200_batched_create.argtypes = [ctypes.POINTER(vp), ctypes.POINTER(_Layer), i, vp, vp,
                                               vp, vp, vp, vp, i, i, i, vp, ll]
        L.qwen_b200_batched_create_paged.restype = i
        L.qwen_b200_batched_create_paged.argtypes = [ctypes.POINTER(vp), ctypes.POINTER(_Layer), i, vp, vp,
                                                     vp, vp, vp, vp, i, vp, i, i, i, i, vp, ll]
        L.qwen_b200_batched_step.restype = i
        L.qwen_b200_batched_step.argtypes = [vp, i, vp, vp, vp, vp, vp, i, ctypes.c_float, vp]
        L.qwen_b200_batched_step_logits.restype = i
        L.qwen_b200_batched_step_logits.argtypes = [vp, i, vp, vp, vp, vp, ll, vp, i, ctypes.c_float, vp]
        L.qwen_b200_batched_step_prefix.restype = i
        L.qwen_b200_batched_step_prefix.argtypes = [vp, i, vp, vp, vp, vp, vp, ll, vp, vp, vp, vp, ll, i,
                                                    ctypes.c_float, vp]
        L.qwen_b200_batched_status.restype = i
        L.qwen_b200_batched_status.argtypes = [vp, ctypes.POINTER(ctypes.c_uint64)]
        L.qwen_b200_batched_destroy.restype = None
        L.qwen_b200_batched_destroy.argtypes = [vp]
        L.qwen_b200_last_error.restype = i
        L.qwen_b200_last_error.argtypes = [ctypes.c_char_p, i]
        _lib = L
    return _lib


def _check(rc: int, what: str) -> None:
    if rc:
        buf = ctypes.create_string_buffer(512)
        lib().qwen_b200_last_error(buf, 512)
        raise RuntimeError(f"{what} failed (code {rc}): {buf.value.decode()}")


def shard_sequences(num_seqs: int, world: int, rank: int) -> range:
    """Contiguous block of sequence indices owned by `rank` of `world`."""
    per = (num_seqs + world - 1) // world
    lo = min(num_seqs, rank * per)
    return range(lo, min(num_seqs, lo + per))


def pack_layer(lw: list) -> dict:
    """Batched-path weights of one layer from its 11 upstream tensors
    (LDGLayerWeight order): q|k|v rows stacked, gate/up rows interleaved."""
    in_norm, q, k, v, q_norm, k_norm, o, post_norm, gate, up, down = lw
    w_qkv = torch.cat([q, k, v], 0).contiguous()
    w_gu = torch.stack([gate, up], 1).reshape(2 * gate.shape[0], gate.shape[1]).contiguous()
    return dict(input_norm=in_norm.contiguous(), w_qkv=w_qkv, q_norm=q_norm.contiguous(),
                k_norm=k_norm.contiguous(), w_o=o.contiguous(), post_norm=post_norm.contiguous(),
                w_gu=w_gu, w_down=down.contiguous())


PAGE = 128  # tokens per KV page


class PagePool:
    """Host bookkeeping of paged KV pools: which page holds positions
    [128 i, 128 i + 128) of each sequence (-1: none), how many sequences hold
    each page, and the free pages.  The methods that change shared pages return
    what has to happen on the device."""

    def __init__(self, num_pages: int, num_seqs: int, max_pages: int):
        self.num_pages, self.num_seqs, self.max_pages = num_pages, num_seqs, max_pages
        self.table = [[-1] * max_pages for _ in range(num_seqs)]
        self.refs = [0] * num_pages
        self.free = list(range(num_pages - 1, -1, -1))  # pop() hands out the lowest page first

    def _take(self) -> int:
        page = self.free.pop()
        self.refs[page] = 1
        return page

    def _drop(self, page: int) -> None:
        self.refs[page] -= 1
        if self.refs[page] == 0:
            self.free.append(page)

    def _enough(self, pages: int) -> None:
        if pages > len(self.free):
            raise RuntimeError(f"KV page pool exhausted ({self.num_pages} pages of {PAGE} tokens)")

    def reserve(self, seq: int, upto_position: int) -> bool:
        """Maps pages for positions 0..upto_position; True if the row changed."""
        missing = self._missing(seq, upto_position)
        self._enough(len(missing))
        self._map(seq, missing)
        return bool(missing)

    def _map(self, seq: int, missing: list[int]) -> None:
        row = self.table[seq]
        for i in missing:
            row[i] = self._take()

    def _missing(self, seq: int, upto_position: int) -> list[int]:
        need = upto_position // PAGE + 1
        if not 0 <= seq < self.num_seqs or not 0 <= upto_position or need > self.max_pages:
            raise ValueError(f"sequence {seq} / position {upto_position} outside the page table")
        row = self.table[seq][:need]
        return [i for i, page in enumerate(row) if page < 0] if -1 in row else []

    def _shared(self, seq: int, write_from: int, upto_position: int) -> list[int]:
        first = write_from // PAGE
        row = self.table[seq][first:upto_position // PAGE + 1]
        return [first + i for i, page in enumerate(row) if page >= 0 and self.refs[page] > 1]

    def claim(self, seq: int, write_from: int, upto_position: int) -> tuple[bool, list[tuple[int, int, int]]]:
        """reserve and unshare, both or (when the pool is exhausted) neither."""
        missing, shared = self._missing(seq, upto_position), self._shared(seq, write_from, upto_position)
        if not missing and not shared:  # the usual call of a step loop
            return False, []
        self._enough(len(missing) + len(shared))
        self._map(seq, missing)
        return bool(missing), self._split(seq, shared, write_from)

    def unshare(self, seq: int, write_from: int, upto_position: int) -> list[tuple[int, int, int]]:
        """Gives sequence `seq` pages of its own for the positions
        write_from..upto_position, which are about to be written, where it
        shares them with another one: (source, destination, tokens to copy) of
        each; the tokens before write_from stay, those behind it are dropped."""
        shared = self._shared(seq, write_from, upto_position)
        self._enough(len(shared))
        return self._split(seq, shared, write_from)

    def _split(self, seq: int, shared: list[int], write_from: int) -> list[tuple[int, int, int]]:
        row, moves = self.table[seq], []
        for i in shared:
            src, row[i] = row[i], self._take()
            self._drop(src)
            moves.append((src, row[i], max(0, write_from - i * PAGE)))
        return moves

    def fork(self, parent: int, children: list[int], length: int) -> list[int]:
        """Makes the children (sequences without pages) copies of the parent's
        first `length` positions: its full pages are shared, the last, partly
        filled one is a new page of each child.  Returns those pages (-1:
        none)."""
        parent, length = _int(parent, "parent"), _int(length, "length")
        children = _host_list(children, "children").tolist()
        full, tail = divmod(length, PAGE)
        if not 0 <= parent < self.num_seqs or not 0 <= length <= self.max_pages * PAGE:
            raise ValueError(f"sequence {parent} / length {length} outside the page table")
        pages = self.table[parent][:full + (tail > 0)]
        if any(p < 0 for p in pages):
            raise ValueError(f"sequence {parent} has no page for some of its first {length} positions")
        if len(set(children)) != len(children) or parent in children:
            raise ValueError("children must be distinct and differ from the parent")
        for c in children:
            if not 0 <= c < self.num_seqs or any(p >= 0 for p in self.table[c]):
                raise ValueError(f"sequence {c} is outside the page table or still holds pages (release it first)")
        if tail:
            self._enough(len(children))
        new = []
        for c in children:
            for i in range(full):
                self.table[c][i] = pages[i]
                self.refs[pages[i]] += 1
            if tail:
                self.table[c][full] = self._take()
            new.append(self.table[c][full] if tail else -1)
        return new

    def release(self, seq: int) -> None:
        row = self.table[seq]
        for i, pg in enumerate(row):
            if pg >= 0:
                self._drop(pg)
                row[i] = -1

    def compact(self) -> tuple[list[int], list[int]]:
        """Renames the pages in use so that they are 0..in_use - 1: the moves
        (sources, destinations)."""
        used = self.in_use
        src = [p for p in range(used, self.num_pages) if self.refs[p]]
        dst = [p for p in range(used) if not self.refs[p]]
        name = dict(zip(src, dst))
        for row in self.table:
            for i, p in enumerate(row):
                if p in name:
                    row[i] = name[p]
        for a, b in name.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.free = list(range(self.num_pages - 1, used - 1, -1))
        return src, dst

    @property
    def in_use(self) -> int:
        return self.num_pages - len(self.free)


class BatchedDecoder:
    """Greedy (or sampled) decode of `num_seqs` independent sequences on one GPU.

    weights: the ``load_weights`` dict (``embed_weight``, ``layer_weights``,
    ``final_norm_weight``, ``cos_table``, ``sin_table``), any device.
    Contiguous pools (default): sequence s owns ``k_pool[s]`` / ``v_pool[s]``
    (fp16 [layers, 8, max_seq, 128], the upstream per-sequence layout).
    Paged pools (``paged=True``, no upstream counterpart): ``num_pages`` pages
    of 128 tokens (fp16 [num_pages, layers, 8, 128, 128] for K and for V)
    shared by all sequences through ``page_table`` (int32 [num_seqs,
    max_seq / 128], -1 = unmapped); ``reserve`` maps pages before positions
    are used (``prefill``, ``prefill_parallel`` and ``generate`` do it), and
    ``release`` returns a finished sequence's pages.  max_seq may then exceed
    2048 (RoPE tables are rebuilt to max_seq rows when the weights' are shorter).
    Sequences can share pages: ``fork`` makes copies of a sequence that share
    its full pages, ``generate_shared`` continues many prompts that begin alike
    (their common part is computed, kept and attended to once), ``compact``
    moves the pages in use to the front of the pools.
    """

    def __init__(self, weights: dict, num_seqs: int, max_rows: int | None = None,
                 max_seq: int = 2048, num_layers: int | None = None, device=None,
                 k_pool: torch.Tensor | None = None, v_pool: torch.Tensor | None = None,
                 paged: bool = False, num_pages: int | None = None):
        self.dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        lw = weights["layer_weights"]
        self.L = num_layers or len(lw) // 11
        self.num_seqs = num_seqs
        self.max_rows = max_rows or num_seqs
        self.max_seq = max_seq
        to = dict(device=self.dev)
        self.embed = weights["embed_weight"].to(**to).contiguous()
        self.final_norm = weights["final_norm_weight"].to(**to).contiguous()
        self.cos = weights["cos_table"].to(**to).contiguous()
        self.sin = weights["sin_table"].to(**to).contiguous()
        if self.cos.shape[0] < max_seq:
            from qwen_weights import rope_tables
            cos, sin = rope_tables(max_seq)
            self.cos, self.sin = cos.to(**to), sin.to(**to)
        self.layers = [pack_layer([t.to(**to) for t in lw[11 * l: 11 * l + 11]]) for l in range(self.L)]
        # Positions a sequence has not reached are never read, so the pools need no clearing.
        # Caller-owned pools (e.g. a Decoder's own cache) must have this exact layout.
        shape = (num_seqs, self.L, NKV, max_seq, HD)
        self.paged = bool(paged)
        if self.paged:
            if k_pool is not None or v_pool is not None:
                raise ValueError("caller-owned pools are contiguous only")
            self.max_pages = (max_seq + PAGE - 1) // PAGE
            self.num_pages = int(num_pages) if num_pages else num_seqs * self.max_pages
            shape = (self.num_pages, self.L, NKV, PAGE, HD)
            self.page_table = torch.full((num_seqs, self.max_pages), -1, dtype=torch.int32, **to)
            self.pages = PagePool(self.num_pages, num_seqs, self.max_pages)
        if k_pool is not None or v_pool is not None:
            for t in (k_pool, v_pool):
                if (t is None or tuple(t.shape) != shape or t.dtype != torch.float16
                        or not t.is_contiguous() or t.device != self.dev):
                    raise ValueError(f"k_pool / v_pool must be contiguous fp16 {shape} on {self.dev}")
            self.k_pool, self.v_pool = k_pool, v_pool
        else:
            self.k_pool = torch.empty(shape, dtype=torch.float16, **to)
            self.v_pool = torch.empty_like(self.k_pool)
        ws = lib().qwen_b200_batched_workspace(self.max_rows, max_seq)
        self.workspace = torch.empty(ws, dtype=torch.uint8, **to)
        self.tokens_out = torch.empty(self.max_rows, dtype=torch.int32, **to)
        self.attn_scale = 1.0 / math.sqrt(HD)
        arr = (_Layer * self.L)()
        for l, d in enumerate(self.layers):
            for name in _Layer._fields_:
                setattr(arr[l], name[0], d[name[0]].data_ptr())
        h = ctypes.c_void_p()
        with torch.cuda.device(self.dev):
            if self.paged:
                _check(lib().qwen_b200_batched_create_paged(
                    ctypes.byref(h), arr, self.L, self.embed.data_ptr(), self.final_norm.data_ptr(),
                    self.cos.data_ptr(), self.sin.data_ptr(), self.k_pool.data_ptr(), self.v_pool.data_ptr(),
                    self.num_pages, self.page_table.data_ptr(), self.max_pages, num_seqs, max_seq,
                    self.max_rows, self.workspace.data_ptr(), ws), "batched_create_paged")
            else:
                _check(lib().qwen_b200_batched_create(
                    ctypes.byref(h), arr, self.L, self.embed.data_ptr(), self.final_norm.data_ptr(),
                    self.cos.data_ptr(), self.sin.data_ptr(), self.k_pool.data_ptr(), self.v_pool.data_ptr(),
                    num_seqs, max_seq, self.max_rows, self.workspace.data_ptr(), ws), "batched_create")
        self._h = h

    # ----------------------------------------------------------- paged pools
    def reserve(self, seq: int, upto_position: int, write_from: int | None = None) -> None:
        """Maps pages for positions 0..upto_position of sequence `seq` (paged
        pools; a no-op otherwise).  Raises when the pool is exhausted.
        Positions write_from (default: upto_position) .. upto_position are about
        to be written: pages of them that the sequence shares with others
        become its own, with the tokens before write_from copied."""
        if not self.paged:
            return
        if not 0 <= upto_position < self.max_seq:
            raise ValueError(f"position {upto_position} outside [0, {self.max_seq})")
        write_from = upto_position if write_from is None else write_from
        if not 0 <= write_from <= upto_position:
            raise ValueError(f"write_from {write_from} outside [0, {upto_position}]")
        changed, moves = self.pages.claim(seq, write_from, upto_position)
        if not changed and not moves:
            return
        if any(t for _, _, t in moves):
            copy_pages(self.k_pool, self.v_pool, *zip(*moves))
        self.page_table[seq].copy_(torch.tensor(self.pages.table[seq], dtype=torch.int32))

    def release(self, seq: int | list[int]) -> None:
        """Returns every page of sequence `seq` (or of each in a list) to the
        pool, once no other sequence holds it (paged pools)."""
        if not self.paged:
            return
        seqs = [seq] if hasattr(seq, "__index__") and not getattr(seq, "ndim", 0) else list(seq)
        seqs = [range(self.num_seqs)[s] for s in seqs]  # what lies outside is refused before anything changes
        for s in seqs:
            self.pages.release(s)
        free_pages(self.page_table, seqs)

    def fork(self, parent: int, children: list[int], length: int) -> None:
        """Makes the sequences `children` (without pages: new or released)
        copies of the first `length` positions of `parent` (paged pools).  The
        parent's full pages are shared, the tokens of the last, partly filled
        one are copied; reserve() before a raw step writes into shared pages
        (``prefill*`` and ``generate*`` do)."""
        if not self.paged:
            raise ValueError("fork needs paged pools")
        children = list(children)
        new = self.pages.fork(parent, children, length)
        n = len(children)
        fork_pages(self.page_table, self.k_pool, self.v_pool, [parent] * n, children, [length] * n, new)

    def compact(self) -> int:
        """Moves the pages in use to the front of the pools (paged pools);
        returns how many moved."""
        if not self.paged:
            raise ValueError("compact needs paged pools")
        src, dst = self.pages.compact()
        compact_pages(self.page_table, self.k_pool, self.v_pool, src, dst)
        return len(src)

    @property
    def pages_in_use(self) -> int:
        return self.pages.in_use if self.paged else 0

    def close(self) -> None:
        if getattr(self, "_h", None):
            lib().qwen_b200_batched_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def step(self, seq_ids: torch.Tensor, positions: torch.Tensor, tokens: torch.Tensor,
             max_position: int, norm_out: torch.Tensor | None = None,
             out: torch.Tensor | None = None, sampling=None,
             prefix: PrefixPlan | None = None) -> torch.Tensor:
        """One step of rows = len(seq_ids) sequences (device int32 tensors):
        greedy, or drawn with ``sampling`` (a ``sampling.SamplingParams``; each
        row's random stream is keyed by its sequence id and position, so a
        draw does not depend on the batch composition).  Returns the device
        int32 tensor of produced tokens.  No host synchronisation.
        prefix (paged pools): the rows' groups that share a prefix, a
        ``paged.PrefixPlan`` for these rows (16 / 8 heads of 128); the shared
        part of each group is then attended to once for all its rows."""
        rows = int(seq_ids.numel())
        for t in (seq_ids, positions, tokens):
            if t.dtype != torch.int32 or t.device != self.dev or not t.is_contiguous():
                raise ValueError("seq_ids, positions and tokens must be contiguous int32 tensors on "
                                 f"{self.dev}")
        out = self.tokens_out[:rows] if out is None else out
        stream = torch.cuda.current_stream(self.dev).cuda_stream
        if sampling is not None:
            from sampling import sample
            if getattr(self, "_logits", None) is None:
                self._logits = torch.empty(self.max_rows, VOCAB, dtype=torch.float32, device=self.dev)
        if prefix is not None:
            if not self.paged:
                raise ValueError("a shared prefix needs paged pools")
            if (prefix.rows, prefix.num_q_heads, prefix.num_kv_heads, prefix.head_dim) != (rows, NQ, NKV, HD):
                raise ValueError(f"the plan is for {prefix.rows} rows of {prefix.num_q_heads} / "
                                 f"{prefix.num_kv_heads} heads of {prefix.head_dim}, the step has {rows} rows")
            if prefix.device != self.dev:
                raise ValueError(f"the plan is on {prefix.device}, the decoder on {self.dev}")
            if not 0 <= max_position < self.max_seq:  # refused as by the steps without a plan
                raise RuntimeError(f"batched_step_prefix failed (code 11): max_position={max_position} outside the KV "
                                   f"cache (max_seq={self.max_seq})")
            if stream != prefix.stream:  # the plan may be dropped while this step still reads it
                prefix.words.record_stream(torch.cuda.current_stream(self.dev))
            # From the caching allocator with every step, so that captured steps have one each.
            ws = torch.empty(prefix.workspace_bytes, dtype=torch.uint8, device=self.dev)
            with torch.cuda.device(self.dev):
                _check(lib().qwen_b200_batched_step_prefix(
                    self._h, rows, seq_ids.data_ptr(), positions.data_ptr(), tokens.data_ptr(),
                    None if sampling is not None else out.data_ptr(),
                    self._logits.data_ptr() if sampling is not None else None, VOCAB,
                    norm_out.data_ptr() if norm_out is not None else None, prefix.header.data_ptr(),
                    prefix.words.data_ptr(), ws.data_ptr(), prefix.workspace_bytes, prefix.max_length, self.attn_scale,
                    ctypes.c_void_p(stream)), "batched_step_prefix")
            if sampling is None:
                return out
            return sample(self._logits[:rows], sampling, out=out, row_seq=seq_ids, row_pos=positions)
        if sampling is not None:
            _check(lib().qwen_b200_batched_step_logits(
                self._h, rows, seq_ids.data_ptr(), positions.data_ptr(), tokens.data_ptr(),
                self._logits.data_ptr(), VOCAB, norm_out.data_ptr() if norm_out is not None else None,
                int(max_position), self.attn_scale, ctypes.c_void_p(stream)), "batched_step_logits")
            return sample(self._logits[:rows], sampling, out=out, row_seq=seq_ids, row_pos=positions)
        _check(lib().qwen_b200_batched_step(
            self._h, rows, seq_ids.data_ptr(), positions.data_ptr(), tokens.data_ptr(),
            out.data_ptr(), norm_out.data_ptr() if norm_out is not None else None,
            int(max_position), self.attn_scale, ctypes.c_void_p(stream)), "batched_step")
        return out

    def status(self) -> int:
        """Synchronises the device; 0, or the code that a step has recorded
        since the last call (1: a bounded wait gave up, 2: a token outside the
        vocabulary, 3: a sequence, position or page outside the tables)."""
        d = ctypes.c_uint64(0)
        return lib().qwen_b200_batched_status(self._h, ctypes.byref(d))

    def prefill(self, prompts: list[list[int]], seqs: list[int] | None = None) -> None:
        """Teacher-forced steps over every prompt token but the last (as
        upstream's ``Decoder.generate`` prefills, one position per step), rows
        = the sequences whose prompt still has tokens at that position."""
        seqs = list(range(len(prompts))) if seqs is None else seqs
        longest = max(len(p) for p in prompts)
        for t in range(longest - 1):
            live = [i for i, p in enumerate(prompts) if t < len(p) - 1]
            for c0 in range(0, len(live), self.max_rows):
                chunk = live[c0: c0 + self.max_rows]
                for i in chunk:
                    self.reserve(seqs[i], t)
                ids = torch.tensor([seqs[i] for i in chunk], dtype=torch.int32, device=self.dev)
                pos = torch.full((len(chunk),), t, dtype=torch.int32, device=self.dev)
                tok = torch.tensor([prompts[i][t] for i in chunk], dtype=torch.int32, device=self.dev)
                self.step(ids, pos, tok, t)

    def prefill_parallel(self, prompts: list[list[int]], seqs: list[int] | None = None,
                         starts: list[int] | None = None) -> None:
        """Parallel prefill (no upstream counterpart; upstream feeds one prompt
        token per step, ``Model/Qwen06B_architecture.py:346-347``): the K/V of
        every prompt token but the last, for all sequences, in as few steps as
        max_rows allows.  Rows of one step may be several positions of the same
        sequence: every row's K/V is appended before the step's attention runs,
        so the row at position p attends to the positions 0..p written by the
        same step.  starts[i] is the position of prompts[i][0] (default 0)."""
        seqs = list(range(len(prompts))) if seqs is None else seqs
        starts = [0] * len(prompts) if starts is None else starts
        rows = [(seqs[i], starts[i] + t, p[t]) for i, p in enumerate(prompts) for t in range(len(p) - 1)]
        for c0 in range(0, len(rows), self.max_rows):
            chunk = rows[c0: c0 + self.max_rows]
            for r in chunk:
                self.reserve(r[0], r[1])
            ids = torch.tensor([r[0] for r in chunk], dtype=torch.int32, device=self.dev)
            pos = torch.tensor([r[1] for r in chunk], dtype=torch.int32, device=self.dev)
            tok = torch.tensor([r[2] for r in chunk], dtype=torch.int32, device=self.dev)
            self.step(ids, pos, tok, max(r[1] for r in chunk),
                      out=torch.empty(len(chunk), dtype=torch.int32, device=self.dev))

    def generate(self, prompts: list[list[int]], max_tokens: int, sampling=None) -> list[list[int]]:
        """Prefill, then `max_tokens` steps of all sequences (at most max_rows
        of them), greedy or with ``sampling``; returns the generated ids per
        sequence."""
        if len(prompts) > self.max_rows:
            raise ValueError(f"{len(prompts)} sequences > max_rows={self.max_rows}")
        self.prefill(prompts)
        n = len(prompts)
        ids = torch.arange(n, dtype=torch.int32, device=self.dev)
        pos = torch.tensor([len(p) - 1 for p in prompts], dtype=torch.int32, device=self.dev)
        tok = torch.tensor([p[-1] for p in prompts], dtype=torch.int32, device=self.dev)
        start_max = max(len(p) - 1 for p in prompts)
        if start_max + max_tokens > self.max_seq:
            raise ValueError("generation would run past max_seq")
        outs = []
        for i, p in enumerate(prompts):
            self.reserve(i, len(p) - 1 + max_tokens - 1, write_from=len(p) - 1)
        for s in range(max_tokens):
            nxt = self.step(ids, pos, tok, start_max + s,
                            out=torch.empty(n, dtype=torch.int32, device=self.dev), sampling=sampling)
            outs.append(nxt)
            tok = nxt
            pos = pos + 1
        return torch.stack(outs, 1).cpu().tolist()

    def generate_shared(self, prefix: list[int], suffixes: list[list[int]], max_tokens: int,
                        sampling=None) -> list[list[int]]:
        """`max_tokens` tokens after each prompt ``prefix + suffixes[i]``
        (suffixes may be empty: several completions of one prompt), greedy or
        drawn with ``sampling``.  Paged pools.  Sequence i holds prompt i; the
        prefix is prefilled once, its full pages are shared by all sequences
        and every step attends to it once for the whole batch.  The sequences
        must hold no pages; they keep theirs afterwards (``release``); none is
        taken when the pool has too few (RuntimeError).  Raises
        RuntimeError when ``status`` reports an error after the last step."""
        if not self.paged:
            raise ValueError("generate_shared needs paged pools")
        n = len(suffixes)
        prompts = [list(prefix) + list(s) for s in suffixes]
        if not 1 <= n <= min(self.max_rows, self.num_seqs) or any(len(p) < 1 for p in prompts):
            raise ValueError(f"{n} prompts: 1 to {min(self.max_rows, self.num_seqs)}, none of them empty")
        if any(p >= 0 for row in self.pages.table[:n] for p in row):
            raise ValueError(f"sequences 0..{n - 1} must hold no pages (release them first)")
        longest = max(len(p) for p in prompts) - 1 + max_tokens
        if max_tokens < 1 or longest > self.max_seq:
            raise ValueError("generation would run past max_seq")
        # Shared positions: the prefix, but for a last token that some prompt still has to feed.
        shared = min(len(prefix), min(len(p) for p in prompts) - 1)
        # All pages or none: the shared ones once, each sequence's own.
        full = shared // PAGE
        self.pages._enough(full + sum((len(p) + max_tokens - 2) // PAGE + 1 - full for p in prompts))
        self.prefill_parallel([prompts[0][:shared + 1]], seqs=[0])
        self.fork(0, list(range(1, n)), shared)
        dev = dict(dtype=torch.int32, device=self.dev)

        def plan(rows: int) -> PrefixPlan:
            return PrefixPlan([rows], [shared], NQ, NKV, HD, max_length=longest, device=self.dev)

        for i, p in enumerate(prompts):
            self.reserve(i, len(p) - 1 + max_tokens - 1, write_from=shared)
        rows = [(i, t, p[t]) for i, p in enumerate(prompts) for t in range(shared, len(p) - 1)]
        for c0 in range(0, len(rows), self.max_rows):
            ids, pos, tok = (torch.tensor(v, **dev) for v in zip(*rows[c0:c0 + self.max_rows]))
            self.step(ids, pos, tok, int(pos.max()), out=torch.empty(len(ids), **dev), prefix=plan(len(ids)))
        ids = torch.arange(n, **dev)
        pos = torch.tensor([len(p) - 1 for p in prompts], **dev)
        tok = torch.tensor([p[-1] for p in prompts], **dev)
        steps, outs = plan(n), []
        for s in range(max_tokens):
            tok = self.step(ids, pos, tok, longest - 1, out=torch.empty(n, **dev), sampling=sampling, prefix=steps)
            outs.append(tok)
            pos = pos + 1
        if code := self.status() or steps.status():
            raise RuntimeError(f"the decoder has recorded error {code}")
        return torch.stack(outs, 1).cpu().tolist()
