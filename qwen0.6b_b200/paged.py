"""Operators on paged KV pools (C ABI include/qwen_b200_paged.h): attention for
a batch whose sequences share their first pages, and copying, forking,
compacting and freeing pages.

No upstream counterpart: upstream keeps one contiguous cache of one sequence
(``Model/Qwen06B_architecture.py:233-237``).  ``BatchedDecoder`` (batched.py)
uses all of them for sequences that share a prompt; they also work on any
pools of the layouts below.

Every call is enqueued on the current stream of the tensors' device, does not
synchronise, and can be captured into a CUDA graph.  The page lists are host
values (they travel with the launch; a captured graph keeps them).  torch only
allocates; every kernel lives in ``libqwen_b200.so``.
"""
from __future__ import annotations

import ctypes
import math
import os

import torch

_PKG = os.path.dirname(os.path.abspath(__file__))
_lib = None
_HEADER = 16


class _Pools(ctypes.Structure):
    _fields_ = [("k_pool", ctypes.c_void_p), ("v_pool", ctypes.c_void_p), ("num_pages", ctypes.c_int),
                ("inner", ctypes.c_int), ("page_tokens", ctypes.c_int), ("token_bytes", ctypes.c_int)]


class _Table(ctypes.Structure):
    _fields_ = [("entries", ctypes.c_void_p), ("num_seqs", ctypes.c_int), ("max_pages", ctypes.c_int),
                ("pitch", ctypes.c_longlong)]


class _Attention(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in ("q", "out", "lse", "k_pool", "v_pool", "page_table", "seq_ids",
                                                "lengths", "plan_header", "plan", "workspace")]
                + [(n, ctypes.c_longlong) for n in ("workspace_bytes", "q_row_stride", "q_head_stride",
                                                    "out_row_stride", "out_head_stride", "page_stride",
                                                    "head_stride", "token_stride", "table_pitch")]
                + [(n, ctypes.c_int) for n in ("rows", "heads", "kv_heads", "dim", "dtype", "num_pages",
                                               "page_tokens", "num_seqs", "max_pages", "max_length", "length_bias")]
                + [("scale", ctypes.c_float)])


def lib() -> ctypes.CDLL:
    global _lib
    if _lib is None:
        path = os.path.join(_PKG, "libqwen_b200.so")
        if not os.path.exists(path):
            raise RuntimeError(f"{path} is missing: build it with qwen0.6b_b200/build.py")
        L = ctypes.CDLL(path)
        vp, i, ll, u64p = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.POINTER(ctypes.c_uint64)
        pools, table = ctypes.POINTER(_Pools), ctypes.POINTER(_Table)
        for name, res, args in [
                ("pages_copy", i, [pools, vp, vp, vp, i, vp]),
                ("pages_fork", i, [pools, table, vp, vp, vp, vp, i, vp]),
                ("pages_compact", i, [pools, table, vp, vp, i, vp]),
                ("pages_free", i, [table, vp, i, vp]),
                ("paged_status", i, [u64p]),
                ("prefix_plan", i, [i, vp, vp, i, i, i, vp, i]),
                ("prefix_workspace", ll, [vp, i, i]),
                ("prefix_attention", i, [ctypes.POINTER(_Attention), vp]),
                ("prefix_status", i, [vp, vp, u64p]),
                ("last_error", i, [ctypes.c_char_p, i])]:
            f = getattr(L, "qwen_b200_" + name)
            f.restype, f.argtypes = res, args
        _lib = L
    return _lib


def _last_error() -> str:
    buf = ctypes.create_string_buffer(512)
    lib().qwen_b200_last_error(buf, 512)
    return buf.value.decode()


# Codes of the C ABI that name a bad argument; the others are launch failures.
_ARGUMENT_CODES = (10, 11, 13, 14, 15)


def _check(rc: int, what: str) -> None:
    if rc:
        kind = ValueError if rc in _ARGUMENT_CODES else RuntimeError
        raise kind(f"{what} failed (code {rc}): {_last_error()}")


def _stream(device) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


# ------------------------------------------------------------------- pages
def _host_list(values, name: str, n: int | None = None) -> torch.Tensor:
    """`values` (a sequence or a CPU integer tensor) as contiguous int32 on the host."""
    if isinstance(values, torch.Tensor):
        if values.device.type != "cpu" or values.dim() != 1 or values.is_floating_point() or values.dtype == torch.bool:
            raise ValueError(f"{name} must be a one-dimensional list of integers on the host")
        t = values
    else:
        t = torch.as_tensor(list(values), dtype=torch.int64)
    if t.dtype != torch.int32:
        if t.numel() and (int(t.min()) < -2**31 or int(t.max()) >= 2**31):
            raise ValueError(f"{name} holds a value outside 32 bits")
        t = t.to(torch.int32)
    t = t.contiguous()
    if n is not None and t.numel() != n:
        raise ValueError(f"{name} has {t.numel()} entries, the other lists {n}")
    return t


def _pools(k_pool: torch.Tensor, v_pool: torch.Tensor) -> _Pools:
    for name, t in (("k_pool", k_pool), ("v_pool", v_pool)):
        if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dim() < 3 or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous CUDA tensor [num_pages, ..., page_tokens, dim]")
    if k_pool.shape != v_pool.shape or k_pool.dtype != v_pool.dtype or k_pool.device != v_pool.device:
        raise ValueError("k_pool and v_pool must have the same shape, type and device")
    s = k_pool.shape
    if k_pool.numel() == 0:
        raise ValueError("the pools are empty")
    return _Pools(k_pool.data_ptr(), v_pool.data_ptr(), s[0], math.prod(s[1:-2]), s[-2], s[-1] * k_pool.element_size())


def _table(page_table: torch.Tensor, device=None) -> _Table:
    t = page_table
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dim() != 2 or t.dtype != torch.int32 or t.stride(1) != 1:
        raise ValueError("page_table must be a CUDA int32 tensor [num_seqs, max_pages] with contiguous rows")
    if device is not None and t.device != device:
        raise ValueError(f"page_table is on {t.device}, the pools on {device}")
    return _Table(t.data_ptr(), t.shape[0], t.shape[1], t.stride(0) if t.shape[0] > 1 else t.shape[1])


def copy_pages(k_pool: torch.Tensor, v_pool: torch.Tensor, src, dst, tokens=None) -> None:
    """Copies the first tokens[i] tokens (default: all) of page src[i] into
    page dst[i], K and V, every layer and head.

    Pools: contiguous [num_pages, ..., page_tokens, dim].  src, dst, tokens:
    host lists.  Destinations are distinct and none is a source (ValueError);
    a source may repeat."""
    p = _pools(k_pool, v_pool)
    src = _host_list(src, "src")
    dst = _host_list(dst, "dst", src.numel())
    tokens = _host_list(tokens, "tokens", src.numel()) if tokens is not None else None
    with torch.cuda.device(k_pool.device):
        _check(lib().qwen_b200_pages_copy(ctypes.byref(p), src.data_ptr(), dst.data_ptr(),
                                          tokens.data_ptr() if tokens is not None else None, src.numel(),
                                          _stream(k_pool.device)), "copy_pages")


def fork_pages(page_table: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, parents, children, lengths,
               new_pages) -> None:
    """Makes sequence children[i] a copy of the first lengths[i] positions of
    sequence parents[i]: it shares the parent's full pages, gets the tokens of
    the last, partly filled one in page new_pages[i] (ignored, e.g. -1, when
    lengths[i] is a multiple of the page), and the rest of its row is -1.

    Host lists; children are distinct and none is a parent, the used new pages
    are distinct (ValueError) and free.  A parent's page outside the pool is
    skipped and recorded (``pages_status``)."""
    p = _pools(k_pool, v_pool)
    t = _table(page_table, k_pool.device)
    parents = _host_list(parents, "parents")
    n = parents.numel()
    children, lengths, new_pages = (_host_list(v, name, n) for v, name in
                                    ((children, "children"), (lengths, "lengths"), (new_pages, "new_pages")))
    with torch.cuda.device(k_pool.device):
        _check(lib().qwen_b200_pages_fork(ctypes.byref(p), ctypes.byref(t), parents.data_ptr(), children.data_ptr(),
                                          lengths.data_ptr(), new_pages.data_ptr(), n, _stream(k_pool.device)),
               "fork_pages")


def compact_pages(page_table: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, src, dst) -> None:
    """Moves page src[i] to page dst[i] (K and V) and renames it in every table
    row.  Host lists; sources are distinct, destinations are distinct and none
    is a source (ValueError); no table row may hold a destination."""
    p = _pools(k_pool, v_pool)
    t = _table(page_table, k_pool.device)
    src = _host_list(src, "src")
    dst = _host_list(dst, "dst", src.numel())
    with torch.cuda.device(k_pool.device):
        _check(lib().qwen_b200_pages_compact(ctypes.byref(p), ctypes.byref(t), src.data_ptr(), dst.data_ptr(),
                                             src.numel(), _stream(k_pool.device)), "compact_pages")


def free_pages(page_table: torch.Tensor, seqs) -> None:
    """Unmaps every page of the sequences `seqs` (a host list): their table rows become -1."""
    t = _table(page_table)
    seqs = _host_list(seqs, "seqs")
    with torch.cuda.device(page_table.device):
        _check(lib().qwen_b200_pages_free(ctypes.byref(t), seqs.data_ptr(), seqs.numel(), _stream(page_table.device)),
               "free_pages")


def pages_status(device=None) -> int:
    """Synchronises the device; 0, or 3 when a page operator has met a table
    entry outside the pool there since the last call (the entry was skipped)."""
    with torch.cuda.device(device):
        return lib().qwen_b200_paged_status(None)


# ------------------------------------------------- shared-prefix attention
class PrefixPlan:
    """The groups of a batch of rows and the split of their work over the SMs.

    group_rows[g] consecutive rows hold the same tokens in their sequences'
    first prefix_lens[g] positions (0: nothing shared).  max_length: about the
    longest row in the plan's lifetime (it chooses how far one row's own part
    is split; longer rows are still right).  Made once when sequences are
    forked and kept for their steps; the lengths may change from call to call.
    The device part is read only (but for the status word), so calls on several
    streams may share a plan."""

    def __init__(self, group_rows, prefix_lens, num_q_heads: int, num_kv_heads: int, head_dim: int, max_length: int,
                 device=None):
        rows = _host_list(group_rows, "group_rows")
        lens = _host_list(prefix_lens, "prefix_lens", rows.numel())
        if head_dim not in (64, 128):
            raise ValueError(f"head_dim={head_dim}: 64 or 128")
        if max_length < 0:
            raise ValueError(f"max_length={max_length}")
        self.device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        if self.device.type != "cuda":
            raise ValueError(f"a plan lives on a CUDA device, not {self.device}")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        words = plan_words(rows, lens, num_q_heads, num_kv_heads,
                           torch.cuda.get_device_properties(self.device).multi_processor_count)
        self.rows = int(words[1])
        self.num_q_heads, self.num_kv_heads, self.head_dim = num_q_heads, num_kv_heads, head_dim
        self.max_length = int(max_length)
        self.header = words[:_HEADER].clone()
        self.words = words.to(self.device)
        self.workspace_bytes = lib().qwen_b200_prefix_workspace(self.header.data_ptr(), head_dim, self.max_length)

    def status(self) -> int:
        """Synchronises the device; 0, or what a call with this plan has
        recorded since the last one (1: a bounded wait gave up, 3: a sequence,
        length or page outside the tables, which was skipped)."""
        with torch.cuda.device(self.device):
            return lib().qwen_b200_prefix_status(self.header.data_ptr(), self.words.data_ptr(), None)


def plan_words(group_rows: torch.Tensor, prefix_lens: torch.Tensor, num_q_heads: int, num_kv_heads: int,
               ctas: int) -> torch.Tensor:
    """The int32 words of a plan (host), as ``qwen_b200_prefix_plan`` fills them."""
    args = (group_rows.numel(), group_rows.data_ptr(), prefix_lens.data_ptr(), num_q_heads, num_kv_heads, ctas)
    n = lib().qwen_b200_prefix_plan(*args, None, 0)
    if n <= 0:
        raise ValueError(f"PrefixPlan: {_last_error()}")
    words = torch.empty(n, dtype=torch.int32)
    if lib().qwen_b200_prefix_plan(*args, words.data_ptr(), n) != n:
        raise ValueError(f"PrefixPlan: {_last_error()}")
    return words


_DTYPES = {torch.float16: 0, torch.bfloat16: 1}


def _strides(t: torch.Tensor) -> tuple:
    """Strides with those of one-element dimensions, which torch leaves arbitrary, as in a contiguous tensor."""
    return tuple(s if n > 1 else math.prod(t.shape[i + 1:]) for i, (n, s) in enumerate(zip(t.shape, t.stride())))


def shared_prefix_attention(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, page_table: torch.Tensor,
                            seq_ids: torch.Tensor, lengths: torch.Tensor, plan: PrefixPlan, scale: float | None = None,
                            out: torch.Tensor | None = None, return_lse: bool = False):
    """softmax(scale q . K^T) V of every row over its sequence's pages, the
    prefix of each of the plan's groups read and multiplied once for all its
    rows (fp32 sums, one rounding at the end).

    q [rows, q heads, dim] (fp16 or bf16, dim 64 or 128): row r is a token of
    sequence seq_ids[r] that sees its positions 0 .. lengths[r] - 1.  Several
    rows may belong to one sequence (draft tokens, a piece of a prompt).
    k_pool, v_pool [num_pages, kv heads, page_tokens, dim], any strides that are
    multiples of 8 elements (e.g. ``pool[:, layer]``), page_tokens a multiple
    of 16; page_table int32 [num_seqs, max_pages]; seq_ids, lengths int32
    [rows].  The pages of a group's prefix are those of its first row's
    sequence; a row shorter than its group's prefix runs on its own pages.  A
    row of length 0 gives 0 (lse -inf).  scale defaults to dim ** -0.5.

    Returns out [rows, q heads, dim], with return_lse also the natural
    logarithm of each softmax sum, fp32 [rows, q heads].  A sequence, length or
    page outside the tables is skipped and recorded (``plan.status()``)."""
    for name, t, nd in (("q", q, 3), ("k_pool", k_pool, 4), ("v_pool", v_pool, 4)):
        if not isinstance(t, torch.Tensor) or t.dim() != nd or t.dtype not in _DTYPES:
            raise ValueError(f"{name} must be an fp16 or bf16 tensor of {nd} dimensions")
        if t.dtype != q.dtype or t.device != q.device:
            raise ValueError(f"{name} is {t.dtype} on {t.device}, q {q.dtype} on {q.device}")
    if not isinstance(plan, PrefixPlan):
        raise ValueError("plan must be a PrefixPlan")
    rows, heads, dim = q.shape
    if (rows, heads, dim) != (plan.rows, plan.num_q_heads, plan.head_dim):
        raise ValueError(f"q is {tuple(q.shape)}, the plan for {(plan.rows, plan.num_q_heads, plan.head_dim)}")
    if k_pool.shape != v_pool.shape or _strides(k_pool) != _strides(v_pool):
        raise ValueError("k_pool and v_pool must have the same shape and strides")
    if k_pool.shape[1] != plan.num_kv_heads or k_pool.shape[3] != dim:
        raise ValueError(f"pools {tuple(k_pool.shape)}: expected {plan.num_kv_heads} kv heads of {dim}")
    if not q.is_cuda or q.device != plan.device:
        raise ValueError(f"q is on {q.device}, the plan on {plan.device}")
    t = _table(page_table, q.device)
    for name, v in (("seq_ids", seq_ids), ("lengths", lengths)):
        if (not isinstance(v, torch.Tensor) or v.dtype != torch.int32 or v.shape != (rows,) or not v.is_contiguous()
                or v.device != q.device):
            raise ValueError(f"{name} must be a contiguous int32 tensor [{rows}] on {q.device}")
    if out is None:
        out = torch.empty(rows, heads, dim, dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != q.device:
        raise ValueError("out must have q's shape, type and device")
    for name, v in (("q", q), ("k_pool", k_pool), ("v_pool", v_pool), ("out", out)):
        if _strides(v)[-1] != 1:
            raise ValueError(f"{name}: the last dimension must be contiguous")
    lse = torch.empty(rows, heads, dtype=torch.float32, device=q.device) if return_lse else None
    # The workspace comes from the caching allocator with each call: calls on
    # several streams, or captured into several graphs, have one each.
    workspace = torch.empty(plan.workspace_bytes, dtype=torch.uint8, device=q.device)
    a = _Attention(
        q.data_ptr(), out.data_ptr(), lse.data_ptr() if return_lse else None, k_pool.data_ptr(), v_pool.data_ptr(),
        t.entries, seq_ids.data_ptr(), lengths.data_ptr(), plan.header.data_ptr(), plan.words.data_ptr(),
        workspace.data_ptr(), plan.workspace_bytes, *_strides(q)[:2], *_strides(out)[:2],
        *_strides(k_pool)[:3], t.pitch, rows, heads, plan.num_kv_heads, dim,
        _DTYPES[q.dtype], k_pool.shape[0], k_pool.shape[2], t.num_seqs, t.max_pages, plan.max_length, 0,
        dim ** -0.5 if scale is None else float(scale))
    with torch.cuda.device(q.device):
        _check(lib().qwen_b200_prefix_attention(ctypes.byref(a), _stream(q.device)), "shared_prefix_attention")
    return (out, lse) if return_lse else out
