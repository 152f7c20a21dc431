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
import operator
import os
import sys

import torch

_PKG = os.path.dirname(os.path.abspath(__file__))
_lib = None
_ext_module = None
_HEADER = 16


def lib() -> ctypes.CDLL:
    global _lib
    if _lib is None:
        path = os.path.join(_PKG, "libqwen_b200.so")
        if not os.path.exists(path):
            raise RuntimeError(f"{path} is missing: build it with qwen0.6b_b200/build.py")
        L = ctypes.CDLL(path)
        vp, i, ll, u64p = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.POINTER(ctypes.c_uint64)
        for name, res, args in [("paged_status", i, [u64p]), ("prefix_plan", i, [i, vp, vp, i, i, i, i, i, vp, i]),
                                ("prefix_workspace", ll, [vp, i, i]), ("prefix_status", i, [vp, vp, u64p]),
                                ("last_error", i, [ctypes.c_char_p, i])]:
            f = getattr(L, "qwen_b200_" + name)
            f.restype, f.argtypes = res, args
        _lib = L
    return _lib


def _last_error() -> str:
    buf = ctypes.create_string_buffer(512)
    lib().qwen_b200_last_error(buf, 512)
    return buf.value.decode()


def _ext():
    """The extension module that makes the calls (tensor checks and allocation in C++)."""
    global _ext_module
    if _ext_module is None:
        if _PKG not in sys.path:
            sys.path.insert(0, _PKG)
        try:
            import paged_C
        except ImportError as e:
            raise RuntimeError(f"the paged_C extension is missing: build it with qwen0.6b_b200/build.py ({e})") from e
        _ext_module = paged_C
    return _ext_module


# ------------------------------------------------------------------- pages
def copy_pages(k_pool: torch.Tensor, v_pool: torch.Tensor, src, dst, tokens=None) -> None:
    """Copies the first tokens[i] tokens (default: all) of page src[i] into
    page dst[i], K and V, every layer and head.

    Pools: contiguous [num_pages, ..., page_tokens, dim].  src, dst, tokens:
    host lists.  Destinations are distinct and none is a source (ValueError);
    a source may repeat."""
    _ext().copy_pages(k_pool, v_pool, src, dst, tokens)


def fork_pages(page_table: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, parents, children, lengths,
               new_pages) -> None:
    """Makes sequence children[i] a copy of the first lengths[i] positions of
    sequence parents[i]: it shares the parent's full pages, gets the tokens of
    the last, partly filled one in page new_pages[i] (ignored, e.g. -1, when
    lengths[i] is a multiple of the page), and the rest of its row is -1.

    Host lists; children are distinct and none is a parent, the used new pages
    are distinct (ValueError) and free.  A parent's page outside the pool is
    skipped (a full one is -1 in the child, a partly filled one is not copied)
    and recorded (``pages_status``)."""
    _ext().fork_pages(page_table, k_pool, v_pool, parents, children, lengths, new_pages)


def compact_pages(page_table: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, src, dst) -> None:
    """Moves page src[i] to page dst[i] (K and V) and renames it in every table
    row.  Host lists; sources are distinct, destinations are distinct and none
    is a source (ValueError); no table row may hold a destination."""
    _ext().compact_pages(page_table, k_pool, v_pool, src, dst)


def free_pages(page_table: torch.Tensor, seqs) -> None:
    """Unmaps every page of the sequences `seqs` (a host list): their table rows become -1."""
    _ext().free_pages(page_table, seqs)


def pages_status(device=None) -> int:
    """Synchronises the device; 0, or 3 when a page operator has met a table
    entry outside the pool there since the last call (the entry was skipped)."""
    with torch.cuda.device(device):
        return lib().qwen_b200_paged_status(None)


# ------------------------------------------------- shared-prefix attention
def _host_list(values, name: str) -> torch.Tensor:
    """A sequence of integers, or a tensor of them, as an int32 tensor on the host."""
    try:
        values = [operator.index(v) for v in (values.tolist() if isinstance(values, torch.Tensor) else values)]
    except TypeError as e:
        raise ValueError(f"{name} must be a one-dimensional list of integers") from e
    if values and not (min(values) >= -2**31 and max(values) < 2**31):
        raise ValueError(f"{name} holds a value outside 32 bits")
    return torch.tensor(values, dtype=torch.int32)


def _int(value, name: str) -> int:
    """An integer of 32 bits (ctypes would cut a larger one down to them)."""
    try:
        value = operator.index(value)
    except TypeError as e:
        raise ValueError(f"{name} must be an integer, not {value!r}") from e
    if not -2**31 <= value < 2**31:
        raise ValueError(f"{name}={value} is outside 32 bits")
    return value


class PrefixPlan:
    """The groups of a batch of rows and the split of their work over the SMs.

    group_rows[g] consecutive rows hold the same tokens in their sequences'
    first prefix_lens[g] positions (0: nothing shared).  max_length: about the
    longest row in the plan's lifetime (it chooses how far one row's own part
    is split; longer rows are still right).  Made once when sequences are
    forked and kept for their steps; the lengths may change from call to call.
    The device part is read only (but for the status word), so calls on several
    streams may share a plan.  It may be dropped when the last call has been
    made; a captured graph needs it for as long as it is replayed."""

    def __init__(self, group_rows, prefix_lens, num_q_heads: int, num_kv_heads: int, head_dim: int, max_length: int,
                 device=None):
        rows, lens = _host_list(group_rows, "group_rows"), _host_list(prefix_lens, "prefix_lens")
        if lens.numel() != rows.numel():
            raise ValueError(f"prefix_lens has {lens.numel()} entries, group_rows {rows.numel()}")
        num_q_heads, num_kv_heads = _int(num_q_heads, "num_q_heads"), _int(num_kv_heads, "num_kv_heads")
        head_dim, max_length = _int(head_dim, "head_dim"), _int(max_length, "max_length")
        if head_dim not in (64, 128):
            raise ValueError(f"head_dim={head_dim}: 64 or 128")
        if max_length < 0:
            raise ValueError(f"max_length={max_length}")
        self.device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        if self.device.type != "cuda":
            raise ValueError(f"a plan lives on a CUDA device, not {self.device}")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        words = plan_words(rows, lens, num_q_heads, num_kv_heads, head_dim, max_length,
                           torch.cuda.get_device_properties(self.device).multi_processor_count)
        self.rows = int(words[1])
        self.num_q_heads, self.num_kv_heads, self.head_dim = num_q_heads, num_kv_heads, head_dim
        self.max_length = max_length
        self.header = words[:_HEADER].clone()
        self.stream = torch.cuda.current_stream(self.device).cuda_stream
        with torch.cuda.device(self.device):
            self.words = words.to(self.device)
        self.workspace_bytes = lib().qwen_b200_prefix_workspace(self.header.data_ptr(), head_dim, self.max_length)

    def status(self) -> int:
        """Synchronises the device; 0, or what a call with this plan has
        recorded since the last one (1: a bounded wait gave up, 3: a sequence,
        length or page outside the tables, which was skipped).  Until a 1 has
        been read, the rows that share a prefix give NaN."""
        with torch.cuda.device(self.device):
            return lib().qwen_b200_prefix_status(self.header.data_ptr(), self.words.data_ptr(), None)


def plan_words(group_rows: torch.Tensor, prefix_lens: torch.Tensor, num_q_heads: int, num_kv_heads: int,
               head_dim: int, max_length: int, ctas: int) -> torch.Tensor:
    """The int32 words of a plan (host), as ``qwen_b200_prefix_plan`` fills them."""
    args = (group_rows.numel(), group_rows.data_ptr(), prefix_lens.data_ptr(), num_q_heads, num_kv_heads, head_dim,
            max_length, ctas)
    n = lib().qwen_b200_prefix_plan(*args, None, 0)
    if n <= 0:
        raise ValueError(f"PrefixPlan: {_last_error()}")
    words = torch.empty(n, dtype=torch.int32)
    if lib().qwen_b200_prefix_plan(*args, words.data_ptr(), n) != n:
        raise ValueError(f"PrefixPlan: {_last_error()}")
    return words


def shared_prefix_attention(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, page_table: torch.Tensor,
                            seq_ids: torch.Tensor, lengths: torch.Tensor, plan: PrefixPlan, scale: float | None = None,
                            out: torch.Tensor | None = None, return_lse: bool = False):
    """softmax(scale q . K^T) V of every row over its sequence's pages, the
    prefix of each of the plan's groups read and multiplied once for all its
    rows.  Scores, softmax statistics and sums are fp32; the weights are rounded
    to q's type for their product with V (bf16: half a step each; fp16: half a
    step, or 2^-32 of the row's largest weight where that is more), and the
    result once at the end.

    q [rows, q heads, dim] (fp16 or bf16, dim 64 or 128): row r is a token of
    sequence seq_ids[r] that sees its positions 0 .. lengths[r] - 1.  Several
    rows may belong to one sequence (draft tokens, a piece of a prompt).
    k_pool, v_pool [num_pages, kv heads, page_tokens, dim], any strides that are
    multiples of 8 elements (e.g. ``pool[:, layer]``), page_tokens a multiple
    of 16; page_table int32 [num_seqs, max_pages]; seq_ids, lengths int32
    [rows].  The pages of a group's prefix are those of its first row that is
    as long as the prefix; a row shorter than that runs on its own pages.  A
    row of length 0 gives 0 (lse -inf; with seq_id 0 a padding row).  scale defaults to dim ** -0.5.

    Returns out [rows, q heads, dim] (the given one, which may be q itself but
    no other memory of q or the pools), with return_lse also the natural
    logarithm of each softmax sum, fp32 [rows, q heads].  A sequence, length or
    page outside the tables is skipped and recorded (``plan.status()``)."""
    if not isinstance(plan, PrefixPlan):
        raise ValueError("plan must be a PrefixPlan")
    out, lse = _ext().prefix_attention(q, k_pool, v_pool, page_table, seq_ids, lengths, plan.header, plan.words,
                                       plan.max_length, plan.workspace_bytes, scale, out, return_lse)
    return (out, lse) if return_lse else out
