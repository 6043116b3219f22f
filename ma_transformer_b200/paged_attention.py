"""Token-by-token attention over a paged key-value cache: ``append`` writes new tokens (rotating keys and queries by
position on the way), ``decode`` attends one new token per sequence, ``select_pages`` picks the pages it reads by a
cheap score.  All three enqueue work on torch's current stream and never synchronise; they may be captured into CUDA
graphs (workspaces come from torch's allocator call by call, so two graphs never share one).

The reference keeps no cache: it recomputes whole sequences (src/model.py:55-87).  Errors follow the rest of the
package: ``RuntimeError`` for tensors and shapes the kernels refuse.

What is on the device is not checked on the host: a page table entry that a call touches and that lies outside the
cache is skipped (its tokens count as absent) and sets bit 1 of ``device_status()``.
"""
from __future__ import annotations

import ctypes as C
from contextlib import nullcontext
from typing import Dict, Optional, Tuple

import torch

from . import _native as nat
from .patterns import PatternSpec, WINDOW

_HERE = nullcontext()
_DTYPES = {torch.float32: nat.MAT_F32, torch.bfloat16: nat.MAT_BF16, torch.float16: nat.MAT_F16}


def rotary_frequencies(dim: int, base: float = 10000.0, device="cuda") -> torch.Tensor:
    """The ``dim / 2`` frequencies base^(-2r/dim) of a rotation over ``dim`` columns, in 64 bits as ``append`` takes
    them.  Scaled or interpolated schemes pass their own."""
    if dim < 2 or dim % 2:
        raise RuntimeError(f"the rotated width must be even and at least 2, got {dim}")
    r = torch.arange(0, dim, 2, dtype=torch.float64)
    return (float(base) ** (-r / dim)).to(device)


class PagedKVCache:
    """Keys and values of many sequences in pages of ``page_size`` tokens: ``k`` and ``v`` are
    [n_pages, page_size, n_kv_heads, head_dim]; ``key_bounds`` (optional, for ``select_pages``) holds each page's
    smallest and largest key column by column, [n_pages, 2, n_kv_heads, head_dim].

    ``page_size``: a power of two from 8 to 1024.  ``head_dim``: a multiple of 8 up to 256.
    """

    def __init__(self, n_pages: int, page_size: int, n_kv_heads: int, head_dim: int, dtype: torch.dtype = torch.bfloat16,
                 device="cuda", key_bounds: bool = False):
        shape = (int(n_pages), int(page_size), int(n_kv_heads), int(head_dim))
        bounds = torch.zeros((shape[0], 2, shape[2], shape[3]), dtype=dtype, device=device) if key_bounds else None
        self._bind(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device), bounds)

    @classmethod
    def from_tensors(cls, k: torch.Tensor, v: torch.Tensor, key_bounds: Optional[torch.Tensor] = None) -> "PagedKVCache":
        """A cache over existing tensors [n_pages, page_size, n_kv_heads, head_dim]; views with other strides (such as
        ``[n_pages, n_kv_heads, page_size, head_dim].transpose(1, 2)``) are used in place, columns must be packed."""
        self = cls.__new__(cls)
        self._bind(k, v, key_bounds)
        return self

    def _bind(self, k, v, key_bounds) -> None:
        if not (k.is_cuda and v.is_cuda):
            raise RuntimeError("the cache's tensors must be CUDA tensors")
        if k.dtype not in _DTYPES or v.dtype != k.dtype:
            raise RuntimeError("Only float32, bfloat16 and float16 are supported (k and v of one dtype)")
        if k.dim() != 4 or v.shape != k.shape:
            raise RuntimeError("k and v must both be [n_pages, page_size, n_kv_heads, head_dim]")
        if v.device != k.device:
            raise RuntimeError("k and v must be on the same device")
        if k.stride(3) != 1 or v.stride(3) != 1:
            raise RuntimeError("the columns of k and v must be packed")
        if key_bounds is not None:
            if (key_bounds.dtype != k.dtype or key_bounds.device != k.device or not key_bounds.is_contiguous()
                    or tuple(key_bounds.shape) != (k.shape[0], 2, k.shape[2], k.shape[3])):
                raise RuntimeError("key_bounds must be a contiguous [n_pages, 2, n_kv_heads, head_dim] tensor of the "
                                   "cache's dtype and device")
        self.k, self.v, self.key_bounds = k, v, key_bounds
        s = nat.MatPagedCache()
        s.k, s.v = k.data_ptr(), v.data_ptr()
        s.key_bounds = key_bounds.data_ptr() if key_bounds is not None else None
        s.n_pages, s.page_size, s.H_kv, s.D = k.shape
        s.k_page_stride, s.k_token_stride, s.k_head_stride = k.stride()[:3]
        s.v_page_stride, s.v_token_stride, s.v_head_stride = v.stride()[:3]
        s.dtype = _DTYPES[k.dtype]
        # sizes, strides and alignment are refused here by the library's own rules: an append of no tokens checks them
        at = k.data_ptr()
        nat.check(nat.lib.mat_paged_append(C.byref(s), None, None, 0, 0, 0, at, at, at, 1, 1, 1, None, None, 0, 0, None, 0, 0, None))
        self._struct, self._ref = s, C.byref(s)
        self.n_pages, self.page_size, self.n_kv_heads, self.head_dim = (int(x) for x in k.shape)
        self.dtype, self.device, self._dev = k.dtype, k.device, k.get_device()
        self._decode_bytes: Dict[tuple, int] = {}     # workspace sizes by the shapes they depend on


# A decoding step is a few microseconds of GPU work, so the checks below go through the cheapest accessors there are:
# get_device() instead of device objects, the raw stream handle instead of a Stream.
_raw_stream = torch._C._cuda_getCurrentRawStream
_lib_append, _lib_decode, _lib_select = nat.lib.mat_paged_append, nat.lib.mat_paged_decode, nat.lib.mat_paged_select


def _table(table: torch.Tensor, cache: PagedKVCache) -> Tuple[int, int, int]:
    """(B, width, elements between rows) of a page table."""
    if table.dtype is not torch.int32 or table.dim() != 2 or table.get_device() != cache._dev:
        raise RuntimeError("page_table must be a 2-d int32 tensor on the cache's device")
    B, width = table.shape
    if table.is_contiguous():
        return B, width, width
    if table.stride(1) != 1:
        raise RuntimeError("the rows of page_table must be packed")
    return B, width, table.stride(0) if B > 1 else width


def _per_sequence(t: torch.Tensor, name: str, cache: PagedKVCache, n: int) -> None:
    if t.dtype is not torch.int32 or t.dim() != 1 or t.get_device() != cache._dev or t.shape[0] != n or not t.is_contiguous():
        raise RuntimeError(f"{name} must be a packed int32 tensor of {n} entries on the cache's device")


def _rows(t: torch.Tensor, name: str, cache: PagedKVCache, n: int, heads: int) -> int:
    """Checks a [n, heads, head_dim] tensor with packed heads; elements between its rows."""
    if t.dtype is not cache.dtype or t.get_device() != cache._dev:
        raise RuntimeError(f"{name} must be of the cache's dtype and on its device")
    if t.shape != (n, heads, cache.head_dim):
        raise RuntimeError(f"{name} must be [{n}, {heads}, {cache.head_dim}], got {list(t.shape)}")
    if t.is_contiguous():
        return heads * cache.head_dim
    if t.stride(2) != 1 or (heads > 1 and t.stride(1) != cache.head_dim):
        raise RuntimeError(f"the heads and columns of {name} must be packed")
    return t.stride(0) if n > 1 else heads * cache.head_dim


def _heads(query: torch.Tensor, cache: PagedKVCache) -> int:
    if query.dim() != 3:
        raise RuntimeError("query must be [rows, heads, head_dim]")
    H = query.shape[1]
    if H < cache.n_kv_heads or H % cache.n_kv_heads:
        raise RuntimeError(f"{H} query heads do not divide over {cache.n_kv_heads} key heads")
    return H


def _on_device(cache: PagedKVCache):
    """A context that makes the cache's device the current one; nothing where it is already."""
    return _HERE if torch.cuda.current_device() == cache._dev else torch.cuda.device(cache._dev)


def _result(out: Optional[torch.Tensor], name: str, like: torch.Tensor) -> torch.Tensor:
    if out is None:
        return torch.empty_like(like) if like.is_contiguous() else torch.empty(like.shape, dtype=like.dtype, device=like.device)
    if out.shape != like.shape or out.dtype is not like.dtype or out.get_device() != like.get_device() or not out.is_contiguous():
        raise RuntimeError(f"{name} must be a contiguous tensor of query's shape, dtype and device")
    return out


def append(cache: PagedKVCache, key: torch.Tensor, value: torch.Tensor, page_table: torch.Tensor, start: torch.Tensor,
           cu_seqlens: Optional[torch.Tensor] = None, query: Optional[torch.Tensor] = None,
           inv_freq: Optional[torch.Tensor] = None, interleaved: bool = False,
           query_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Writes new tokens into the cache.

    key, value: [N, n_kv_heads, head_dim], tokens of all sequences one after another (heads packed; the tokens may lie a
    stride apart, as the slices of a fused projection do).  ``cu_seqlens`` [B + 1] int32 says where each sequence's rows
    begin; without it every sequence gets one token (N == B).  Rows behind ``cu_seqlens[B]`` are padding and left alone.
    start: [B] int32, the position of each sequence's first new token.  page_table: [B, width] int32.
    inv_freq: [rot / 2] float64 turns the first ``rot`` columns of each key (and query) by position * inv_freq; column
    pairs are (2r, 2r + 1) when ``interleaved``, else (r, r + rot / 2).
    query: [N, H, head_dim] gets the same rotation; the result is returned (``query_out`` or a new packed tensor, whose
    padding rows are not written).
    Sequences of one call may not share a page that the call writes to; otherwise pages may be shared.
    """
    N = key.shape[0] if key.dim() == 3 else -1
    k_ts = _rows(key, "key", cache, N, cache.n_kv_heads)
    v_ts = _rows(value, "value", cache, N, cache.n_kv_heads)
    B, width, t_stride = _table(page_table, cache)
    _per_sequence(start, "start", cache, B)
    if cu_seqlens is not None:
        _per_sequence(cu_seqlens, "cu_seqlens", cache, B + 1)
    elif N != B:
        raise RuntimeError(f"without cu_seqlens every sequence gets one token: got {N} for {B}")
    rot = 0
    if inv_freq is not None:
        if inv_freq.dtype is not torch.float64 or inv_freq.dim() != 1 or inv_freq.get_device() != cache._dev or not inv_freq.is_contiguous():
            raise RuntimeError("inv_freq must be a contiguous 1-d float64 tensor on the cache's device")
        rot = 2 * inv_freq.shape[0]
        if rot == 0 or rot > cache.head_dim:
            raise RuntimeError(f"inv_freq must have 1 to {cache.head_dim // 2} entries")
    H = q_ts = 0
    q_ptr = out_ptr = None
    if query is not None:
        H = _heads(query, cache)
        q_ts = _rows(query, "query", cache, N, H)
        query_out = _result(query_out, "query_out", query)
        q_ptr, out_ptr = query.data_ptr(), query_out.data_ptr()
    elif query_out is not None:
        raise RuntimeError("query_out needs a query")
    if N == 0:
        return query_out
    with _on_device(cache):
        rc = _lib_append(
            cache._ref, key.data_ptr(), value.data_ptr(), k_ts, v_ts, N, cu_seqlens.data_ptr() if cu_seqlens is not None else None,
            start.data_ptr(), page_table.data_ptr(), width, t_stride, B, q_ptr, out_ptr, H, q_ts,
            inv_freq.data_ptr() if inv_freq is not None else None, rot, bool(interleaved), _raw_stream(cache._dev))
    if rc:
        nat.check(rc)
    return query_out


def decode(query: torch.Tensor, cache: PagedKVCache, page_table: torch.Tensor, lengths: torch.Tensor,
           spec: Optional[PatternSpec] = None, pages: Optional[torch.Tensor] = None, scale: Optional[float] = None,
           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of one new token per sequence over the cached ones: [B, H, head_dim].

    query: [B, H, head_dim], H a multiple of the cache's heads (query head h reads key head h // (H / n_kv_heads)).
    lengths: [B] int32 cached tokens, the new one included; 0 gives a zero row, as do scores that are all -inf.
    spec: a window ``PatternSpec`` (its ``right`` taps lie in the future and select nothing); pages: the
    [B, n_kv_heads, n] int32 result of ``select_pages``.  With neither, every cached token is read.
    """
    H = _heads(query, cache)
    B, width, t_stride = _table(page_table, cache)
    q_stride = _rows(query, "query", cache, B, H)
    _per_sequence(lengths, "lengths", cache, B)
    left, dilation, n_sel, pages_ptr = -1, 1, 0, None
    if spec is not None:
        if spec.kind != WINDOW or spec.q_offset:
            raise RuntimeError("decode takes window patterns without an offset")
        if pages is not None:
            raise RuntimeError("spec and pages cannot be combined")
        left, dilation = int(spec.left), int(spec.dilation)
    if pages is not None:
        if pages.dtype is not torch.int32 or pages.get_device() != cache._dev or not pages.is_contiguous() or pages.dim() != 3 \
                or pages.shape[:2] != (B, cache.n_kv_heads) or pages.shape[2] < 1:
            raise RuntimeError(f"pages must be a contiguous int32 [{B}, {cache.n_kv_heads}, n] tensor on the cache's device")
        n_sel, pages_ptr = pages.shape[2], pages.data_ptr()
    out = _result(out, "out", query)
    nbytes = cache._decode_bytes.get((B, H, width, left, n_sel))
    if nbytes is None:
        nbytes = cache._decode_bytes[B, H, width, left, n_sel] = \
            nat.lib.mat_paged_decode_workspace_bytes(cache._ref, B, H, width, left, n_sel)
    with _on_device(cache):
        ws = torch.empty(nbytes, dtype=torch.uint8, device=cache.device) if nbytes else None
        rc = _lib_decode(
            cache._ref, query.data_ptr(), q_stride, out.data_ptr(), B, H, page_table.data_ptr(), width, t_stride,
            lengths.data_ptr(), left, dilation, pages_ptr, n_sel, float(scale) if scale else 0.0,
            ws.data_ptr() if ws is not None else None, nbytes, _raw_stream(cache._dev))
    if rc:
        nat.check(rc)
    return out


def select_pages(query: torch.Tensor, cache: PagedKVCache, page_table: torch.Tensor, lengths: torch.Tensor,
                 topk: int) -> torch.Tensor:
    """The ``topk`` logical pages each new token reads, [B, n_kv_heads, topk] int32, ascending, -1 behind the last: the
    page of the token itself and the best others by an upper bound of the group's q . k that the cache's ``key_bounds``
    give (sum over query heads and columns of max(q * lo, q * hi)).  Scores are compared in 64 bits, equal ones go to
    the lower page, one that is not a number (a NaN key) ranks last."""
    H = _heads(query, cache)
    B, width, t_stride = _table(page_table, cache)
    q_stride = _rows(query, "query", cache, B, H)
    _per_sequence(lengths, "lengths", cache, B)
    topk = int(topk)
    if topk < 1:
        raise RuntimeError("topk must be >= 1")
    pages = torch.empty((B, cache.n_kv_heads, topk), dtype=torch.int32, device=cache.device)
    nbytes = 8 * B * cache.n_kv_heads * width       # what mat_paged_select_workspace_bytes says
    with _on_device(cache):
        ws = torch.empty(nbytes, dtype=torch.uint8, device=cache.device)
        rc = _lib_select(
            cache._ref, query.data_ptr(), q_stride, B, H, page_table.data_ptr(), width, t_stride, lengths.data_ptr(), topk,
            pages.data_ptr(), ws.data_ptr(), nbytes, _raw_stream(cache._dev))
    if rc:
        nat.check(rc)
    return pages
