"""Attention over blocks of keys that a cheap score selects for each query, with its gradients.

``select_blocks`` picks the blocks, ``forward_selected`` / ``backward_selected`` attend over them, and
``selected_block_attention`` is the differentiable call of the three.  The selection itself has no gradient.  The
serving form for single tokens is ``paged_attention.select_pages`` with ``paged_attention.decode``: with pages of
``block`` tokens it reads the keys that the last row of a sequence reads here.

Tensors are contiguous [B, S, heads, head_dim], as everywhere in this package; ``key`` and ``value`` may have fewer
heads than ``query`` (query head h reads key head h // (H / H_kv)), and the heads that share a key head share one
selection.  Work is enqueued on torch's current stream; ``RuntimeError`` for what the kernels refuse.
"""
from __future__ import annotations

import ctypes as C
from typing import List, Optional, Tuple

import torch

from . import _native as nat
from .sparse_attention_cuda import _DTYPES, _check_inputs


def _shapes(query: torch.Tensor, key: torch.Tensor, value: Optional[torch.Tensor]):
    _check_inputs(query, key, *(() if value is None else (value,)))
    B, S, H, D = query.shape
    if key.shape[0] != B or key.shape[1] != S or key.shape[3] != D or (value is not None and value.shape != key.shape):
        raise RuntimeError("key and value must be [B, S, H_kv, D] beside a query of [B, S, H, D]")
    return B, S, H, int(key.shape[2]), D, _DTYPES[query.dtype]


def _check_blocks(blocks: torch.Tensor, query: torch.Tensor, Hkv: int) -> int:
    if (blocks.dtype is not torch.int32 or blocks.dim() != 4 or blocks.device != query.device or not blocks.is_contiguous()
            or tuple(blocks.shape[:3]) != (query.shape[0], query.shape[1], Hkv)):
        raise RuntimeError("blocks must be a contiguous int32 [B, S, H_kv, topk] tensor on the inputs' device")
    return int(blocks.shape[3])


def _scratch(nbytes: int, device: torch.device) -> torch.Tensor:
    # from torch's allocator call by call: graphs captured from different calls never share it
    return torch.empty(max(int(nbytes), 256), dtype=torch.uint8, device=device)


def select_blocks(query: torch.Tensor, key: torch.Tensor, block: int, topk: int, causal: bool = True) -> torch.Tensor:
    """The ``topk`` blocks of ``block`` keys each query reads: [B, S, H_kv, topk] int32, ascending, -1 behind the last.

    A query's own block is always among them; the others are the best by an upper bound of the group's q . k over the
    block's keys (sum over query heads and columns of max(q * lo, q * hi), lo and hi the block's smallest and largest
    key).  ``causal``: blocks behind the query's own are not eligible.  Scores are compared in 64 bits, equal ones go to
    the lower block, one that is not a number (a NaN key) ranks last.  ``block``: a multiple of 16 up to 128; head widths: multiples of 8 up to 128.
    """
    B, S, H, Hkv, D, dt = _shapes(query, key, None)
    topk, block = int(topk), int(block)
    if topk < 1:
        raise RuntimeError("topk must be >= 1")
    out = torch.empty((B, S, Hkv, topk), dtype=torch.int32, device=query.device)
    with torch.cuda.device(query.device):
        ws = _scratch(nat.lib.mat_select_blocks_workspace_bytes(B, S, H, Hkv, D, dt, block, topk), query.device)
        nat.check(nat.lib.mat_select_blocks(
            query.data_ptr(), key.data_ptr(), B, S, H, Hkv, D, dt, block, topk, bool(causal), out.data_ptr(), ws.data_ptr(),
            ws.numel(), C.c_void_p(torch.cuda.current_stream(query.device).cuda_stream)))
    return out


def forward_selected(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, blocks: torch.Tensor, block: int,
                     causal: bool = True, scale: Optional[float] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Attention over the listed blocks: (out [B, S, H, D], lse [B, S, H] fp32, the natural logarithm of each row's sum).

    An entry of ``blocks`` counts when it names a block of the sequence, is above every entry before it in its row and,
    with ``causal``, not behind the query's own block; other entries are skipped.  A row without keys is zero, its lse
    -inf; a row whose keys all score -inf is NaN, as its softmax."""
    B, S, H, Hkv, D, dt = _shapes(query, key, value)
    topk = _check_blocks(blocks, query, Hkv)
    out = torch.empty_like(query)
    lse = torch.empty((B, S, H), dtype=torch.float32, device=query.device)
    with torch.cuda.device(query.device):
        ws = _scratch(nat.lib.mat_selected_attn_fwd_workspace_bytes(B, S, H, Hkv, D, dt, int(block), topk), query.device)
        nat.check(nat.lib.mat_selected_attn_fwd(
            query.data_ptr(), key.data_ptr(), value.data_ptr(), out.data_ptr(), lse.data_ptr(), B, S, H, Hkv, D, dt,
            blocks.data_ptr(), int(block), topk, bool(causal), float(scale) if scale else 0.0, ws.data_ptr(), ws.numel(),
            C.c_void_p(torch.cuda.current_stream(query.device).cuda_stream)))
    return out, lse


def backward_selected(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, out: torch.Tensor, lse: torch.Tensor,
                      grad_out: torch.Tensor, blocks: torch.Tensor, block: int, causal: bool = True,
                      scale: Optional[float] = None) -> List[torch.Tensor]:
    """[dQ, dK, dV] of ``forward_selected``, given its results.  Deterministic (no atomics); the gradients of a shared
    key head sum over its query heads.  Infinities and NaN reach the gradients of the pairs that see them only."""
    B, S, H, Hkv, D, dt = _shapes(query, key, value)
    topk = _check_blocks(blocks, query, Hkv)
    _check_inputs(query, out, grad_out)
    if out.shape != query.shape or grad_out.shape != query.shape:
        raise RuntimeError("out and grad_out must have query's shape")
    if lse.dtype is not torch.float32 or tuple(lse.shape) != (B, S, H) or not lse.is_contiguous() or lse.device != query.device:
        raise RuntimeError("lse must be the contiguous float32 [B, S, H] tensor that forward_selected returned")
    dq, dk, dv = torch.empty_like(query), torch.empty_like(key), torch.empty_like(value)
    with torch.cuda.device(query.device):
        ws = _scratch(nat.lib.mat_selected_attn_bwd_workspace_bytes(B, S, H, Hkv, D, dt, int(block), topk), query.device)
        nat.check(nat.lib.mat_selected_attn_bwd(
            query.data_ptr(), key.data_ptr(), value.data_ptr(), out.data_ptr(), lse.data_ptr(), grad_out.data_ptr(),
            dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), B, S, H, Hkv, D, dt, blocks.data_ptr(), int(block), topk, bool(causal),
            float(scale) if scale else 0.0, ws.data_ptr(), ws.numel(),
            C.c_void_p(torch.cuda.current_stream(query.device).cuda_stream)))
    return [dq, dk, dv]


class SelectedBlockAttentionFunction(torch.autograd.Function):
    """Autograd function around the three calls; non-contiguous inputs are copied."""

    @staticmethod
    def forward(ctx, query, key, value, block, topk, causal, scale):
        q, k, v = query.contiguous(), key.contiguous(), value.contiguous()
        blocks = select_blocks(q, k, block, topk, causal)
        out, lse = forward_selected(q, k, v, blocks, block, causal, scale)
        ctx.save_for_backward(q, k, v, out, lse, blocks)
        ctx.block, ctx.causal, ctx.scale = block, causal, scale
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_output):
        q, k, v, out, lse, blocks = ctx.saved_tensors
        grads = backward_selected(q, k, v, out, lse, grad_output.contiguous(), blocks, ctx.block, ctx.causal, ctx.scale)
        need = ctx.needs_input_grad
        return (*(g if n else None for g, n in zip(grads, need)), None, None, None, None)


def selected_block_attention(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, block: int = 64, topk: int = 16,
                             causal: bool = True, scale: Optional[float] = None) -> torch.Tensor:
    """Differentiable block-selected attention over [B, S, heads, head_dim] tensors."""
    return SelectedBlockAttentionFunction.apply(query, key, value, int(block), int(topk), bool(causal), scale)
