"""Attention over the paged FP8 cache of ``aklr_amd.kv_cache``: decode, trees of drafted tokens, chunks of a prompt.

``tree_attention_fp8(q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, starts, tree_mask=None, *,
softmax_scale=None, return_lse=False, out=None)``:

  q: bf16 or fp16 [tokens, q_heads, head_dim], query tokens ``starts[b]`` to ``starts[b + 1] - 1`` (int32 [batch + 1],
  ascending) are sequence b's; q_heads is a multiple of the cache's kv_heads, head h attends kv head
  h // (q_heads // kv_heads). Their keys and values are already in the cache, as the last of the sequence's
  ``seq_lens[b]`` (int32) positions; ``block_table`` (int32 [batch, columns]) names its pages in order. A length past
  the table's columns counts as what they hold; positions in pages that the cache does not have are not seen.
  Every query token sees all positions before its sequence's query tokens. Of those, query token i (counted over q)
  sees the j-th where ``tree_mask[i, j]`` (bool or uint8 [tokens, columns], columns at least the most query tokens a
  sequence has), or without a mask those up to itself: one token a sequence is decode, several a chunk of a prompt or a
  chain of drafts. ``softmax_scale``: head_dim ** -0.5 unless given.

  Keys' pages lie as far apart as values', and their scales' likewise (the cache's own layout, or both in one
  allocation). A block table reaches 2^28 positions, tokens * q_heads 2^28, sequences times kv_heads about 2^24.

  Scores, their maxima and sums are fp32. A position's weight times its value scale is rounded before the product with
  its codes: to 16 bits in calls of up to 32 rows (query tokens x q_heads // kv_heads) a sequence on the mean, in calls of
  few rows altogether, and for fp16 queries always; to 8 bits (bf16, half a step of the output's type) for bf16 queries in
  larger calls. Such a weight may reach 2^20, so values past 2^100 can overflow, and
  make a row NaN, for both types.

  Returns q's shape and dtype, with ``return_lse`` also the fp32 [tokens, q_heads] log of each softmax's sum, by which
  parts of a context can be joined. A token that sees nothing gets zeros and -inf. Nothing of a position that a token
  does not see reaches it, NaN included. Query tokens behind the last sequence (a padded batch) leave ``out`` as it
  was. Lengths stay on the device: nothing waits for the GPU, and a captured call serves other lengths, tables and
  masks of the same shapes.

Calls it does not serve return a ``FallbackReason``; so does a call that wants gradients or tangents. The reference's
attention ops are outside this library's scope; the op follows the conventions of its other ops.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _lib, workspace
from .dispatch import FallbackReason, aligned, api, on_gpu
from .kv_cache import _OUT, cache_strides, starts_ok, table_ok, table_stride
from .rotary import apart, flag_ok, number_ok, stream, tensors_ok, vectors_ok, wants_grad

_OOC = FallbackReason.OUT_OF_CONTRACT


@dataclass
class _AttentionPlan:
    q: torch.Tensor
    cache: tuple
    strides: list
    block_table: torch.Tensor
    seq_lens: torch.Tensor
    starts: torch.Tensor
    mask: torch.Tensor | None
    scale: float
    return_lse: bool
    out: torch.Tensor | None
    variant: str
    kernel_ref: str = "aklr_tree_attention_fp8"


def _run_attention(p: _AttentionPlan):
    q, dev = p.q, p.q.device
    tokens, heads, head_dim = q.shape
    pages, kv_heads, page, _ = p.cache[0].shape
    out = p.out if p.out is not None else torch.empty((tokens, heads, head_dim), dtype=q.dtype, device=dev)
    lse = torch.empty((tokens, heads), dtype=torch.float32, device=dev) if p.return_lse else None
    batch, cols = p.seq_lens.numel(), p.block_table.shape[1]
    if tokens and batch:
        L = _lib.lib()
        mask = p.mask
        with torch.cuda.device(dev):
            nbytes = L.aklr_tree_attention_fp8_workspace_bytes(tokens, batch, heads, kv_heads, head_dim, cols * page)
            ws = workspace.get(dev, nbytes)
            st = L.aklr_tree_attention_fp8(
                q.data_ptr(), q.stride(0), q.stride(1), *(t.data_ptr() for t in p.cache), p.strides[0],
                p.strides[2], p.block_table.data_ptr(), table_stride(p.block_table), cols, p.seq_lens.data_ptr(), p.starts.data_ptr(),
                mask.data_ptr() if mask is not None else None, mask.stride(0) if mask is not None else 0,
                mask.shape[1] if mask is not None else 0, out.data_ptr(), lse.data_ptr() if lse is not None else None,
                tokens, batch, heads, kv_heads, head_dim, pages, page, p.scale, _OUT[q.dtype],
                ws.data_ptr() if ws is not None else None, nbytes, stream(dev))
        _lib.check(st, "tree_attention_fp8")
    return (out, lse) if p.return_lse else out


@api("tree_attention_fp8@1.0", _run_attention, native="tree_attention")
def tree_attention_fp8(q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, starts, tree_mask=None, *,
                       softmax_scale=None, return_lse=False, out=None):
    cache = (k_cache, v_cache, k_scale, v_scale)
    inputs = [q, *cache, block_table, seq_lens, starts] + ([tree_mask] if tree_mask is not None else [])
    given = inputs + ([out] if out is not None else [])
    if not tensors_ok(*given) or not flag_ok(return_lse):
        return _OOC
    strides = cache_strides(*cache)
    if strides is None or strides[0] != strides[1] or strides[2] != strides[3] or q.dim() != 3 or q.dtype not in _OUT:
        return _OOC
    tokens, heads, head_dim = q.shape
    _, kv_heads, page, cache_dim = k_cache.shape
    if head_dim != cache_dim or heads < kv_heads or heads % kv_heads or heads > 65536:
        return _OOC
    if not vectors_ok(q, tokens, heads, head_dim, q.dtype):
        return _OOC
    if seq_lens.dtype != torch.int32 or seq_lens.dim() != 1 or not seq_lens.is_contiguous():
        return _OOC
    batch = seq_lens.numel()
    if batch > 65536 or not starts_ok(starts) or starts.numel() != batch + 1 or not table_ok(block_table, batch):
        return _OOC
    if block_table.shape[1] * page > 2**28 or strides[0] >= 2**32 or strides[2] >= 2**30 or tokens * heads >= 2**28:
        return _OOC
    if tree_mask is not None:
        if tree_mask.dtype not in (torch.bool, torch.uint8) or tree_mask.dim() != 2 or tree_mask.shape[0] != tokens:
            return _OOC
        if tree_mask.shape[1] > 1 and tree_mask.stride(1) != 1:
            return _OOC
    if softmax_scale is None:
        softmax_scale = head_dim ** -0.5
    elif not number_ok(softmax_scale):
        return _OOC
    if not on_gpu(*given) or wants_grad(q, out):
        return _OOC
    if out is not None:
        if tuple(out.shape) != tuple(q.shape) or out.dtype != q.dtype or not out.is_contiguous() or not aligned(out):
            return _OOC
        if not all(apart(out, t) for t in inputs):
            return _OOC
    if tokens and batch and not _lib.lib().aklr_tree_attention_fp8_rows(
            tokens, batch, heads, kv_heads, head_dim, block_table.shape[1] * page, None):
        return _OOC  # more workgroups than a launch has room for
    return _AttentionPlan(q, cache, strides, block_table, seq_lens, starts, tree_mask, float(softmax_scale),
                          bool(return_lse), out, "tree" if tree_mask is not None else "causal")
