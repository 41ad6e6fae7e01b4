"""Verification of drafted tokens: which of them stand, and the token that follows.

``verify_drafts(target_probs, draft_tokens, starts, accept_uniforms, sample_uniforms, most, *, draft_probs=None,
parents=None)`` comes after a pass of ``tree_attention_fp8`` over the same query tokens: ``starts[b]`` to
``starts[b + 1] - 1`` (int32 [batch + 1], ascending) are sequence b's, the first its last token that stands, the others
drafts. Drafted token i follows ``parents[i]`` (int32 [tokens], counted within the sequence and before i), or without
``parents`` the token before it: a chain. ``target_probs`` [tokens, vocabulary] (8 to 2^24 tokens) holds the target model's
probabilities after each query token, ``draft_probs`` (the same shape and type, bf16, fp16 or fp32) those that the drafts
after it were drawn from, independently of each other; without it the drafts were certain (a greedy draft, the likeliest tokens).

  At a node with rows p and q its drafts are tried in their order, from W = p, S = 1. Draft i with token x stands if
  ``accept_uniforms[i]`` * S * q(x) < W(x) (without q: ``accept_uniforms[i]`` * S < W(x)), and the search goes on at it; else
  W = max(W - S q, 0) and S = sum(W) (without q: S -= W(x), then W(x) = 0). Where none stands, the next token is the
  least v for which W(0) + ... + W(v) > ``sample_uniforms[b]`` * sum(W). Drafts drawn from q and uniform numbers make the
  tokens that come out the target's own samples. Where nothing is left of W, p itself is sampled; a row without any
  probability gives -1. All of it is computed in 64 bits, the sums in an order that the sizes alone set, so a call repeats
  itself; another order of the same sums may decide otherwise where a number is within some 2^-50 of a row's sum of a border.

  uniforms: fp32 [tokens] and [batch], in [0, 1); others count as the nearest that is, NaN as 0. Entries of the rows that
  are negative, infinite or NaN count as 0; rows need not add up to 1. Rows may lie apart, each is contiguous. A draft whose
  token (int32 or int64) is not in the vocabulary, or whose parent does not come before it, is passed over.
  most: the most query tokens that a sequence has, up to 1024; those of a sequence past it are not tried.

Returns (tokens, path, counts): tokens [batch, most] of ``draft_tokens``' type, the drafts that stand and then the next
token, path int32 [batch, most], which query tokens of the sequence they follow: 0, then the drafts that stand; both -1
behind ``counts[b]`` (int32 [batch]) entries. A sequence without query tokens has a count of 0. ``kv_cache_compact_fp8``
takes path and counts, ``seq_lens - (starts[1:] - starts[:-1]) + counts`` are the lengths that stand. Nothing waits for
the GPU: a captured call serves other lengths, trees and numbers of the same shapes.

Calls it does not serve return a ``FallbackReason``; so does a call that wants gradients or tangents. The reference has no
such op in this library's scope; the op follows the conventions of its other ops.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _lib, workspace
from .dispatch import FallbackReason, api, on_gpu
from .kv_cache import starts_ok
from .rotary import _DTYPES, stream, tensors_ok, wants_grad

_OOC = FallbackReason.OUT_OF_CONTRACT
_MOST, _MIN_VOCAB, _MAX_VOCAB, _MAX_BATCH = 1024, 8, 1 << 24, 65536


@dataclass
class _VerifyPlan:
    target: torch.Tensor
    tokens: torch.Tensor
    starts: torch.Tensor
    accept: torch.Tensor
    sample: torch.Tensor
    most: int
    draft: torch.Tensor | None
    parents: torch.Tensor | None
    variant: str
    kernel_ref: str = "aklr_verify_drafts"


def row_stride(t) -> int:
    """Elements from one row of a 2-D tensor to the next."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def rows_ok(t, like=None) -> bool:
    """A 2-D tensor of contiguous rows that do not meet."""
    if t.dim() != 2 or t.layout != torch.strided or (like is not None and (t.shape != like.shape or t.dtype != like.dtype)):
        return False
    return (t.shape[1] <= 1 or t.stride(1) == 1) and row_stride(t) >= t.shape[1] and t.data_ptr() % t.element_size() == 0


def vector_ok(t, n, *dtypes) -> bool:
    return t.dtype in dtypes and tuple(t.shape) == (n,) and t.layout == torch.strided and t.is_contiguous()


def _run_verify(p: _VerifyPlan):
    t, dev = p.target, p.target.device
    batch = p.sample.numel()
    out = torch.empty((batch, p.most), dtype=p.tokens.dtype, device=dev)
    path = torch.empty((batch, p.most), dtype=torch.int32, device=dev)
    counts = torch.empty(batch, dtype=torch.int32, device=dev)
    if batch:
        L = _lib.lib()
        with torch.cuda.device(dev):
            nbytes = L.aklr_verify_drafts_workspace_bytes(batch, t.shape[1], p.most)
            ws = workspace.get(dev, nbytes)
            st = L.aklr_verify_drafts(
                t.data_ptr(), row_stride(t), p.draft.data_ptr() if p.draft is not None else None,
                row_stride(p.draft) if p.draft is not None else 0, t.shape[0], t.shape[1], p.tokens.data_ptr(),
                int(p.tokens.dtype == torch.int64), p.parents.data_ptr() if p.parents is not None else None,
                p.starts.data_ptr(), p.accept.data_ptr(), p.sample.data_ptr(), batch, p.most, out.data_ptr(),
                path.data_ptr(), counts.data_ptr(), _DTYPES[t.dtype], ws.data_ptr(), nbytes, stream(dev))
        _lib.check(st, "verify_drafts")
    return out, path, counts


@api("verify_drafts@1.0", _run_verify, native="verify")
def verify_drafts(target_probs, draft_tokens, starts, accept_uniforms, sample_uniforms, most, *, draft_probs=None,
                  parents=None):
    given = [target_probs, draft_tokens, starts, accept_uniforms, sample_uniforms]
    given += [t for t in (draft_probs, parents) if t is not None]
    if not tensors_ok(*given) or target_probs.dtype not in _DTYPES or not rows_ok(target_probs):
        return _OOC
    if isinstance(most, bool) or not isinstance(most, int) or not 1 <= most <= _MOST:
        return _OOC
    tokens, vocab = target_probs.shape
    if not _MIN_VOCAB <= vocab <= _MAX_VOCAB or tokens >= 2**31 or not starts_ok(starts) or starts.numel() > _MAX_BATCH + 1:
        return _OOC
    if draft_probs is not None and not rows_ok(draft_probs, target_probs):
        return _OOC
    if not vector_ok(draft_tokens, tokens, torch.int32, torch.int64) or not vector_ok(accept_uniforms, tokens, torch.float32):
        return _OOC
    if not vector_ok(sample_uniforms, starts.numel() - 1, torch.float32):
        return _OOC
    if parents is not None and not vector_ok(parents, tokens, torch.int32):
        return _OOC
    if not on_gpu(*given) or wants_grad(target_probs, accept_uniforms, sample_uniforms, draft_probs):
        return _OOC
    return _VerifyPlan(target_probs, draft_tokens, starts, accept_uniforms, sample_uniforms, most, draft_probs, parents,
                       ("chain" if parents is None else "tree") + ("" if draft_probs is not None else "_certain"))
