"""Low-rank adapters of many requests at once, beside a projection that all of them share.

``lora_project(x, a, b, adapters, base, *, scales=None, ranks=None, out=None)`` returns
``base[t] + scales[i] * (x[t] a[i]^T) b[i]^T`` with i = ``adapters[t]``:

  x [tokens, K] is what the projection took, base [tokens, N] what it gave (``gemm_a8w8_blockwise_scaled``'s output, say);
  a [adapters, R, K] and b [adapters, N, R] hold the adapters, all bf16 or all fp16. ``adapters`` (int32 or int64 [tokens]):
  each token's, in any order; a token whose number is no adapter's keeps its base. ``scales``: fp32 [adapters], 1 unless
  given. ``ranks``: int32 [adapters], 0 to R: the rows of a[i] and columns of b[i] from there on are not read (they may hold
  anything). K, N and R are multiples of 8, K up to 65536, N up to 262144, R up to 128; up to 2^20 tokens and 4096 adapters.
  x, base and out may be rows of something wider, a and b slices of what several projections stack: the last dimension is
  contiguous and everything else lies on 16 bytes. ``out``: where the result goes, base itself for in place (x may then be
  base too), else apart from all that is read.

  x a^T is held in 32 bits and enters the second product as 16-bit pieces: whole (bf16, three pieces) or off by 2^-23 of it
  or 2^-39 of the token's largest (fp16, two); base is added in fp32, and the sum rounded once. What is not finite in a token or in its adapter
  comes out not finite, an infinity perhaps as NaN, and no other token sees it.

Nothing waits for the GPU, and a captured call serves other adapters of the same shapes. Calls it does not serve return a
``FallbackReason``; so does a call that wants gradients or tangents. The reference has no such op in this library's scope.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _lib, workspace
from .dispatch import FallbackReason, aligned, api, on_gpu
from .drafts import vector_ok
from .kv_cache import _OUT
from .rotary import apart, no_inner_overlap, same_place, stream, tensors_ok, wants_grad

_OOC = FallbackReason.OUT_OF_CONTRACT


@dataclass
class _LoraPlan:
    x: torch.Tensor
    a: torch.Tensor
    b: torch.Tensor
    adapters: torch.Tensor
    base: torch.Tensor
    scales: torch.Tensor | None
    ranks: torch.Tensor | None
    out: torch.Tensor | None
    variant: str
    kernel_ref: str = "aklr_lora_project"


def _pieces_ok(t, dtype, *shape) -> bool:
    """A tensor of 16-byte pieces along its last dimension."""
    if tuple(t.shape) != shape or t.dtype != dtype or t.layout != torch.strided or t.stride(-1) != 1 or not aligned(t):
        return False
    return all(s % 8 == 0 for s in t.stride()[:-1])


def _run_lora(p: _LoraPlan):
    x, a, b, base, dev = p.x, p.a, p.b, p.base, p.x.device
    out = p.out if p.out is not None else torch.empty(base.shape, dtype=base.dtype, device=dev)
    tokens, k = x.shape
    count, n, rank = b.shape
    if tokens:
        L = _lib.lib()
        with torch.cuda.device(dev):
            nbytes = L.aklr_lora_project_workspace_bytes(tokens, k, n, rank, count)
            ws = workspace.get(dev, nbytes)
            st = L.aklr_lora_project(
                x.data_ptr(), x.stride(0), a.data_ptr(), a.stride(0), a.stride(1), b.data_ptr(), b.stride(0), b.stride(1),
                p.adapters.data_ptr(), int(p.adapters.dtype == torch.int64), p.scales.data_ptr() if p.scales is not None else None,
                p.ranks.data_ptr() if p.ranks is not None else None, base.data_ptr(), base.stride(0), out.data_ptr(),
                out.stride(0), tokens, k, n, rank, count, _OUT[x.dtype], ws.data_ptr(), nbytes, stream(dev))
        _lib.check(st, "lora_project")
    return out


@api("lora_project@1.0", _run_lora, native="lora")
def lora_project(x, a, b, adapters, base, *, scales=None, ranks=None, out=None):
    given = [x, a, b, adapters, base] + [t for t in (scales, ranks, out) if t is not None]
    if not tensors_ok(*given) or x.dim() != 2 or b.dim() != 3 or x.dtype not in _OUT:
        return _OOC
    (tokens, k), (count, n, rank) = x.shape, b.shape
    if not (8 <= k <= 65536 and k % 8 == 0 and 8 <= n <= 262144 and n % 8 == 0 and 8 <= rank <= 128 and rank % 8 == 0):
        return _OOC
    if tokens > 2**20 or not 1 <= count <= 4096:
        return _OOC
    if not _pieces_ok(x, x.dtype, tokens, k) or not _pieces_ok(a, x.dtype, count, rank, k):
        return _OOC
    if not _pieces_ok(b, x.dtype, count, n, rank):
        return _OOC
    if not _pieces_ok(base, x.dtype, tokens, n) or not vector_ok(adapters, tokens, torch.int32, torch.int64):
        return _OOC
    if scales is not None and not vector_ok(scales, count, torch.float32):
        return _OOC
    if ranks is not None and not vector_ok(ranks, count, torch.int32):
        return _OOC
    if not on_gpu(*given) or wants_grad(x, a, b, base, scales, out):
        return _OOC
    if out is not None:
        if not _pieces_ok(out, x.dtype, tokens, n) or not no_inner_overlap(out):
            return _OOC
        if not (same_place(out, base) or apart(out, base)) or not all(apart(out, t) for t in (a, b, adapters, scales, ranks)):
            return _OOC
        if not (apart(out, x) or (same_place(out, x) and same_place(out, base))):
            return _OOC
    return _LoraPlan(x, a, b, adapters, base, scales, ranks, out, "decode" if tokens <= 256 else "sorted")
