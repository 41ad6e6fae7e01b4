"""A paged key/value cache in FP8: written, quantized on the way, and read back.

The cache is four tensors, ``new_kv_cache_fp8`` makes them: e4m3fn codes ``k_cache``, ``v_cache`` [pages, kv_heads,
page_size, head_dim] and their fp32 scales ``k_scale``, ``v_scale`` [pages, kv_heads, page_size], one for each token
and head. Pages may lie apart (keys and values of one allocation, ``both[:, 0]`` and ``both[:, 1]``), a page itself is
contiguous. page_size is a multiple of 16, up to 1024; head_dim 64, 128 or 256.

- ``kv_cache_write_fp8(k, v, k_cache, v_cache, k_scale, v_scale, slots)`` stores [tokens, kv_heads, head_dim] keys and
  values (bf16, fp16 or fp32) at ``slots`` (int32 or int64 [tokens]: page * page_size + place in the page; negative
  ones skip their token, as do those past the cache) and returns the four tensors. The arithmetic is
  ``per_group_quant_fp8``'s (aklr/ops/quant/reference.py:9-28) with one group a head. A vector that holds a NaN or an
  infinity reads as NaN throughout. The slots of one call are distinct: a slot given twice may end with parts of both
  tokens.
- ``rotary_kv_cache_write_fp8(q, k, v, positions, frequencies, k_cache, ..., slots, *, interleaved, magnitude, out)``
  is ``rotary_embedding`` and the write in one launch: it returns the rotated q and stores the rotated k, which is
  rounded only once, to its code.
- ``kv_cache_read_fp8(k_cache, ..., block_table, starts, total, *, out_dtype, out_k, out_v)`` packs cached prefixes:
  rows ``starts[b]`` to ``starts[b + 1] - 1`` of the returned [total, kv_heads, head_dim] keys and values are
  positions 0, 1, ... of sequence b. ``block_table`` int32 [batch, columns] names each sequence's pages in order,
  ``starts`` int32 [batch + 1] ascends. Rows behind the last sequence are left as they were; a page that the cache
  does not have reads as zeros.

The reference's quantizers are the model (this cache is not in its scope here). Calls they do not serve return a
``FallbackReason``; so does a call that wants gradients or tangents.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _lib
from .dispatch import FallbackReason, aligned, api, on_gpu
from .rotary import (_DTYPES, _MAX_HEADS, apart, no_inner_overlap, rotary_ok, same_place, stream, tensors_ok,
                     vectors_ok, wants_grad)

_OOC = FallbackReason.OUT_OF_CONTRACT
_OUT = {torch.bfloat16: _lib.OUT_BF16, torch.float16: _lib.OUT_F16}


def new_kv_cache_fp8(pages, kv_heads, head_dim, page_size, device="cuda"):
    """(k_cache, v_cache, k_scale, v_scale), zeroed."""
    shape = (pages, kv_heads, page_size)
    codes = [torch.zeros(shape + (head_dim,), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn) for _ in "kv"]
    return (*codes, *(torch.zeros(shape, dtype=torch.float32, device=device) for _ in "kv"))


def _page_stride(t) -> int | None:
    """Elements from one page to the next of a cache tensor whose pages are contiguous, or None."""
    inner = 1
    for d in range(t.dim() - 1, 0, -1):
        if t.shape[d] != 1 and t.stride(d) != inner:
            return None
        inner *= t.shape[d]
    if t.shape[0] == 1:
        return inner
    return t.stride(0) if t.stride(0) >= inner else None


def cache_strides(k_cache, v_cache, k_scale, v_scale):
    """The four page strides of a cache the kernels take, or None."""
    if k_cache.dim() != 4 or k_cache.dtype != torch.float8_e4m3fn or v_cache.dtype != torch.float8_e4m3fn:
        return None
    pages, heads, page, head_dim = k_cache.shape
    if head_dim not in (64, 128, 256) or not 16 <= page <= 1024 or page % 16 or not 1 <= heads <= 1024:
        return None
    if pages < 1 or pages * page >= 2**31 or v_cache.shape != k_cache.shape:
        return None
    if k_scale.dtype != torch.float32 or v_scale.dtype != torch.float32:
        return None
    if k_scale.shape != k_cache.shape[:3] or v_scale.shape != k_cache.shape[:3]:
        return None
    if wants_grad(k_cache, v_cache, k_scale, v_scale):
        return None
    strides = []
    for t, multiple in ((k_cache, 16), (v_cache, 16), (k_scale, 4), (v_scale, 4)):
        s = _page_stride(t)
        if s is None or s % multiple or not aligned(t):
            return None
        strides.append(s)
    return strides


def table_ok(block_table, batch) -> bool:
    return (block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.shape[0] == batch
            and (block_table.shape[1] <= 1 or block_table.stride(1) == 1)
            and (batch <= 1 or block_table.stride(0) >= block_table.shape[1]))


def table_stride(block_table) -> int:
    return block_table.stride(0) if block_table.shape[0] > 1 else block_table.shape[1]


def starts_ok(starts) -> bool:
    return starts.dtype == torch.int32 and starts.dim() == 1 and starts.numel() >= 1 and starts.is_contiguous()


# ---------------------------------------------------------------------------------------------
@dataclass
class _WritePlan:
    q: torch.Tensor | None
    k: torch.Tensor
    v: torch.Tensor
    positions: torch.Tensor | None
    frequencies: torch.Tensor | None
    cache: tuple
    strides: list
    slots: torch.Tensor
    interleaved: bool
    magnitude: float
    out: torch.Tensor | None
    variant: str
    kernel_ref: str = "aklr_kv_cache_write_fp8"


def _run_write(p: _WritePlan):
    k, v, q, out = p.k, p.v, p.q, p.out
    tokens, heads, head_dim = k.shape
    turned = (None, 0, 0, None, 0, 0, 0)
    angles = (None, 0, None, 0, 0, 1.0)
    if q is not None:
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        turned = (q.data_ptr(), q.stride(0), q.stride(1), out.data_ptr(), out.stride(0), out.stride(1), q.shape[1])
        angles = (p.positions.data_ptr(), int(p.positions.dtype == torch.int64), p.frequencies.data_ptr(),
                  2 * p.frequencies.numel(), int(p.interleaved), p.magnitude)
    if tokens:
        with torch.cuda.device(k.device):
            st = _lib.lib().aklr_kv_cache_write_fp8(
                *turned, k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), *angles,
                p.slots.data_ptr(), int(p.slots.dtype == torch.int64), *(t.data_ptr() for t in p.cache), *p.strides,
                tokens, heads, head_dim, p.cache[0].shape[0], p.cache[0].shape[2], _DTYPES[k.dtype], stream(k.device))
        _lib.check(st, "kv_cache_write_fp8")
    return p.cache if q is None else out


def _write_plan(k, v, cache, slots):
    """The checks of both writes on what they share: the cache's strides, or None."""
    if not tensors_ok(k, v, slots, *cache):
        return None
    strides = cache_strides(*cache)
    if strides is None or k.dim() != 3 or k.dtype not in _DTYPES:
        return None
    tokens, (_, heads, _, head_dim) = k.shape[0], cache[0].shape
    if tokens >= 2**31 or not vectors_ok(k, tokens, heads, head_dim, k.dtype) or not vectors_ok(v, tokens, heads, head_dim, k.dtype):
        return None
    if slots.dtype not in (torch.int32, torch.int64) or tuple(slots.shape) != (tokens,) or not slots.is_contiguous():
        return None
    if not on_gpu(k, v, slots, *cache) or wants_grad(k, v):
        return None
    if not all(apart(c, t) for c in cache for t in (k, v, slots)):
        return None
    if not all(apart(cache[i], cache[j]) for i in range(4) for j in range(i)):
        return None
    return strides


@api("kv_cache_write_fp8@1.0", _run_write, native="kv_write")
def kv_cache_write_fp8(k, v, k_cache, v_cache, k_scale, v_scale, slots):
    cache = (k_cache, v_cache, k_scale, v_scale)
    strides = _write_plan(k, v, cache, slots)
    if strides is None:
        return _OOC
    return _WritePlan(None, k, v, None, None, cache, strides, slots, False, 1.0, None, "write")


@api("rotary_kv_cache_write_fp8@1.0", _run_write, native="rotary_kv_write")
def rotary_kv_cache_write_fp8(q, k, v, positions, frequencies, k_cache, v_cache, k_scale, v_scale, slots, *,
                              interleaved=False, magnitude=1.0, out=None):
    cache = (k_cache, v_cache, k_scale, v_scale)
    more = [q, positions, frequencies] + ([out] if out is not None else [])
    if not tensors_ok(*more):
        return _OOC
    strides = _write_plan(k, v, cache, slots)
    if strides is None or q.dim() != 3 or not 1 <= q.shape[1] <= _MAX_HEADS:
        return _OOC
    tokens, _, head_dim = k.shape
    if not vectors_ok(q, tokens, q.shape[1], head_dim, k.dtype):
        return _OOC
    if not rotary_ok(positions, frequencies, interleaved, magnitude, tokens, head_dim):
        return _OOC
    if not on_gpu(k, *more) or wants_grad(q, out):
        return _OOC
    if not all(apart(c, t) for c in cache for t in more):
        return _OOC
    if out is not None:
        if not vectors_ok(out, tokens, q.shape[1], head_dim, k.dtype) or not no_inner_overlap(out):
            return _OOC
        if not (same_place(out, q) or apart(out, q)) or not all(apart(out, t) for t in (k, v, positions, frequencies, slots)):
            return _OOC
    return _WritePlan(q, k, v, positions, frequencies, cache, strides, slots, interleaved, float(magnitude), out,
                      "rotary_interleaved" if interleaved else "rotary_half")


# ---------------------------------------------------------------------------------------------
@dataclass
class _ReadPlan:
    cache: tuple
    strides: list
    block_table: torch.Tensor
    starts: torch.Tensor
    total: int
    out_dtype: torch.dtype
    out_k: torch.Tensor | None
    out_v: torch.Tensor | None
    variant: str = "packed"
    kernel_ref: str = "aklr_kv_cache_read_fp8"


def _run_read(p: _ReadPlan):
    kc = p.cache[0]
    pages, heads, page, head_dim = kc.shape
    outs = [o if o is not None else torch.empty((p.total, heads, head_dim), dtype=p.out_dtype, device=kc.device)
            for o in (p.out_k, p.out_v)]
    batch = p.starts.numel() - 1
    if p.total and batch:
        with torch.cuda.device(kc.device):
            st = _lib.lib().aklr_kv_cache_read_fp8(
                *(t.data_ptr() for t in p.cache), *p.strides, p.block_table.data_ptr(), table_stride(p.block_table),
                p.block_table.shape[1], p.starts.data_ptr(), batch, p.total, outs[0].data_ptr(), outs[1].data_ptr(),
                heads, head_dim, pages, page, _OUT[p.out_dtype], stream(kc.device))
        _lib.check(st, "kv_cache_read_fp8")
    return outs[0], outs[1]


@api("kv_cache_read_fp8@1.0", _run_read, native="kv_read")
def kv_cache_read_fp8(k_cache, v_cache, k_scale, v_scale, block_table, starts, total, *, out_dtype=None, out_k=None,
                      out_v=None):
    cache = (k_cache, v_cache, k_scale, v_scale)
    outs = [o for o in (out_k, out_v) if o is not None]
    if not tensors_ok(*cache, block_table, starts, *outs):
        return _OOC
    if isinstance(total, bool) or not isinstance(total, int) or not 0 <= total < 2**31:
        return _OOC
    if out_dtype is None:
        out_dtype = outs[0].dtype if outs else torch.bfloat16
    strides = cache_strides(*cache)
    if strides is None or out_dtype not in _OUT or not starts_ok(starts) or not table_ok(block_table, starts.numel() - 1):
        return _OOC
    _, heads, _, head_dim = k_cache.shape
    for o in outs:
        if tuple(o.shape) != (total, heads, head_dim) or o.dtype != out_dtype or not o.is_contiguous() or not aligned(o):
            return _OOC
        if not all(apart(o, t) for t in (*cache, block_table, starts)):
            return _OOC
    if not apart(out_k, out_v) or not on_gpu(*cache, block_table, starts, *outs) or wants_grad(*outs):
        return _OOC
    return _ReadPlan(cache, strides, block_table, starts, total, out_dtype, out_k, out_v)
