"""Pages of the FP8 cache of ``aklr_amd.kv_cache``: copied, compacted, and handed from sequence to sequence.

- ``kv_cache_copy_pages_fp8(k_cache, v_cache, k_scale, v_scale, src, dst)`` copies page ``src[i]`` onto page ``dst[i]``
  (int32 or int64 [pages to copy], both the same) and returns the four tensors. The same page may be copied to several
  places; the pages of ``dst`` are distinct and none of ``src``. Pairs of which one is not a page of the cache are skipped.
- ``kv_cache_compact_fp8(k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, starts, path, counts)`` moves kept
  positions together. Of the last T = ``starts[b + 1] - starts[b]`` of sequence b's ``seq_lens[b]`` positions, the
  ``counts[b]`` with the numbers ``path[b]`` (int32 [batch, most], ascending) become the first ones: position
  ``seq_lens[b] - T + path[b, i]`` moves to ``seq_lens[b] - T + i``. That is what ``verify_drafts`` returns for the drafts of
  ``tree_attention_fp8``'s call; with T the whole length it cuts a context to the positions worth keeping. Returns the four
  tensors. Positions in pages that the cache does not have stay, and so does what is not kept, behind. Entries of a path that
  are none of the T positions, wherever they stand, are passed over; the others ascend. The pages that
  positions move to belong to one sequence. Those behind what ``kv_cache_update_pages`` was last told to keep do; whoever cuts
  a context whose first pages others hold too copies them before.
- ``kv_cache_update_pages(page_refs, block_table, lens, new_lens, page_size, parents=None)`` says which pages each sequence
  holds next, for all layers that share a block table. ``page_refs`` (int32 [pages], zeros to begin with) counts the entries
  of block tables, and whoever else, that hold each page; a page with 0 is free. It is updated in place. Sequence b had
  ``lens[b]`` positions (int32 [batch]) in the pages of row b of ``block_table`` (int32 [batch, columns]) and gets
  ``new_lens[b]``: it goes on from the first of them that its parent had, itself or ``parents[b]`` (int32 [batch]; one that
  is no sequence: it begins empty). So a sequence grows, gives up what was not kept, ends (0), or becomes a fork of another,
  and beams change places, in one call.

  Whole pages that are kept are shared. A page of which a part is kept is written on: if nobody else holds it any more, the
  lowest of the sequences that keep a part goes on in it, and the others get a copy, as all do where somebody else holds it.
  New pages are the lowest free ones, in the order of sequences and columns; pages given up in the call are among them.
  Returns (table, granted, src, dst): the new block table [batch, columns], -1 behind what a sequence holds, the positions it
  has pages for (``new_lens`` up to the columns' room, less where the free pages end), and for ``kv_cache_copy_pages_fp8``,
  once a layer and before anything is written, the pages to copy (int32 [batch], -1: none). Entries that name no page
  stay -1 and hold nothing.

The cache is as ``aklr_amd.kv_cache`` describes it, up to 65536 sequences, a block table reaches 2^28 positions. Nothing
waits for the GPU, and a captured call serves other values of the same shapes. Calls that are not served return a
``FallbackReason``; so does a call that wants gradients or tangents. The reference has no such ops in this library's scope.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _lib, workspace
from .dispatch import FallbackReason, aligned, api, on_gpu
from .drafts import row_stride, vector_ok
from .kv_cache import cache_strides, starts_ok, table_ok, table_stride
from .rotary import apart, stream, tensors_ok

_OOC = FallbackReason.OUT_OF_CONTRACT
_MAX_BATCH = 65536


def new_kv_page_refs(pages, device="cuda"):
    """The holders of a cache's pages, for ``kv_cache_update_pages``: nobody."""
    return torch.zeros(pages, dtype=torch.int32, device=device)


def _cache_ok(cache, *others):
    """The strides of a cache whose tensors share no memory with each other or with the others, or None."""
    strides = cache_strides(*cache)
    if strides is None or not on_gpu(*cache, *others):
        return None
    if not all(apart(cache[i], cache[j]) for i in range(4) for j in range(i)):
        return None
    if not all(apart(c, t) for c in cache for t in others):
        return None
    return strides


def _rows_ok(t, batch) -> bool:
    """An int32 table with a row for each sequence, one of no rows with any strides."""
    return table_ok(t, batch) or (batch == 0 and t.dtype == torch.int32 and t.dim() == 2 and t.shape[0] == 0)


# ---------------------------------------------------------------------------------------------
@dataclass
class _CopyPlan:
    cache: tuple
    strides: list
    src: torch.Tensor
    dst: torch.Tensor
    variant: str = "pages"
    kernel_ref: str = "aklr_kv_cache_copy_pages_fp8"


def _run_copy(p: _CopyPlan):
    kc = p.cache[0]
    pages, heads, page, head_dim = kc.shape
    if p.src.numel():
        with torch.cuda.device(kc.device):
            st = _lib.lib().aklr_kv_cache_copy_pages_fp8(
                *(t.data_ptr() for t in p.cache), *p.strides, p.src.data_ptr(), p.dst.data_ptr(),
                int(p.src.dtype == torch.int64), p.src.numel(), heads, head_dim, pages, page, stream(kc.device))
        _lib.check(st, "kv_cache_copy_pages_fp8")
    return p.cache


@api("kv_cache_copy_pages_fp8@1.0", _run_copy, native="kv_copy")
def kv_cache_copy_pages_fp8(k_cache, v_cache, k_scale, v_scale, src, dst):
    cache = (k_cache, v_cache, k_scale, v_scale)
    if not tensors_ok(*cache, src, dst) or src.dim() != 1 or src.numel() >= 2**31:
        return _OOC
    if not vector_ok(src, src.numel(), torch.int32, torch.int64) or not vector_ok(dst, src.numel(), src.dtype):
        return _OOC
    strides = _cache_ok(cache, src, dst)
    if strides is None:
        return _OOC
    return _CopyPlan(cache, strides, src, dst)


# ---------------------------------------------------------------------------------------------
@dataclass
class _CompactPlan:
    cache: tuple
    strides: list
    block_table: torch.Tensor
    seq_lens: torch.Tensor
    starts: torch.Tensor
    path: torch.Tensor
    counts: torch.Tensor
    variant: str
    kernel_ref: str = "aklr_kv_cache_compact_fp8"


def _run_compact(p: _CompactPlan):
    kc = p.cache[0]
    pages, heads, page, head_dim = kc.shape
    batch, most = p.path.shape
    if batch and most and p.block_table.shape[1]:
        L = _lib.lib()
        with torch.cuda.device(kc.device):
            nbytes = L.aklr_kv_cache_compact_fp8_workspace_bytes(batch, most, heads, head_dim)
            ws = workspace.get(kc.device, nbytes)
            st = L.aklr_kv_cache_compact_fp8(
                *(t.data_ptr() for t in p.cache), *p.strides, p.block_table.data_ptr(), table_stride(p.block_table),
                p.block_table.shape[1], p.seq_lens.data_ptr(), p.starts.data_ptr(), p.path.data_ptr(), row_stride(p.path), most,
                p.counts.data_ptr(), batch, heads, head_dim, pages, page, ws.data_ptr() if ws is not None else None, nbytes,
                stream(kc.device))
        _lib.check(st, "kv_cache_compact_fp8")
    return p.cache


@api("kv_cache_compact_fp8@1.0", _run_compact, native="kv_compact")
def kv_cache_compact_fp8(k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, starts, path, counts):
    cache = (k_cache, v_cache, k_scale, v_scale)
    if not tensors_ok(*cache, block_table, seq_lens, starts, path, counts) or seq_lens.dim() != 1:
        return _OOC
    batch = seq_lens.numel()
    if batch > _MAX_BATCH or not starts_ok(starts) or starts.numel() != batch + 1 or not _rows_ok(block_table, batch):
        return _OOC
    if not vector_ok(seq_lens, batch, torch.int32) or not vector_ok(counts, batch, torch.int32):
        return _OOC
    if not _rows_ok(path, batch) or path.shape[1] > 2**28:
        return _OOC
    strides = _cache_ok(cache, block_table, seq_lens, starts, path, counts)
    if strides is None or block_table.shape[1] * k_cache.shape[2] > 2**28:
        return _OOC
    return _CompactPlan(cache, strides, block_table, seq_lens, starts, path, counts, "short" if path.shape[1] <= 64 else "long")


# ---------------------------------------------------------------------------------------------
@dataclass
class _UpdatePlan:
    refs: torch.Tensor
    block_table: torch.Tensor
    lens: torch.Tensor
    new_lens: torch.Tensor
    page_size: int
    parents: torch.Tensor | None
    variant: str
    kernel_ref: str = "aklr_kv_cache_update_pages"


def _run_update(p: _UpdatePlan):
    dev = p.refs.device
    batch, cols = p.block_table.shape
    table = torch.empty((batch, cols), dtype=torch.int32, device=dev)
    granted, src, dst = (torch.empty(batch, dtype=torch.int32, device=dev) for _ in range(3))
    if batch:
        L = _lib.lib()
        with torch.cuda.device(dev):
            nbytes = L.aklr_kv_cache_update_pages_workspace_bytes(batch)
            ws = workspace.get(dev, nbytes)
            st = L.aklr_kv_cache_update_pages(
                p.refs.data_ptr(), p.refs.numel(), p.block_table.data_ptr(), table_stride(p.block_table), cols,
                p.lens.data_ptr(), p.new_lens.data_ptr(), p.parents.data_ptr() if p.parents is not None else None, batch,
                p.page_size, table.data_ptr(), granted.data_ptr(), src.data_ptr(), dst.data_ptr(), ws.data_ptr(), nbytes,
                stream(dev))
        _lib.check(st, "kv_cache_update_pages")
    return table, granted, src, dst


@api("kv_cache_update_pages@1.0", _run_update, native="kv_update")
def kv_cache_update_pages(page_refs, block_table, lens, new_lens, page_size, parents=None):
    given = [block_table, lens, new_lens] + ([parents] if parents is not None else [])
    if not tensors_ok(page_refs, *given) or page_refs.dim() != 1 or lens.dim() != 1:
        return _OOC
    if isinstance(page_size, bool) or not isinstance(page_size, int) or page_size < 1:
        return _OOC
    batch, pages = lens.numel(), page_refs.numel()
    if batch > _MAX_BATCH or pages < 1 or pages * page_size >= 2**31 or not _rows_ok(block_table, batch):
        return _OOC
    cols = block_table.shape[1]
    if cols * page_size > 2**28 or batch * cols >= 2**31:
        return _OOC
    if not vector_ok(page_refs, pages, torch.int32) or not aligned(page_refs):
        return _OOC
    if not all(vector_ok(t, batch, torch.int32) for t in (lens, new_lens, parents) if t is not None):
        return _OOC
    if not on_gpu(page_refs, *given) or not all(apart(page_refs, t) for t in given):
        return _OOC
    return _UpdatePlan(page_refs, block_table, lens, new_lens, page_size, parents, "grow" if parents is None else "fork")
