"""Pages of a cache as such: records copied from page to page, bounds of the keys of a page."""
from __future__ import annotations

import ctypes
from array import array

import torch

from . import _lib
from .attention import PagedKVCache
from .workspace import default_workspace


def copy_pages(caches, src, dst) -> None:
    """Record ``src[i]`` -> record ``dst[i]`` in every one of ``caches`` (a ``PagedKVCache``, a contiguous tensor of records along its first
    dimension, or a list of them: the layers of a model), in one launch per 64 of them.

    The page numbers are on the host, as those who hand pages out have them.  No page is written twice or read as well as written, so the
    order of the copies does not matter; a captured call copies the same pages in every replay."""
    if not isinstance(caches, (list, tuple)):
        caches = [caches]
    arrays = [c.data if isinstance(c, PagedKVCache) else c for c in caches]
    src, dst = array("i", src), array("i", dst)
    n = len(src)
    if n != len(dst):
        raise ValueError(f"{n} pages to copy to {len(dst)}")
    if not n or not arrays:
        return
    written = set(dst)
    if len(written) != n or not written.isdisjoint(src):
        raise ValueError("a page is written twice, or written and read")
    lo, hi, index = min(min(src), min(dst)), max(max(src), max(dst)), arrays[0].get_device()
    if lo < 0:
        raise IndexError(f"page {lo}")
    at, sizes = array("Q"), array("q")
    shape = dtype = None                          # of the array before: a model's layers are alike, and there are many
    for a in arrays:
        if a.shape != shape or a.dtype != dtype:
            shape, dtype = a.shape, a.dtype
            records = shape[0] if len(shape) > 1 else 0
            if hi >= records:
                raise IndexError(f"pages {lo} to {hi} of {records}")
            size = a.nbytes // records
        start = a.data_ptr()
        if a.get_device() != index or index < 0 or not a.is_contiguous():
            raise ValueError("records lie in contiguous tensors on one GPU")
        if size % 16 or start % 16:
            raise ValueError("records are whole pieces of 16 bytes")
        if size:
            at.append(start)
            sizes.append(size)
    rc = _lib.on_device(arrays[0].device, _lib.lib().b200_copy_pages, at.buffer_info()[0], sizes.buffer_info()[0], len(at), src.buffer_info()[0],
                        dst.buffer_info()[0], n)
    _lib.check(rc, "copy_pages")


def bounds_for(cache: PagedKVCache) -> torch.Tensor:
    """Room for the bounds of every page of ``cache``: [pages][kv_heads][2 (smallest, largest)][dk]."""
    return torch.zeros((cache.num_pages, cache.kv_heads, 2, cache.dk), dtype=cache.data.dtype, device=cache.data.device)


def check_bounds(cache: PagedKVCache, bounds: torch.Tensor) -> None:
    data = cache.data
    if bounds.shape != (cache.num_pages, cache.kv_heads, 2, cache.dk) or bounds.dtype != data.dtype or not bounds.is_contiguous() \
            or bounds.get_device() != data.get_device():
        raise ValueError(f"bounds {tuple(bounds.shape)} {bounds.dtype} of a cache of {cache.num_pages} pages, {cache.kv_heads} heads of {cache.dk}, {cache.data.dtype}")


def on_one_gpu(*tensors: torch.Tensor | None) -> None:
    """Kernels are given addresses: those of one GPU's memory."""
    index = tensors[0].get_device()
    for t in tensors:
        if t is not None and (t.get_device() != index or index < 0):
            raise ValueError("tensors on one GPU")


def page_bounds(cache: PagedKVCache, page_table: torch.Tensor, starts: torch.Tensor, ends: torch.Tensor, seq_ids: torch.Tensor | None, max_tokens: int,
                bounds: torch.Tensor) -> torch.Tensor:
    """Smallest and largest element of the keys of a page, per KV head and dimension, for all pages that hold tokens ``starts[i]`` to
    ``ends[i] - 1`` (int32) of sequence ``seq_ids[i]`` (None: i); all tokens of such a page up to ``ends[i]`` count, nothing behind them is read.
    ``max_tokens``: the most that a portion has; one that has more pages than that may is left out, which the status word says.  A page is touched by one
    portion only.  A portion of no tokens, as of an empty slot, changes nothing.  Exact; NaN where a key is."""
    check_bounds(cache, bounds)
    on_one_gpu(bounds, page_table, starts, ends, seq_ids)
    n = starts.numel()
    assert starts.dtype == ends.dtype == page_table.dtype == torch.int32 and ends.numel() == n and starts.is_contiguous() and ends.is_contiguous() and page_table.is_contiguous()
    if seq_ids is None:
        if n > page_table.shape[0]:
            raise ValueError(f"{n} portions of {page_table.shape[0]} sequences")
    else:
        assert seq_ids.dtype == torch.int32 and seq_ids.is_contiguous() and seq_ids.numel() == n
    rc = _lib.on_device(bounds.device, _lib.lib().b200_page_bounds, ctypes.byref(cache.desc(page_table)), starts.data_ptr(), ends.data_ptr(), _lib.ptr(seq_ids),
                        n, int(max_tokens), bounds.data_ptr(), default_workspace(bounds.device).status.data_ptr())
    _lib.check(rc, "page_bounds")
    return bounds
