"""Pages of a cache as such: records copied from page to page, bounds of the keys of a page."""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .attention import PagedKVCache
from .workspace import default_workspace


def copy_pages(caches, src, dst) -> None:
    """Record ``src[i]`` -> record ``dst[i]`` in every one of ``caches`` (a ``PagedKVCache``, a contiguous tensor of records along its first
    dimension, or a list of them: the layers of a model), in one launch per 64 of them.

    The page numbers are on the host, as those who hand pages out have them.  No page is written twice or read as well as written, so the
    order of the copies does not matter; a captured call copies the same pages in every replay."""
    arrays = [c.data if isinstance(c, PagedKVCache) else c for c in (caches if isinstance(caches, (list, tuple)) else [caches])]
    src, dst = [int(p) for p in src], [int(p) for p in dst]
    if len(src) != len(dst):
        raise ValueError(f"{len(src)} pages to copy to {len(dst)}")
    if not src or not arrays:
        return
    written = set(dst)
    if len(written) != len(dst) or not written.isdisjoint(src):
        raise ValueError("a page is written twice, or written and read")
    lo, hi = min(min(src), min(written)), max(max(src), max(written))
    device = arrays[0].device
    for a in arrays:
        if a.device != device or not a.is_cuda or not a.is_contiguous() or a.dim() < 2:
            raise ValueError("records lie in contiguous tensors on one GPU")
        if lo < 0 or hi >= a.shape[0]:
            raise IndexError(f"pages {lo} to {hi} of {a.shape[0]}")
    arrays = [a for a in arrays if a.numel() > 0]
    if not arrays:
        return
    sizes = [a.stride(0) * a.element_size() for a in arrays]
    if any(n % 16 or a.data_ptr() % 16 for n, a in zip(sizes, arrays)):
        raise ValueError("records are whole pieces of 16 bytes")
    n = len(src)
    with torch.cuda.device(device):
        rc = _lib.lib().b200_copy_pages((ctypes.c_void_p * len(arrays))(*[a.data_ptr() for a in arrays]), (ctypes.c_longlong * len(arrays))(*sizes),
                                        len(arrays), (ctypes.c_int * n)(*src), (ctypes.c_int * n)(*dst), n, _lib.stream())
    _lib.check(rc, "copy_pages")


def bounds_for(cache: PagedKVCache) -> torch.Tensor:
    """Room for the bounds of every page of ``cache``: [pages][kv_heads][2 (smallest, largest)][dk]."""
    return torch.zeros((cache.num_pages, cache.kv_heads, 2, cache.dk), dtype=cache.data.dtype, device=cache.data.device)


def check_bounds(cache: PagedKVCache, bounds: torch.Tensor) -> None:
    if tuple(bounds.shape) != (cache.num_pages, cache.kv_heads, 2, cache.dk) or bounds.dtype != cache.data.dtype or not bounds.is_contiguous() \
            or bounds.device != cache.data.device:
        raise ValueError(f"bounds {tuple(bounds.shape)} {bounds.dtype} of a cache of {cache.num_pages} pages, {cache.kv_heads} heads of {cache.dk}, {cache.data.dtype}")


def page_bounds(cache: PagedKVCache, page_table: torch.Tensor, starts: torch.Tensor, ends: torch.Tensor, seq_ids: torch.Tensor | None, max_tokens: int,
                bounds: torch.Tensor) -> torch.Tensor:
    """Smallest and largest element of the keys of a page, per KV head and dimension, for all pages that hold tokens ``starts[i]`` to
    ``ends[i] - 1`` (int32) of sequence ``seq_ids[i]`` (None: i); all tokens of such a page up to ``ends[i]`` count, nothing behind them is read.
    ``max_tokens``: the most that a portion has.  A portion of none, as of an empty slot, changes nothing.  Exact; NaN where a key is."""
    check_bounds(cache, bounds)
    n = starts.numel()
    assert starts.dtype == ends.dtype == page_table.dtype == torch.int32 and ends.numel() == n and all(t.is_contiguous() for t in (starts, ends, page_table))
    if seq_ids is None:
        if n > page_table.shape[0]:
            raise ValueError(f"{n} portions of {page_table.shape[0]} sequences")
    else:
        assert seq_ids.dtype == torch.int32 and seq_ids.is_contiguous() and seq_ids.numel() == n
    with torch.cuda.device(cache.data.device):
        rc = _lib.lib().b200_page_bounds(ctypes.byref(cache.desc(page_table)), starts.data_ptr(), ends.data_ptr(), _lib.ptr(seq_ids), n, int(max_tokens),
                                         bounds.data_ptr(), default_workspace(bounds.device).status.data_ptr(), _lib.stream())
    _lib.check(rc, "page_bounds")
    return bounds
