"""Attention over the pages of a long cache that look most promising, per row of queries and KV head."""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .attention import PagedKVCache
from .pages import check_bounds
from .workspace import default_workspace

MAX_HEAD_DIM = 512
MAX_ROWS = 65535
LIST_PER_CTA = 16384           # pages that a CTA may have to read


def pick_sparse_splits(pairs: int, pages: int, num_sms: int = 148, least: int = 16) -> int:
    """CTAs (one cluster of up to eight) per row and group of heads, which share ``pages`` pages: as many as still make one wave of one per SM, with
    ``least`` pages (16: two for a warp) each, and so many that their lists have room."""
    s = 1
    while s < 8 and ((pairs * s * 2 <= num_sms and pages // (2 * s) >= least) or pages > s * LIST_PER_CTA):
        s *= 2
    return s


def attn_paged_sparse(q: torch.Tensor, hq: int, positions: torch.Tensor, seq_ids: torch.Tensor | None, cache: PagedKVCache, page_table: torch.Tensor,
                      bounds: torch.Tensor, spec, out: torch.Tensor, *, top: int, first: int = 1, last: int = 2, seq_lens: torch.Tensor | None = None,
                      chosen: torch.Tensor | None = None, splits: int | None = None) -> torch.Tensor:
    """Rows of q (already rotated; [M, hq dk], row stride free) against the cached keys of their sequence, as ``attn_paged`` does it, but of every
    KV head only ``top`` pages: the ``first`` pages that the row sees, the ``last`` up to its own (which counts among them), and those others whose
    score is highest, the lower page first where scores are equal.  A page's score is the largest product that any query head of the group could
    have with a key within the page's ``bounds`` (``page_bounds``; those of the last pages are not read).  A row that sees no more than ``top``
    pages attends to all.

    ``chosen`` int32 [M, kv_heads, top]: receives the pages read (their place in the sequence, ascending, -1 behind them)."""
    M = positions.numel()
    if not (first >= 0 and last >= 1 and top >= first + last):
        raise ValueError(f"{top} pages with the first {first} and the last {last} among them")
    if not spec.scale > 0:
        raise ValueError("scores bound products with a positive scale")
    check_bounds(cache, bounds)
    assert q.dtype == cache.data.dtype == out.dtype and q.stride(1) == 1 and out.stride(1) == 1 and q.shape[0] == out.shape[0] == M
    assert q.shape[1] >= hq * cache.dk and out.shape[1] >= hq * cache.dv and hq % cache.kv_heads == 0
    assert positions.dtype == page_table.dtype == torch.int32 and page_table.is_contiguous() and positions.is_contiguous()
    for t in (seq_ids, seq_lens):
        assert t is None or (t.dtype == torch.int32 and t.is_contiguous() and t.numel() == M)
    if max(cache.dk, cache.dv) > MAX_HEAD_DIM or cache.dv == 0 or (hq // cache.kv_heads) * (cache.dk + 127 & ~127) > 50 << 10:
        raise ValueError(f"{hq} heads of {cache.dk} and {cache.dv} over {cache.kv_heads}")
    if M > MAX_ROWS or min(top, page_table.shape[1]) > 8 * LIST_PER_CTA:
        raise ValueError(f"{M} rows and {top} pages in one call")
    if seq_ids is None and M > page_table.shape[0]:
        raise ValueError(f"{M} rows of {page_table.shape[0]} sequences")
    if chosen is not None:
        assert chosen.dtype == torch.int32 and tuple(chosen.shape) == (M, cache.kv_heads, top) and chosen.is_contiguous()
    most = page_table.shape[1]
    if splits is None:
        seen = min(most, spec.chunk // cache.page_size + 2) if spec.chunk > 0 else most
        splits = pick_sparse_splits(M * cache.kv_heads * ((hq // cache.kv_heads + 15) // 16), min(top, seen), _lib.num_sms(q.device.index),
                                    16 if q.dtype == torch.bfloat16 else 4)
    scores = torch.empty(M * cache.kv_heads * most, dtype=torch.int32, device=q.device)
    rc = _lib.on_device(
        q.device, _lib.lib().b200_attn_paged_sparse, q.data_ptr(), q.stride(0), out.data_ptr(), out.stride(0), hq, M, positions.data_ptr(), _lib.ptr(seq_ids),
        _lib.ptr(seq_lens), ctypes.byref(cache.desc(page_table)), bounds.data_ptr(), ctypes.byref(spec), int(top), int(first), int(last), splits,
        scores.data_ptr(), _lib.ptr(chosen), default_workspace(q.device).status.data_ptr())
    _lib.check(rc, "attn_paged_sparse")
    _lib.LAUNCHES[0] += 1                        # two kernels
    return out
