"""Attention over the pages of a long cache that look most promising, per row of queries and KV head."""
from __future__ import annotations

import ctypes
from functools import lru_cache

import torch

from . import _lib
from .attention import PagedKVCache, check_spec
from .pages import check_bounds, on_one_gpu
from .workspace import default_workspace

MAX_HEAD_DIM = 512
MAX_ROWS = 65535
MAX_QUERIES = 50 << 10         # numbers of a group's queries, heads padded to 128, that shared memory holds
LIST_PER_CTA = 16384           # pages that a CTA may have to read


@lru_cache(maxsize=None)
def clusters_at_once(device_index: int) -> dict[int, int]:
    """Clusters of 2, 4 and 8 CTAs, one per SM, that run at once."""
    with torch.cuda.device(device_index):
        return {s: _lib.lib().b200_sparse_clusters(s) or _lib.num_sms(device_index) // (2 * s) for s in (2, 4, 8)}


def pick_sparse_splits(pairs: int, pages: int, at_once: dict[int, int]) -> int:
    """CTAs (one cluster of up to eight) per row and group of heads, which share ``pages`` pages: as many as still run at once (16 clusters of eight, of which 15 do,
    take 21.4 us where clusters of four take 14.6), with four pages each (one row, 64 pages, 8 KV heads: 12.2 us in eight, 13.2 in four; 16 pages, one KV head:
    11.1 in four, 12.5 in one), and so many that their lists have room."""
    s = 1
    while s < 8 and ((pairs <= at_once[2 * s] and pages // (2 * s) >= 4) or pages > s * LIST_PER_CTA):
        s *= 2
    return s


def attn_paged_sparse(q: torch.Tensor, hq: int, positions: torch.Tensor, seq_ids: torch.Tensor | None, cache: PagedKVCache, page_table: torch.Tensor,
                      bounds: torch.Tensor, spec, out: torch.Tensor, *, top: int, first: int = 1, last: int = 2, seq_lens: torch.Tensor | None = None,
                      chosen: torch.Tensor | None = None, splits: int | None = None) -> torch.Tensor:
    """Rows of q (already rotated; [M, hq dk], row stride free) against the cached keys of their sequence, as ``attn_paged`` does it, but of every
    KV head only ``top`` pages: the ``first`` pages that the row sees, the ``last`` up to its own (which counts among them), and those others whose
    score is highest, the lower page first where scores are equal.  A page's score is the largest product that any query head of the group could
    have with a key within the page's ``bounds`` (``page_bounds``; those of the last pages are not read); where these are not finite it counts as the
    highest.  A row that sees no more than ``top`` pages attends to all.

    ``chosen`` int32 [M, kv_heads, top]: receives the pages read (their place in the sequence, ascending, -1 behind them)."""
    M = positions.numel()
    if not (first >= 0 and last >= 1 and top >= first + last):
        raise ValueError(f"{top} pages with the first {first} and the last {last} among them")
    if not spec.scale > 0:
        raise ValueError("scores bound products with a positive scale")
    check_bounds(cache, bounds)
    dk, dv, kv_heads, dtype, device = cache.dk, cache.dv, cache.kv_heads, cache.data.dtype, q.device
    (rows, width), (out_rows, out_width), (seqs, most) = q.shape, out.shape, page_table.shape
    (ldq, q_step), (ldo, out_step) = q.stride(), out.stride()
    assert q.dtype == dtype == out.dtype and q_step == 1 and out_step == 1 and rows == out_rows == M
    assert width >= hq * dk and out_width >= hq * dv and hq % kv_heads == 0
    assert positions.dtype == page_table.dtype == torch.int32 and page_table.is_contiguous() and positions.is_contiguous()
    for t in (seq_ids, seq_lens):
        assert t is None or (t.dtype == torch.int32 and t.is_contiguous() and t.numel() == M)
    group = hq // kv_heads
    if dk > MAX_HEAD_DIM or dv > MAX_HEAD_DIM or dv == 0 or group * (dk + 127 & ~127) > MAX_QUERIES:
        raise ValueError(f"{hq} heads of {dk} and {dv} over {kv_heads}")
    read = min(top, most, spec.chunk // cache.page_size + 2 if spec.chunk > 0 else most)      # pages of a row at most
    if M > MAX_ROWS or read > 8 * LIST_PER_CTA:
        raise ValueError(f"{M} rows and {top} pages in one call")
    if seq_ids is None and M > seqs:
        raise ValueError(f"{M} rows of {seqs} sequences")
    on_one_gpu(q, out, bounds, page_table, positions, seq_ids, seq_lens, chosen)
    check_spec(spec, M, hq, q)
    if chosen is not None:
        assert chosen.dtype == torch.int32 and tuple(chosen.shape) == (M, kv_heads, top) and chosen.is_contiguous()
    if splits is None:
        splits = pick_sparse_splits(M * kv_heads * ((group + 15) // 16), read, clusters_at_once(device.index))
    scores = torch.empty(M * kv_heads * most, dtype=torch.int32, device=device)
    rc = _lib.on_device(
        device, _lib.lib().b200_attn_paged_sparse, q.data_ptr(), ldq, out.data_ptr(), ldo, hq, M, positions.data_ptr(), _lib.ptr(seq_ids),
        _lib.ptr(seq_lens), ctypes.byref(cache.desc(page_table)), bounds.data_ptr(), ctypes.byref(spec), int(top), int(first), int(last), splits,
        scores.data_ptr(), _lib.ptr(chosen), default_workspace(device).status.data_ptr())
    _lib.check(rc, "attn_paged_sparse")
    _lib.LAUNCHES[0] += 1                        # two kernels
    return out
