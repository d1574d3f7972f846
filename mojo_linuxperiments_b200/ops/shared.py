"""Decode attention of sequences that share a prefix: the keys of the prefix are read once for all of them."""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .attention import PAGE, PagedKVCache
from .workspace import default_workspace


class SharedPrefixes:
    """Which sequence slots share the pages of their first tokens: groups of slots, each with a number of tokens (whole pages of 16).  A slot is in
    one group at most; one in none reads its keys alone.  Kept from step to step, like the page table."""

    def __init__(self, num_seqs: int, device):
        self.num_seqs, self.device = num_seqs, torch.device(device)
        self.groups: list[tuple[list[int], int]] = []

    def set(self, groups) -> None:
        """``groups``: (slots, tokens) each."""
        groups = [([int(s) for s in slots], int(tokens)) for slots, tokens in groups]
        every = [s for slots, _ in groups for s in slots]
        if len(set(every)) != len(every) or any(not 0 <= s < self.num_seqs for s in every):
            raise ValueError(f"slots {sorted(every)} of {self.num_seqs}")
        if any(tokens < 0 or tokens % PAGE for _, tokens in groups):
            raise ValueError(f"prefixes of {[t for _, t in groups]} tokens: whole pages of {PAGE} are shared")
        self.groups = [(slots, tokens) for slots, tokens in groups if slots and tokens]


def attn_decode_shared(q: torch.Tensor, hq: int, seq_lens: torch.Tensor, cache: PagedKVCache, page_table: torch.Tensor, shared: SharedPrefixes, spec,
                       out: torch.Tensor) -> torch.Tensor:
    """The last token of every slot (row b of q, already rotated, [B, hq dk], row stride free; its key is in the cache) against the first
    ``seq_lens[b]`` cached tokens of slot b.  Slots of a group of ``shared`` have the same pages in front; an empty slot (length 0) gets zeros."""
    B = seq_lens.numel()
    assert q.dtype == cache.data.dtype == out.dtype and q.stride(1) == 1 and out.stride(1) == 1 and q.shape[0] == out.shape[0] == B
    assert q.shape[1] >= hq * cache.dk and out.shape[1] >= hq * cache.dv and hq % cache.kv_heads == 0
    assert seq_lens.dtype == page_table.dtype == torch.int32 and page_table.is_contiguous() and seq_lens.is_contiguous()
    if B > page_table.shape[0] or B != shared.num_seqs:
        raise ValueError(f"{B} rows, {page_table.shape[0]} sequences, a plan for {shared.num_seqs}")
    with torch.cuda.device(q.device):
        rc = _lib.lib().b200_attn_paged(
            q.data_ptr(), q.stride(0), out.data_ptr(), out.stride(0), hq, B, None, None, seq_lens.data_ptr(), ctypes.byref(cache.desc(page_table)),
            ctypes.byref(spec), default_workspace(q.device).status.data_ptr(), _lib.stream())
    _lib.check(rc, "attn_decode_shared")
    return out
