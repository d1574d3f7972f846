"""Paged KV cache of all layers of one rank plus the page table / lengths of the running batch.

Every model family describes what its layers store (``cfg.cache_layout``: heads, key and value sizes, element type, how
far back a position looks); pages of 16 tokens (``rt.page_size``) are handed out per sequence and shared by all layers,
i.e. page *p* of a sequence is record *p* of every layer's storage.  Layers that look back only to the start of their
own chunk let go of older tokens: when no layer can see a page any more it returns to the free list (``retire``).

Sequences may share pages: ``fork`` gives a slot the full pages of another one's tokens and a copy of the last, partly filled page, so that
nobody ever writes a page that somebody else reads; a page returns to the free list when the last slot lets go of it.  ``compact`` moves the pages in use to the
front of the pool.

Beside the pages every sequence slot has a fixed-size fp32 state per layer (``cfg.state_layout``: the previous token's row
of a token shift, the state of a recurrence).  Kernels take a sequence's state as zero at position 0, so a slot needs no
clearing between sequences, and change it only where ``active`` says that the slot takes part in the step."""
from __future__ import annotations

import torch

from ..ops import attention as A
from ..ops import pages as P
from ..ops.shared import SharedPrefixes
from .config import CacheSpec, ModelConfig, RuntimeConfig

_DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def _record(s: CacheSpec | None, page_size: int) -> int:
    return s.kv_heads * page_size * (s.dk + s.dv) if s is not None else 0


def _states(cfg) -> list[dict[str, int]]:
    return cfg.state_layout() if hasattr(cfg, "state_layout") else []


class KVState:
    @staticmethod
    def pool_pages(cfg, rt: RuntimeConfig, num_seqs: int, max_seq_len: int) -> int:
        """Pages the free list starts with: what the slots can hold at once, unless ``rt.kv_pool_tokens`` says less."""
        ps = rt.page_size
        per_seq = (max_seq_len + ps - 1) // ps
        chunks = [s.chunk for s in cfg.cache_layout(rt) if s is not None]
        if all(chunks):
            # what lies before the oldest visible chunk is given back between portions of a prompt
            per_seq = min(per_seq, (max(chunks, default=0) + rt.max_prefill_tokens + ps - 1) // ps + 2)
        total = num_seqs * per_seq
        if rt.kv_pool_tokens > 0:
            total = min(total, (rt.kv_pool_tokens + ps - 1) // ps + 2 * num_seqs)
        return total

    @staticmethod
    def nbytes(cfg, rt: RuntimeConfig, num_seqs: int, max_seq_len: int) -> int:
        """Device bytes of a cache for ``num_seqs`` sequences of up to ``max_seq_len`` tokens (storage + tables)."""
        max_pages = (max_seq_len + rt.page_size - 1) // rt.page_size
        pages = KVState.pool_pages(cfg, rt, num_seqs, max_seq_len) + 1
        layout = cfg.cache_layout(rt)
        size = max((_DTYPES[s.dtype].itemsize for s in layout if s is not None), default=0)
        states = sum(n for run in _states(cfg) for n in run.values()) * num_seqs * 4
        bounds = sum(2 * s.kv_heads * s.dk for s in layout if s is not None and s.dv > 0) * pages * size + 1024 * len(layout) if rt.sparse_pages > 0 else 0
        return sum(_record(s, rt.page_size) for s in layout) * pages * size + bounds + states + num_seqs * max_pages * 4 + num_seqs * 8 + 3 * 1024

    def __init__(self, cfg: ModelConfig, rt: RuntimeConfig, device, num_seqs: int, max_seq_len: int, alloc=None):
        """``alloc(shape, dtype) -> zeroed tensor``: where the cache lives (the rank's HBM arena); default torch.zeros.

        Pages are handed out on demand (``admit`` as a sequence grows) from a host-side free list.  The last page is
        a scratch page no sequence owns: the page-table rows of empty slots point at it, so a kernel that runs over
        an empty slot of the batch has somewhere harmless to write."""
        if alloc is None:
            def alloc(shape, dtype):
                return torch.zeros(shape, dtype=dtype, device=device)
        self.page_size = rt.page_size
        self.num_seqs = num_seqs
        self.max_pages = (max_seq_len + rt.page_size - 1) // rt.page_size
        self.num_pages = self.pool_pages(cfg, rt, num_seqs, max_seq_len) + 1
        self.scratch_page = self.num_pages - 1
        self.layout = cfg.cache_layout(rt)
        assert len({s.dtype for s in self.layout if s is not None}) <= 1
        sizes = [_record(s, rt.page_size) * self.num_pages for s in self.layout]
        dtype = next((s.dtype for s in self.layout if s is not None), rt.dtype)
        self.storage = alloc((max(1, sum(sizes)),), _DTYPES[dtype])
        self.layers, at = [], 0
        for s, n in zip(self.layout, sizes):
            self.layers.append(A.PagedKVCache(self.num_pages, s.kv_heads, rt.page_size, device, storage=self.storage[at:at + n],
                                              dk=s.dk, dv=s.dv) if s is not None else None)
            at += n
        # smallest and largest keys of every page, where decoding selects pages by them (latents have no values beside their keys)
        self.bounds: list[torch.Tensor | None] = [None] * len(self.layers)
        if rt.sparse_pages > 0:
            self.bounds = [alloc((self.num_pages, c.kv_heads, 2, c.dk), c.data.dtype) if c is not None and c.dv > 0 else None for c in self.layers]
        # [sequence][numbers] per run and name; the numbers of a run are multiples of eight
        self.states: list[dict[str, torch.Tensor]] = []
        layout = _states(cfg)
        flat, at = alloc((max(1, sum(n for run in layout for n in run.values()) * num_seqs),), torch.float32), 0
        for run in layout:
            self.states.append({})
            for name, n in run.items():
                self.states[-1][name] = flat[at:at + n * num_seqs].view(num_seqs, n)
                at += n * num_seqs
        self.active = alloc((num_seqs,), torch.int32)         # 1: the slot takes part in the next decode step
        self.page_table = alloc((num_seqs, self.max_pages), torch.int32)
        self.seq_lens = alloc((num_seqs,), torch.int32)
        self.free_pages = list(range(self.num_pages - 2, -1, -1))
        self.owned: dict[int, list[int]] = {}       # page ids of a slot in token order; -1: given back by ``retire``
        self._sharers: dict[int, int] = {}          # slots that hold a page, where these are more than one
        self.shared = SharedPrefixes(num_seqs, device) if rt.share_prefix else None
        self._regroup = False                       # ``shared`` has to be looked at again
        self._periods = {self.page_size, *(s.chunk for s in self.layout if s is not None and s.chunk)}
        self._retired: dict[int, int] = {}          # leading entries of ``owned`` that are -1
        # host mirror of the page table: rows are edited here; ``flush`` sends a snapshot (a ring of pinned buffers, so
        # that a copy still queued on the stream never sees an edit that belongs to a later step)
        self.table_host = torch.full((num_seqs, self.max_pages), self.scratch_page, dtype=torch.int32)
        self._table = self.table_host.numpy()       # the same memory
        self._cuda = torch.cuda.is_available() and torch.device(device).type == "cuda"
        self._ring = [(self.table_host.clone().pin_memory(), torch.cuda.Event()) for _ in range(4)] if self._cuda else []
        self._turn = 0
        self._dirty = True
        self.pages_high_water = 0

    def admit(self, seq: int, n_tokens: int) -> None:
        """Make sure sequence slot ``seq`` owns pages for ``n_tokens`` tokens (grows, never shrinks)."""
        need = (n_tokens + self.page_size - 1) // self.page_size
        if need > self.max_pages:
            raise RuntimeError(f"{n_tokens} tokens exceed the {self.max_pages * self.page_size} a page-table row can describe")
        have = self.owned.setdefault(seq, [])
        if need - len(have) > len(self.free_pages):
            raise RuntimeError("KV cache exhausted")
        if len(have) < need:
            # one slice per call: an element of a tensor costs microseconds to set, and a batch of prompts takes thousands of pages
            new = self.free_pages[len(have) - need:][::-1]
            del self.free_pages[len(have) - need:]
            self._table[seq, len(have):need] = new
            have += new
            self._dirty = True
        self.pages_high_water = max(self.pages_high_water, self.num_pages - 1 - len(self.free_pages))

    def first_visible(self, pos: int) -> int:
        """Oldest position that some layer of a token at ``pos`` (or any later one) can still see."""
        return min(((pos - pos % s.chunk) if s.chunk else 0 for s in self.layout if s is not None), default=pos)

    def next_change(self, pos: int) -> int:
        """First position after ``pos`` at which a growing sequence needs another page or stops seeing one."""
        return min((pos // n + 1) * n for n in self._periods)

    def retire(self, seq: int, pos: int) -> None:
        """The next token of slot ``seq`` goes to position ``pos``: pages that lie wholly before everything it can see
        return to the free list."""
        pages = self.owned.get(seq)
        if not pages:
            return
        n0, n1 = self._retired.get(seq, 0), min(self.first_visible(pos) // self.page_size, len(pages))
        for i in range(n0, n1):
            self._let_go(pages[i])
            pages[i] = -1
        if n1 > n0:
            self._table[seq, n0:n1] = self.scratch_page
            self._retired[seq] = n1
            self._dirty = True

    def _let_go(self, page: int) -> None:
        n = self._sharers.get(page, 1)
        if n == 1:
            self.free_pages.append(page)
            return
        self._regroup = True
        if n == 2:
            del self._sharers[page]
        else:
            self._sharers[page] = n - 1

    def release(self, seq: int) -> None:
        """Give the pages of slot ``seq`` back; its page-table row points at the scratch page again."""
        pages = self.owned.pop(seq, [])
        self._retired.pop(seq, None)
        if pages:
            for p in reversed(pages):
                if p >= 0:
                    self._let_go(p)
            self._table[seq] = self.scratch_page
            self._dirty = True

    def _copy_pages(self, arrays, src: list[int], dst: list[int]) -> None:
        if self._cuda:
            P.copy_pages(arrays, src, dst)
            return
        for a in arrays:
            a[dst] = a[src]

    def _records(self) -> list[torch.Tensor]:
        """Everything that a page has a record in."""
        return [c.data for c in self.layers if c is not None] + [b for b in self.bounds if b is not None]

    def fork(self, seq: int, to: list[int], n_tokens: int) -> None:
        """The slots ``to``, whose own sequences are given up, hold the first ``n_tokens`` tokens of slot ``seq`` too: its full pages are shared, the
        last one, if it is not full, is copied, and so are the slot's states.  Stream-ordered; the page table follows with ``flush``."""
        pages = self.owned.get(seq, [])
        full, rest = divmod(n_tokens, self.page_size)
        if seq in to or len(set(to)) != len(to) or any(not 0 <= t < self.num_seqs for t in to):
            raise ValueError(f"slot {seq} to {to} of {self.num_seqs}")
        if not 0 < n_tokens <= len(pages) * self.page_size:
            raise ValueError(f"{n_tokens} tokens of a slot with pages for {len(pages) * self.page_size}")
        if rest:
            given: dict[int, int] = {}
            for t in to:
                for p in self.owned.get(t, []):
                    given[p] = given.get(p, 0) + 1
            freed = sum(p >= 0 and n == self._sharers.get(p, 1) for p, n in given.items())
            if len(to) > len(self.free_pages) + freed:
                raise RuntimeError("KV cache exhausted")
        for t in to:
            self.release(t)
        copied = []
        for t in to:
            mine = pages[:full]
            for p in mine:
                if p >= 0:
                    self._sharers[p] = self._sharers.get(p, 1) + 1
            if rest and pages[full] >= 0:
                copied.append(self.free_pages.pop())
                mine = mine + [copied[-1]]
            elif rest:
                mine = mine + [-1]
            self.owned[t] = mine
            self._table[t, :len(mine)] = [p if p >= 0 else self.scratch_page for p in mine]
            self._retired[t] = min(self._retired.get(seq, 0), len(mine))
        self._dirty = self._regroup = True
        if copied:
            self._copy_pages(self._records(), [pages[full]] * len(copied), copied)
        states = [t for run in self.states for t in run.values()]
        if states:
            self._copy_pages(states, [seq] * len(to), list(to))
        self.pages_high_water = max(self.pages_high_water, self.num_pages - 1 - len(self.free_pages))

    def compact(self) -> int:
        """Move pages so that those in use are the first of the pool; how many were moved."""
        used = {p for pages in self.owned.values() for p in pages if p >= 0}
        n = len(used)
        high, holes = sorted(p for p in used if p >= n), sorted(set(range(n)) - used)
        if not high:
            return 0
        to = dict(zip(high, holes))
        self._copy_pages(self._records(), high, holes)
        for seq, pages in self.owned.items():
            self.owned[seq] = [to.get(p, p) for p in pages]
            self._table[seq, :len(pages)] = [p if p >= 0 else self.scratch_page for p in self.owned[seq]]
        self._sharers = {to.get(p, p): k for p, k in self._sharers.items()}
        self.free_pages = list(range(self.num_pages - 2, n - 1, -1))
        self._dirty = True
        return len(high)

    def prefix_groups(self) -> list[tuple[list[int], int]]:
        """(slots, tokens) of groups of slots with the same pages in front, such that as many reads of pages as possible fall away."""
        def common(slots: list[int], at: int) -> int:
            end = min(len(self.owned[s]) for s in slots)
            rows = self._table[slots, at:end]
            differ = (rows != rows[0]).any(0)
            return at + (int(differ.argmax()) if differ.any() else end - at)

        def best(slots: list[int], at: int, real: int):
            """saved reads and groups, for slots with the same first ``at`` pages, ``real`` of which are there"""
            end = common(slots, at)
            real += int((self._table[slots[0], at:end] != self.scratch_page).sum())
            parts: dict[int, list[int]] = {}
            for s in slots:
                if len(self.owned[s]) > end:
                    parts.setdefault(int(self._table[s, end]), []).append(s)
            saved, groups = 0, []
            for page, members in parts.items():
                if len(members) > 1:
                    n, g = best(members, end, real)
                    saved, groups = saved + n, groups + g
            whole = (len(slots) - 1) * real
            return (saved, groups) if saved > whole else (whole, [(slots, end * self.page_size)] if whole else [])

        slots = sorted(s for s, pages in self.owned.items() if pages)
        return best(slots, 0, 0)[1] if self._sharers and len(slots) > 1 else []

    def flush(self) -> None:
        """Copy the page table to the device if a row changed since the last flush (asynchronous, stream-ordered)."""
        if self._regroup:
            self._regroup = False
            if self.shared is not None:
                # (a plan counts in pages of 16 tokens, whatever the pages of the pool have)
                groups = [(slots, t // A.PAGE * A.PAGE) for slots, t in self.prefix_groups() if t >= A.PAGE]
                if groups != self.shared.groups:
                    self.shared.set(groups)
        if not self._dirty:
            return
        if self._cuda:
            buf, done = self._ring[self._turn]
            self._turn = (self._turn + 1) % len(self._ring)
            done.synchronize()                       # its previous copy has left the buffer
            buf.copy_(self.table_host)
            self.page_table.copy_(buf, non_blocking=True)
            done.record()
        else:
            self.page_table.copy_(self.table_host)
        self._dirty = False

    def note_keys(self, run: int, starts: torch.Tensor, ends: torch.Tensor, seq_ids: torch.Tensor | None, max_tokens: int) -> None:
        """Keys ``starts[i]`` to ``ends[i] - 1`` of the sequences have been written in layer ``run``: the bounds of their pages, where these are kept."""
        if self.bounds[run] is not None:
            P.page_bounds(self.layers[run], self.page_table, starts, ends, seq_ids, max_tokens, self.bounds[run])

    def pages_in_use(self) -> int:
        return self.num_pages - 1 - len(self.free_pages)
