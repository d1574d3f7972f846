"""Decode attention of sequences that share a prefix: the keys of the prefix are read once for all of them."""
from __future__ import annotations

import ctypes
from functools import lru_cache

import torch

from . import _lib
from .attention import PAGE, PagedKVCache, check_spec
from .pages import on_one_gpu
from .workspace import default_workspace

KEY_TILE = 128                 # keys of a step of the kernel
ROW_TILE = 128                 # rows (member x query head) of one of its two units
MAX_PARTS = 32                 # parts of a prefix
MAX_SPLITS = 8                 # CTAs of a cluster
_INFO, _PIECE = 16, 8          # where the numbers per slot start, numbers per piece
_ROWS, _KEYS, _ONE = 0, 1, 2   # two tiles of rows; one, and every other tile of keys for each unit; one unit


def room_for(num_seqs: int, per_head: int, kv_heads: int, ctas: int) -> tuple[int, int]:
    """Pieces, and rows of partial results per KV head, that a plan has room for: every prefix as one run, and two rounds of the CTAs beyond that."""
    more = -(-2 * ctas // kv_heads)
    return num_seqs * per_head // (2 * ROW_TILE) + num_seqs + more, 2 * num_seqs * per_head + 2 * ROW_TILE * more


def cut_prefixes(groups, num_seqs: int, per_head: int, kv_heads: int, ctas: int, others: int = 0, chunk: int = 0):
    """How the prefixes of ``groups`` (slots, tokens) are shared out: (four numbers per slot, pieces, slots in order, rows of partial results).

    A piece is up to 256 rows of a group and a run of tiles of 128 keys, for every KV head.  The two units of a CTA have 128 rows each, or, in a group of no
    more than 128, the same rows and every other tile.  Runs are as long as ends soonest: pieces of L steps take L + 4 (their start and end), ``ctas`` of
    them at a time, and ``others``, the CTAs of the slots' own keys, three of which fit where there is no piece, another 4 if some of
    them have to wait.  Where that is the same, fewer pieces if they wait and shorter runs if not (25 slots behind 1,657 tokens: 13.6 us in six, 14.9 in four).  With
    ``chunk`` only the keys from the last multiple of it are seen, and shared from the next page on.  A slot's numbers: first row of its partial results, rows between the parts, parts (none: it shares nothing), tokens."""
    info, pieces, order, base = [0] * (4 * num_seqs), [], [], 0
    begins = [-(-((tokens - 1) // chunk * chunk) // PAGE) * PAGE if chunk else 0 for _, tokens in groups]
    groups, begins = [g for g, a in zip(groups, begins) if a < g[1]], [a for (_, tokens), a in zip(groups, begins) if a < tokens]
    if not groups:
        return info, pieces, order, base
    sizes = [(len(slots) * per_head, -(-(tokens - begin) // KEY_TILE)) for (slots, tokens), begin in zip(groups, begins)]
    most = room_for(num_seqs, per_head, kv_heads, ctas)

    def shape(rows, tiles, steps):
        """mode, runs of keys of ``steps`` steps each at most, parts of the results"""
        if rows > ROW_TILE:
            runs = min(MAX_PARTS, -(-tiles // steps))
            return _ROWS, runs, runs
        runs = min(MAX_PARTS // 2, max(1, tiles // 2), -(-tiles // (2 * steps)))
        return (_ONE, 1, 1) if tiles == 1 else (_KEYS, runs, 2 * runs)

    def took(steps):
        longest = count = room = 0
        for rows, tiles in sizes:
            mode, runs, parts = shape(rows, tiles, steps)
            run = -(-tiles // runs)
            longest = max(longest, run if mode == _ROWS else -(-run // 2))
            count += -(-rows // (2 * ROW_TILE)) * runs
            room += rows * parts
        fits, count = count <= most[0] and room <= most[1], kv_heads * count
        wait = others > 3 * max(0, ctas - count)
        return not fits, -(-count // ctas) * (longest + 4) + 4 * wait, wait, count if wait else steps

    tried, at = [], max(tiles for _, tiles in sizes)       # one run each always fits
    while at >= 1:
        tried.append(at)
        at = min(at - 1, int(at / 1.06))
    steps = min(tried, key=took)
    for (slots, tokens), begin, (rows, tiles) in zip(groups, begins, sizes):
        mode, runs, parts = shape(rows, tiles, steps)
        for i, s in enumerate(slots):
            info[4 * s:4 * s + 4] = [base + i * per_head, rows, parts, tokens]
        for k in range(runs):
            a, b = begin + tiles * k // runs * KEY_TILE, min(tokens, begin + tiles * (k + 1) // runs * KEY_TILE)
            for row0 in range(0, rows, 2 * ROW_TILE):
                pieces.append([len(order), row0, min(2 * ROW_TILE, rows - row0), a, b, base + k * (parts // runs) * rows, slots[0], mode + 4 * rows])
        base += rows * parts
        order += slots
    return info, pieces, order, base


@lru_cache(maxsize=1024)
def pick_own_splits(pairs: int, keys: int, per_head: int, num_sms: int) -> int:
    """CTAs (one cluster) that share a slot's own keys, up to ``keys`` where it shares none, for a group of heads: as many as find a place at once with some left for the
    prefix, and at least 128 keys each.  Not by what slots share at the moment: a captured call keeps its clusters while groups change.
    Up to eight heads leave places for three CTAs per SM (80 pairs with up to 2,000 keys: 22.5 us in four, 29.2 in two; 60: 20.2 in four, 25.5
    in eight), more for two (34: 19.2 in four, 26.3 in eight).  16 slots with up to 150 keys take 8.9 us, 9.8 in two; 28 with up to 698 take 10.5 in four, 11.3 in eight."""
    s, most = 1, (4 * (3 if per_head <= 8 else 2) - 1) * num_sms // 4
    while s < MAX_SPLITS and pairs * 2 * s <= most and keys // (2 * s) >= KEY_TILE:
        s *= 2
    return s


class _Cut:
    """A plan as the kernels read it, for one number of heads and of CTAs that share a slot's own keys, and room for partial results."""

    def __init__(self, num_seqs: int, per_head: int, kv_heads: int, dv: int, chunk: int, splits: int, device: torch.device):
        self.per_head, self.kv_heads, self.chunk, self.splits, self.sms = per_head, kv_heads, chunk, splits, _lib.num_sms(device.index)
        self.max_pieces, self.rows = room_for(num_seqs, per_head, kv_heads, self.sms)
        self.pieces_at = (_INFO + 4 * num_seqs + 7) // 8 * 8
        self.slots_at = self.pieces_at + _PIECE * self.max_pieces
        n = self.slots_at + num_seqs
        self.plan = torch.zeros(n, dtype=torch.int32, device=device)
        self.part = torch.empty(kv_heads * self.rows * (dv + 2), dtype=torch.float32, device=device)
        # a ring: a copy still queued on the stream never sees an edit that belongs to a later step
        self.ring = [(buf, torch.cuda.Event()) for buf in torch.zeros(4, n, dtype=torch.int32, pin_memory=True)]
        self.turn = 0

    def send(self, groups, num_seqs: int) -> None:
        others = num_seqs * self.kv_heads * -(-self.per_head // 16) * self.splits
        info, pieces, order, rows = cut_prefixes(groups, num_seqs, self.per_head, self.kv_heads, self.sms, others, self.chunk)
        assert len(pieces) <= self.max_pieces and rows <= self.rows
        buf, done = self.ring[self.turn]
        self.turn = (self.turn + 1) % len(self.ring)
        done.synchronize()                       # its previous copy has left the buffer
        buf[0] = len(pieces)                     # the counters behind it are the kernels' own: zero between calls
        buf[_INFO:_INFO + 4 * num_seqs] = torch.tensor(info, dtype=torch.int32)
        if pieces:
            buf[self.pieces_at:self.pieces_at + _PIECE * len(pieces)] = torch.tensor(pieces, dtype=torch.int32).flatten()
            buf[self.slots_at:self.slots_at + len(order)] = torch.tensor(order, dtype=torch.int32)
        with torch.cuda.device(self.plan.device):
            self.plan.copy_(buf, non_blocking=True)
            done.record()


class SharedPrefixes:
    """Which sequence slots share the pages of their first tokens: groups of slots, each with a number of tokens (whole pages of 16).  A slot is in
    one group at most; one in none reads its keys alone.

    Kept from step to step, like the page table; ``set`` changes it between steps, also under captured calls, which follow it.  It holds the room for
    partial results as well: calls that may overlap on the GPU (different streams) use different objects, and an object is kept until the calls with it have ended."""

    def __init__(self, num_seqs: int, device):
        self.num_seqs, self.device = int(num_seqs), torch.device(device)
        self.groups: list[tuple[list[int], int]] = []
        self.longest = 0                          # tokens of the longest prefix
        self._cuts: dict[tuple, _Cut] = {}

    def set(self, groups) -> None:
        """``groups``: (slots, tokens) each.  Stream-ordered, like ``KVState.flush``, and not part of a captured call.  The pages of a prefix are read by the
        row that the group's first slot has in the page table: a group is set anew before that slot lets go of them."""
        groups = [([int(s) for s in slots], int(tokens)) for slots, tokens in groups]
        every = [s for slots, _ in groups for s in slots]
        if len(set(every)) != len(every) or any(not 0 <= s < self.num_seqs for s in every):
            raise ValueError(f"slots {sorted(every)} of {self.num_seqs}")
        if any(tokens < 0 or tokens % PAGE for _, tokens in groups):
            raise ValueError(f"prefixes of {[t for _, t in groups]} tokens: whole pages of {PAGE} are shared")
        if self._cuts and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("groups are set between captured calls, which follow them")
        self.groups = [(slots, tokens) for slots, tokens in groups if len(slots) > 1 and tokens]      # a slot alone shares nothing
        self.longest = max((t for _, t in self.groups), default=0)
        for cut in self._cuts.values():
            cut.send(self.groups, self.num_seqs)

    def nbytes(self) -> int:
        """Device bytes of what the calls so far have made: lists of pieces and room for partial results (128 slots, 32 heads of 128 over 8: 42 MiB)."""
        return sum(cut.plan.nbytes + cut.part.nbytes for cut in self._cuts.values())

    def cut_for(self, hq: int, cache: PagedKVCache, room: int, chunk: int = 0, splits: int | None = None) -> _Cut:
        device, per_head = cache.data.device, hq // cache.kv_heads
        if not splits:
            splits = pick_own_splits(self.num_seqs * cache.kv_heads * -(-per_head // 16), min(room, chunk) if chunk > 0 else room, per_head, _lib.num_sms(device.index))
        key = (hq, cache.kv_heads, cache.dv, chunk, splits, device.index)
        cut = self._cuts.get(key)
        if cut is None:
            if device != self.device and (device.type != self.device.type or self.device.index is not None):
                raise ValueError(f"a plan for {self.device} and a cache on {device}")
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("the first call with a plan sends it to the device: make one before the capture")
            cut = self._cuts[key] = _Cut(self.num_seqs, per_head, cache.kv_heads, cache.dv, chunk, splits, device)
            cut.send(self.groups, self.num_seqs)
        return cut


def reads_prefixes_once(cache: PagedKVCache) -> bool:
    """Whether the kernels of prefixes take the heads and pages of ``cache``; otherwise sharing changes nothing, and the decode kernel for one sequence is the better one."""
    return cache.data.dtype == torch.bfloat16 and cache.page_size == PAGE and cache.dk <= 128 and cache.dv <= 128 and (cache.dk | cache.dv) % 8 == 0


def attn_decode_shared(q: torch.Tensor, hq: int, seq_lens: torch.Tensor, cache: PagedKVCache, page_table: torch.Tensor, shared: SharedPrefixes, spec,
                       out: torch.Tensor, *, splits: int | None = None) -> torch.Tensor:
    """The last token of every slot (row b of q, already rotated, [B, hq dk], row stride free; its key is in the cache) against the first
    ``seq_lens[b]`` cached tokens of slot b.  Slots of a group of ``shared`` have the same pages in front, which are read once for all of them (bf16 heads of up
    to 128, pages of 16, a positive scale; otherwise every slot reads its own way through ``attn_paged``); a slot that does not see the prefix up to its
    end, being shorter or in a later chunk, reads alone.  An empty slot (length 0) gets zeros.

    ``splits``: CTAs that share a slot's own keys.  The first call for each number of them sends the plan to the device and is not part of a capture."""
    B, dk, dv, kv_heads, data = seq_lens.numel(), cache.dk, cache.dv, cache.kv_heads, cache.data
    (rows, width), (out_rows, out_width), (seqs, pages) = q.shape, out.shape, page_table.shape
    (ldq, q_step), (ldo, out_step), dtype, device = q.stride(), out.stride(), data.dtype, q.device
    assert q.dtype == dtype == out.dtype and q_step == 1 and out_step == 1 and rows == out_rows == B
    assert width >= hq * dk and out_width >= hq * dv and hq % kv_heads == 0
    assert seq_lens.dtype == page_table.dtype == torch.int32 and page_table.is_contiguous() and seq_lens.is_contiguous()
    room = pages * cache.page_size
    if splits and not 1 <= splits <= MAX_SPLITS:
        raise ValueError(f"{splits} CTAs in a cluster of up to {MAX_SPLITS}")
    if B > seqs or B != shared.num_seqs or shared.longest > room:
        raise ValueError(f"{B} rows, {seqs} sequences of up to {room} tokens, a plan for {shared.num_seqs} with prefixes of up to {shared.longest}")
    on_one_gpu(q, out, data, page_table, seq_lens)
    check_spec(spec, B, hq, q)
    L, desc, q_at, out_at, status = _lib.lib(), cache.desc(page_table), q.data_ptr(), out.data_ptr(), default_workspace(device).status.data_ptr()
    # (the kernels of prefixes take maxima before they scale)
    if not spec.scale > 0 or not reads_prefixes_once(cache) or ldq % 8 or ldo % 4 or q_at % 16 or out_at % 8 or data.data_ptr() % 16:
        rc = _lib.on_device(device, L.b200_attn_paged, q_at, ldq, out_at, ldo, hq, B, None, None, seq_lens.data_ptr(), ctypes.byref(desc), ctypes.byref(spec), status)
        _lib.check(rc, "attn_paged")
        return out
    cut = shared.cut_for(hq, cache, room, spec.chunk, splits)
    rc = _lib.on_device(
        device, L.b200_attn_decode_shared, q_at, ldq, out_at, ldo, hq, B, seq_lens.data_ptr(), ctypes.byref(desc),
        ctypes.byref(spec), cut.plan.data_ptr(), cut.pieces_at, cut.slots_at, cut.max_pieces, cut.part.data_ptr(), cut.rows, cut.splits, cut.sms,
        status)
    _lib.check(rc, "attn_decode_shared")
    _lib.LAUNCHES[0] += 1                        # two kernels
    return out
