"""Slots that share pages, on the host: forks, pages let go of, compaction, groups - against sequences kept as plain lists."""
import random

import pytest
import torch

from mojo_linuxperiments_b200.models.config import CacheSpec, RuntimeConfig
from mojo_linuxperiments_b200.models.kvcache import KVState


class Cfg:
    def __init__(self, chunks=(None, None), states=True):
        self.chunks, self.states = chunks, states

    def cache_layout(self, rt):
        return [CacheSpec(1, 8, 8, "float32", chunk=c) for c in self.chunks] + [None]

    def state_layout(self):
        return [{"x": 8}, {}, {"y": 16}] if self.states else []


class World:
    """A cache whose tokens are numbered, and what every slot should hold."""

    def __init__(self, cfg, slots, most, **rt):
        self.kv = KVState(cfg, RuntimeConfig(**rt), "cpu", slots, most)
        self.seqs: dict[int, list[int]] = {}
        self.next = 1

    def grow(self, slot, n):
        for _ in range(n):
            seq = self.seqs.setdefault(slot, [])
            pos = len(seq)
            self.kv.retire(slot, pos)
            self.kv.admit(slot, pos + 1)
            page = int(self.kv.table_host[slot, pos // 16])
            assert page != self.kv.scratch_page
            for c in self.kv.layers[:-1]:
                c.keys()[page, 0, pos % 16] = float(self.next)
                c.values()[page, 0, pos % 16] = -float(self.next)
            for run in self.kv.states:
                for t in run.values():
                    t[slot] = float(self.next)
            seq.append(self.next)
            self.next += 1

    def fork(self, slot, to):
        self.kv.fork(slot, to, len(self.seqs[slot]))
        for t in to:
            self.seqs[t] = list(self.seqs[slot])

    def release(self, slot):
        self.kv.release(slot)
        self.seqs.pop(slot, None)

    def check(self):
        kv = self.kv
        kv.flush()
        assert torch.equal(kv.page_table, kv.table_host)
        held: dict[int, int] = {}
        for slot, seq in self.seqs.items():
            for pos, token in enumerate(seq):
                if pos < kv.first_visible(len(seq) - 1) // 16 * 16:
                    continue                                   # may be given back
                page = int(kv.page_table[slot, pos // 16])
                for c in kv.layers[:-1]:
                    assert c.keys()[page, 0, pos % 16, 0] == token and c.values()[page, 0, pos % 16, 7] == -token
            for run in kv.states:
                for t in run.values():
                    assert (t[slot] == seq[-1]).all()
            for p in kv.owned[slot]:
                if p >= 0:
                    held[p] = held.get(p, 0) + 1
        assert kv._sharers == {p: n for p, n in held.items() if n > 1}
        assert sorted([*held, *kv.free_pages]) == list(range(kv.num_pages - 1)) and kv.pages_in_use() == len(held)
        for slots, tokens in kv.prefix_groups():
            rows = [kv.owned[s][:tokens // 16] for s in slots]
            assert len(slots) > 1 and tokens > 0 and all(r == rows[0] and len(r) == tokens // 16 for r in rows)


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("chunks", [(None, None), (48, None), (40, 24)])
def test_forks_growth_release_and_compaction_keep_every_sequence(seed, chunks):
    rng = random.Random(seed)
    w = World(Cfg(chunks), 6, 512, max_prefill_tokens=32, share_prefix=True)
    for _ in range(60):
        full = [s for s in w.seqs if w.seqs[s]]
        what = rng.choice(["grow", "grow", "grow", "fork", "fork", "release", "compact"])
        try:
            if what == "grow":
                slot = rng.randrange(6)
                w.grow(slot, min(rng.choice([1, 5, 16, 33, 70]), 500 - len(w.seqs.get(slot, []))))
            elif what == "fork" and full:
                slot = rng.choice(full)
                w.fork(slot, rng.sample([s for s in range(6) if s != slot], rng.randint(1, 3)))
            elif what == "release" and full:
                w.release(rng.choice(full))
            elif what == "compact":
                used = w.kv.pages_in_use()
                moved = w.kv.compact()
                assert moved <= used and all(p < used for pages in w.kv.owned.values() for p in pages)
        except RuntimeError as e:
            assert "exhausted" in str(e)
            break
        w.check()
        if w.kv.shared is not None:
            assert w.kv.shared.groups == w.kv.prefix_groups()
    for s in list(w.seqs):
        w.release(s)
    assert w.kv.pages_in_use() == 0 and not w.kv._sharers


def test_a_fork_shares_full_pages_and_copies_the_last():
    w = World(Cfg(states=False), 4, 256)
    w.grow(0, 40)
    before = w.kv.pages_in_use()
    w.fork(0, [1, 3])
    assert w.kv.pages_in_use() == before + 2
    assert w.kv.owned[1][:2] == w.kv.owned[0][:2] and len({w.kv.owned[s][2] for s in (0, 1, 3)}) == 3
    w.grow(1, 3), w.grow(0, 1)
    w.check()
    w.fork(1, [2])
    w.release(2)
    w.grow(2, 48)
    w.fork(2, [0])                                          # whole pages: nothing to copy
    assert w.kv.owned[0] == w.kv.owned[2]
    w.check()


def test_groups_save_most_reads():
    w = World(Cfg((None,), states=False), 7, 1024)
    w.grow(0, 64)
    w.fork(0, [1, 2, 3])
    assert w.kv.prefix_groups() == [([0, 1, 2, 3], 64)]
    w.grow(1, 160)
    w.fork(1, [4])
    # five share 4 pages (16 reads saved), two of them 14 (10 saved by themselves): apart 10 + 2 x 4 = 18
    assert sorted(w.kv.prefix_groups()) == [([0, 1, 2, 3, 4], 64)] or sorted(w.kv.prefix_groups()) == [([1, 4], 224)]
    saved = sum((len(s) - 1) * t // 16 for s, t in w.kv.prefix_groups())
    assert saved == max(4 * 4, 13)
    w.grow(1, 160)
    w.fork(1, [5, 6])
    saved = sum((len(s) - 1) * t // 16 for s, t in w.kv.prefix_groups())
    assert saved == max(6 * 4, 2 * 24)
    w.check()


def test_forks_that_cannot_be_are_refused_and_change_nothing():
    w = World(Cfg(), 3, 64, kv_pool_tokens=16)              # 7 pages
    w.grow(0, 20), w.grow(1, 33)
    for seq, to, n in ((0, [0], 20), (0, [1, 1], 20), (0, [3], 20), (0, [-1], 20), (0, [2], 0), (0, [2], 33), (2, [0], 1)):
        with pytest.raises(ValueError):
            w.kv.fork(seq, to, n)
    w.check()
    w.grow(2, 30)
    assert len(w.kv.free_pages) == 0
    held = {s: list(p) for s, p in w.kv.owned.items()}
    w.kv.fork(0, [2], 20)                                   # what slot 2 gives up is enough
    w.seqs[2] = list(w.seqs[0])
    w.check()
    assert held[0] == w.kv.owned[0] and held[1] == w.kv.owned[1]


def test_an_exhausted_pool_refuses_a_fork_before_anything_is_given_up():
    w = World(Cfg(), 3, 64, kv_pool_tokens=16)
    w.grow(0, 40), w.grow(1, 49)
    assert len(w.kv.free_pages) == 0
    with pytest.raises(RuntimeError, match="exhausted"):
        w.kv.fork(0, [2], 40)
    w.check()
    assert 2 not in w.kv.owned


def test_options_that_exclude_each_other():
    from mojo_linuxperiments_b200.engine.engine import Engine
    from mojo_linuxperiments_b200.models.layered_config import tiny_volonex
    for rt in (RuntimeConfig(share_prefix=True, sparse_pages=8), RuntimeConfig(sparse_pages=2), RuntimeConfig(sparse_pages=-1)):
        with pytest.raises(ValueError):
            Engine(tiny_volonex(), rt)


def test_bounds_are_kept_only_where_they_are_used():
    kv = KVState(Cfg(), RuntimeConfig(), "cpu", 2, 64)
    assert kv.bounds == [None, None, None]
    rt = RuntimeConfig(sparse_pages=8)
    kv = KVState(Cfg(), rt, "cpu", 2, 64)
    assert [b is not None for b in kv.bounds] == [True, True, False] and tuple(kv.bounds[0].shape) == (kv.num_pages, 1, 2, 8)
    assert KVState.nbytes(Cfg(), rt, 2, 64) >= KVState.nbytes(Cfg(), RuntimeConfig(), 2, 64) + sum(b.nbytes for b in kv.bounds[:2])
