"""What copies of pages, their bounds and the attentions that select or share them refuse, before anything is launched."""
from types import SimpleNamespace

import pytest
import torch

from mojo_linuxperiments_b200.ops import attention as A
from mojo_linuxperiments_b200.ops import pages as PG
from mojo_linuxperiments_b200.ops import shared as SH
from mojo_linuxperiments_b200.ops import sparse as SP


@pytest.mark.parametrize("src,dst,error", [([0], [1, 2], ValueError), ([0, 1], [2, 2], ValueError), ([0, 1], [1, 2], ValueError), ([3], [3], ValueError)])
def test_copies_that_depend_on_their_order_are_refused(src, dst, error):
    with pytest.raises(error):
        PG.copy_pages(torch.zeros(4, 8), src, dst)


def test_copies_of_nothing_and_of_tensors_elsewhere():
    PG.copy_pages(torch.zeros(4, 8), [], [])
    PG.copy_pages([], [1], [2])
    with pytest.raises(ValueError):
        PG.copy_pages(torch.zeros(4, 8), [0], [1])          # not on a GPU


def _cache(dtype=torch.bfloat16, dk=32, dv=16):
    return A.PagedKVCache(6, 2, 16, "cpu", dk=dk, dv=dv, dtype=dtype)


def test_bounds_have_the_shape_and_type_of_the_keys():
    c = _cache()
    b = PG.bounds_for(c)
    assert tuple(b.shape) == (6, 2, 2, 32) and b.dtype == torch.bfloat16
    for bad in (b.float(), b[:5], b.transpose(2, 3), b[:, :1]):
        with pytest.raises(ValueError):
            PG.check_bounds(c, bad)


def _sparse(**kw):
    c = kw.pop("cache", _cache())
    q, out = torch.zeros(3, 4 * c.dk, dtype=c.data.dtype), torch.zeros(3, 4 * c.dv, dtype=c.data.dtype)
    args = dict(top=8, first=1, last=2)
    args.update(kw)
    scale, table = args.pop("scale", 0.1), args.pop("table", torch.zeros(3, 40, dtype=torch.int32))
    return SP.attn_paged_sparse(q, 4, torch.zeros(3, dtype=torch.int32), None, c, table, args.pop("bounds", PG.bounds_for(c)), A.attn_spec(scale), out, **args)


@pytest.mark.parametrize("kw", [dict(top=2), dict(last=0), dict(first=-1), dict(scale=0.0), dict(scale=-1.0), dict(table=torch.zeros(2, 40, dtype=torch.int32)),
                                dict(cache=_cache(dk=520)), dict(cache=_cache(dv=0)), dict(top=140000, table=torch.zeros(3, 150000, dtype=torch.int32)), dict(bounds=torch.zeros(6, 2, 2, 32))])
def test_selections_that_make_no_sense_are_refused(kw):
    with pytest.raises(ValueError):
        _sparse(**kw)


@pytest.mark.parametrize("groups", [[([0, 0], 16)], [([0, 1], 16), ([1, 2], 32)], [([0, 4], 16)], [([0, -1], 16)], [([0, 1], 20)], [([0, 1], -16)]])
def test_groups_that_make_no_sense_are_refused(groups):
    with pytest.raises(ValueError):
        SH.SharedPrefixes(4, "cpu").set(groups)


@pytest.mark.parametrize("pairs,pages,want", [(8, 128, 8), (15, 128, 8), (16, 128, 4), (33, 64, 4), (34, 64, 2), (74, 64, 2), (75, 64, 1), (2, 31, 4), (1, 32, 8), (3, 7, 1), (4000, 65536, 4), (300, 16384, 1)])
def test_clusters_for_selections(pairs, pages, want):
    assert SP.pick_sparse_splits(pairs, pages, {2: 74, 4: 33, 8: 15}) == want


@pytest.mark.parametrize("pairs,keys,per_head,want", [(1, 100, 4, 1), (16, 150, 4, 1), (28, 698, 8, 4), (80, 2000, 4, 4), (80, 2000, 16, 2), (74, 2000, 9, 2), (64, 2000, 16, 4), (34, 2000, 16, 4), (60, 2000, 4, 4),
                                                      (50, 2000, 4, 8), (1024, 1000, 4, 1), (4, -100, 4, 1)])
def test_clusters_for_own_keys(pairs, keys, per_head, want):
    assert SH.pick_own_splits(pairs, keys, per_head, 148) == want


@pytest.mark.parametrize("per_head,kv_heads,groups", [
    (4, 8, [(list(range(32)), 2048)]), (4, 8, [(list(range(128)), 32768)]), (20, 1, [([3, 1, 2], 16), ([0, 7], 160), ([5], 4096)]),
    (160, 1, [([1, 0, 2], 272)]), (1, 1, [(list(range(200)), 16)]), (7, 3, [([i, 199 - i], 16 * (1 + i)) for i in range(90)]), (4, 8, []),
    (16, 4, [(list(range(i, 200, 16)), 16 * (300 + 7 * i)) for i in range(16)]), (4, 8, [([i], 16) for i in range(200)]), (4, 1, [([7, 9], 16 * 60000)])])
def test_pieces_of_prefixes_cover_every_row_and_key_once(per_head, kv_heads, groups):
    n, ctas = 200, 148
    info, pieces, order, rows = SH.cut_prefixes(groups, n, per_head, kv_heads, ctas)
    room = SH.room_for(n, per_head, kv_heads, ctas)
    assert len(pieces) <= room[0] and rows <= room[1] and len(order) <= n
    size = {slots[0]: (len(slots) * per_head, tokens) for slots, tokens in groups}
    seen, used = {}, set()
    for member0, row0, count, key0, key1, part, lead, mode in pieces:
        group_rows, tokens = size[lead]
        assert mode >> 2 == group_rows
        mode &= 3
        assert order[member0] == lead and 0 < count <= 256 and row0 + count <= group_rows and key0 % 128 == 0 and key0 < key1 <= tokens
        tiles = list(range(key0, key1, 128))
        assert count <= 128 or mode == 0
        assert len(tiles) > 1 or mode != 1
        for unit in range(2 if mode == 1 else 1):
            for r in range(row0, row0 + count):
                slot, head = order[member0 + r // per_head], r % per_head
                at = part + unit * group_rows + r
                assert at not in used
                used.add(at)
                seen.setdefault((slot, head), []).append((tiles[unit::2] if mode == 1 else tiles, at))
    assert all(0 <= u < rows for u in used)
    for slots, tokens in groups:
        for s in slots:
            first, step, parts, t = info[4 * s:4 * s + 4]
            assert t == tokens and 0 < parts <= SH.MAX_PARTS
            for h in range(per_head):
                runs = seen.pop((s, h))
                assert sorted(k for tiles, _ in runs for k in tiles) == list(range(0, tokens, 128))
                assert sorted(at for _, at in runs) == [first + h + k * step for k in range(parts)]
    assert not seen and all(info[4 * s + 2] == 0 for s in range(n) if s not in set(order))


@pytest.mark.parametrize("chunk", [1, 16, 50, 128, 300, 4096])
def test_pieces_begin_where_the_chunk_of_a_prefix_does(chunk):
    """From the first page behind the last multiple of the chunk: what every slot sees that is as long and whose own chunk begins in front of the prefix's end."""
    groups = [([2 * i, 2 * i + 1], 16 * (1 + 3 * i)) for i in range(20)]
    info, pieces, order, rows = SH.cut_prefixes(groups, 40, 4, 2, 148, 0, chunk)
    for slots, tokens in groups:
        begin = min(tokens, -(-((tokens - 1) // chunk * chunk) // 16) * 16)
        mine = sorted((p[3], p[4]) for p in pieces if p[6] == slots[0])
        assert all(info[4 * s + 2] == 0 for s in slots) if begin == tokens else all(info[4 * s + 3] == tokens for s in slots)
        assert [a for a, _ in mine] + [tokens] == [begin] + [b for _, b in mine]
        for n in range(tokens, tokens + 2 * chunk, max(1, chunk // 7)):
            low = (n - 1) - (n - 1) % chunk
            assert low >= tokens or begin - 16 < low <= begin


class _OnGpu(torch.Tensor):
    """A tensor that says it is on the GPU"""

    def get_device(self):
        return 0


def _gpu(t):
    return t.as_subclass(_OnGpu)


@pytest.fixture
def launches(monkeypatch):
    """Stands in for the library: what would have been launched"""
    calls = []
    for m in (PG, SP, SH):
        monkeypatch.setattr(m._lib, "lib", lambda: SimpleNamespace(b200_page_bounds="page_bounds", b200_attn_paged_sparse="attn_paged_sparse"))
        monkeypatch.setattr(m._lib, "on_device", lambda device, fn, *args: calls.append((fn, args)) or 0)
        monkeypatch.setattr(m, "default_workspace", lambda device: SimpleNamespace(status=torch.zeros(4, dtype=torch.int32)))
    return calls


def _i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


@pytest.mark.parametrize("host", ["all", "bounds", "page_table", "starts", "ends", "seq_ids", None])
def test_bounds_of_tensors_on_the_host_are_refused(host, launches):
    c = _cache()
    t = {"page_table": _i32(3, 2), "starts": _i32(3), "ends": _i32(3), "seq_ids": _i32(3), "bounds": PG.bounds_for(c)}
    c.data = c.data if host == "all" else _gpu(c.data)
    t = {k: x if host in ("all", k) else _gpu(x) for k, x in t.items()}
    if host is None:
        PG.page_bounds(c, t["page_table"], t["starts"], t["ends"], t["seq_ids"], 1, t["bounds"])
        assert len(launches) == 1
        return
    with pytest.raises(ValueError):
        PG.page_bounds(c, t["page_table"], t["starts"], t["ends"], t["seq_ids"], 1, t["bounds"])
    assert not launches


@pytest.mark.parametrize("host", ["q", "page_table", "positions", "seq_ids", "seq_lens", "chosen", "out", None])
def test_selections_by_tensors_on_the_host_are_refused(host, launches):
    c = _cache()
    c.data = _gpu(c.data)
    t = {"q": torch.zeros(3, 4 * c.dk, dtype=torch.bfloat16), "out": torch.zeros(3, 4 * c.dv, dtype=torch.bfloat16), "page_table": _i32(3, 40), "positions": _i32(3),
         "seq_ids": _i32(3), "seq_lens": _i32(3), "chosen": _i32(3, 2, 8)}
    t = {k: x if k == host else _gpu(x) for k, x in t.items()}

    def call():
        SP.attn_paged_sparse(t["q"], 4, t["positions"], t["seq_ids"], c, t["page_table"], _gpu(PG.bounds_for(c)), A.attn_spec(0.1), t["out"],
                             top=8, seq_lens=t["seq_lens"], chosen=t["chosen"], splits=1)
    if host is None:
        call()
        assert len(launches) == 1
        return
    with pytest.raises(ValueError):
        call()
    assert not launches


_SPECS = {"fits": {}, "sink on the host": {"sink": lambda: torch.zeros(4)}, "gate on the host": {"gate": lambda: torch.zeros(3, 4, dtype=torch.bfloat16)},
          "few sinks": {"sink": lambda: _gpu(torch.zeros(3))}, "few rows": {"gate": lambda: _gpu(torch.zeros(2, 4, dtype=torch.bfloat16))},
          "few heads": {"gate": lambda: _gpu(torch.zeros(3, 3, dtype=torch.bfloat16))}, "another type": {"gate": lambda: _gpu(torch.zeros(3, 4))},
          "heads apart": {"gate": lambda: _gpu(torch.zeros(4, 3, dtype=torch.bfloat16).t())}, "one dimension": {"gate": lambda: _gpu(torch.zeros(12, dtype=torch.bfloat16))}}


@pytest.mark.parametrize("what", list(_SPECS))
@pytest.mark.parametrize("op", ["sparse", "shared"])
def test_sinks_and_gates_that_do_not_fit_are_refused(op, what, launches, monkeypatch):
    c = _cache()
    c.data = _gpu(c.data)
    given = {"sink": lambda: _gpu(torch.zeros(4)), "gate": lambda: _gpu(torch.zeros(3, 9, dtype=torch.bfloat16)[:, :4]), **_SPECS[what]}
    spec = A.attn_spec(0.1, **{k: f() for k, f in given.items()})
    q, out, table, n = _gpu(torch.zeros(3, 4 * c.dk, dtype=torch.bfloat16)), _gpu(torch.zeros(3, 4 * c.dv, dtype=torch.bfloat16)), _gpu(_i32(3, 40)), _gpu(_i32(3))
    monkeypatch.setattr(SH._lib, "lib", lambda: SimpleNamespace(b200_attn_paged_sparse="sparse", b200_attn_decode_shared="shared"))
    no_plan = torch.zeros(1, dtype=torch.int32)
    monkeypatch.setattr(SH.SharedPrefixes, "cut_for", lambda *a: SimpleNamespace(plan=no_plan, pieces_at=0, slots_at=0, max_pieces=0, part=no_plan, rows=1,
                                                                                                    splits=1, sms=1))

    def call():
        if op == "sparse":
            SP.attn_paged_sparse(q, 4, n, None, c, table, _gpu(PG.bounds_for(c)), spec, out, top=8, splits=1)
        else:
            SH.attn_decode_shared(q, 4, n, c, table, SH.SharedPrefixes(3, "cpu"), spec, out)
    if what == "fits":
        call()
        assert len(launches) == 1
        return
    with pytest.raises(ValueError):
        call()
    assert not launches


def test_sinks_and_gates_live_as_long_as_their_spec():
    import weakref
    gate = torch.zeros(3, 4)
    alive, spec = weakref.ref(gate), A.attn_spec(0.1, gate=gate)
    del gate
    assert alive() is not None and spec.gate == alive().data_ptr()
