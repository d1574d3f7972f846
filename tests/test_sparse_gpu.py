"""Attention over selected pages: what is selected, and the attention over it, against the definition in 64 bits."""
import pytest
import torch

from paged_cases import DEV, Sequences, status_ok, worst

pytestmark = pytest.mark.gpu
HEADS = [(4, 2, 64, 48), (6, 1, 40, 64), (8, 2, 128, 128), (3, 3, 24, 96), (20, 1, 64, 64), (2, 1, 200, 136), (32, 1, 128, 128), (8, 8, 64, 64), (6, 2, 104, 56)]


def _bounds(S):
    from mojo_linuxperiments_b200.ops import pages as PG
    b = PG.bounds_for(S.cache).fill_(float("nan"))
    z = torch.zeros(len(S.lens), dtype=torch.int32, device=DEV)
    return PG.page_bounds(S.cache, S.table, z, torch.tensor(S.lens, dtype=torch.int32, device=DEV), None, max(S.lens), b)


def _scores(S, q, row, seq, bounds, n_pages):
    """fp64 scores [hkv][pages] of a row, and how far off sums in fp32 may be"""
    per = S.hq // S.hkv
    x = q[row, :S.hq * S.dk].double().view(S.hkv, per, 1, S.dk)
    b = bounds[torch.tensor(S.rows[seq][:n_pages], device=DEV)].double().permute(1, 2, 0, 3)
    lo, hi = b[:, None, 0], b[:, None, 1]
    t = torch.maximum(x * lo, x * hi)
    return t.sum(-1).amax(1), 2 * S.dk * 2.0 ** -24 * float(t.abs().sum(-1).nan_to_num().max())


def _check(S, q, positions, seqs, bounds, *, top, first, last, scale, sink=None, gate=None, chunk=None, splits=None, live=None):
    from mojo_linuxperiments_b200.ops import attention as A
    from mojo_linuxperiments_b200.ops import sparse as SP
    n = len(positions)
    out = torch.full((n, S.hq * S.dv + 8), float("nan"), dtype=S.dtype, device=DEV)
    chosen = torch.full((n, S.hkv, top), -9, dtype=torch.int32, device=DEV)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    spec = A.attn_spec(scale, chunk=chunk, sink=sink, gate=gate)
    SP.attn_paged_sparse(q, S.hq, ints(positions), ints(seqs), S.cache, S.table, bounds, spec, out[:, :S.hq * S.dv], top=top, first=first, last=last,
                         chosen=chosen, splits=splits, seq_lens=None if live is None else ints(live))
    status_ok()
    assert torch.isnan(out[:, S.hq * S.dv:]).all()
    picked = chosen.tolist()
    for i, (pos, seq) in enumerate(zip(positions, seqs)):
        if live is not None and live[i] <= 0:
            assert float(out[i, :S.hq * S.dv].abs().max()) == 0 and all(p == -1 for h in picked[i] for p in h)
            continue
        low = pos - pos % chunk if chunk else 0
        p0, n_pages = low // S.ps, pos // S.ps + 1
        seen = n_pages - p0
        places = []
        score, off = _scores(S, q, i, seq, bounds, n_pages) if seen > top else (None, 0)
        for h in range(S.hkv):
            got = picked[i][h]
            k = min(seen, top)
            assert got[:k] == sorted(set(got[:k])) and got[k:] == [-1] * (top - k) and got[0] >= p0 and got[k - 1] == n_pages - 1
            if seen <= top:
                assert got[:k] == list(range(p0, n_pages))
            else:
                always = set(range(p0, p0 + first)) | set(range(n_pages - last, n_pages))
                assert always <= set(got)
                free = [p for p in got if p not in always]
                rest = [p for p in range(p0, n_pages) if p not in always and p not in set(free)]
                if free and rest:
                    assert score[h, free].min() >= score[h, rest].max() - 2 * off
            places.append([t for p in got[:k] for t in range(max(low, p * S.ps), min(pos + 1, (p + 1) * S.ps))])
        want, tol = S.want(q, i, seq, places, scale, sink, gate)
        assert worst(out[i, :S.hq * S.dv], want, tol) <= 1, (i, pos, worst(out[i, :S.hq * S.dv], want, tol))
    return out, chosen


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("hq,hkv,dk,dv", HEADS)
def test_heads_lengths_and_numbers_of_pages(hq, hkv, dk, dv, dtype):
    S = Sequences([1, 16, 17, 40, 300, 777], hq, hkv, dk, dv, dtype, seed=dk)
    bounds = _bounds(S)
    for top, first, last, sink, gate, splits in ((4, 1, 2, True, True, 1), (1, 0, 1, False, True, 2), (17, 0, 3, True, False, 4), (5, 2, 3, False, False, 8),
                                                (60, 1, 2, True, True, None), (3, 1, 1, False, False, 3)):
        q = S.rows_of(6, 8)
        s, g = S.heads_of(6, sink, gate)
        _check(S, q, [n - 1 for n in S.lens], list(range(6)), bounds, top=top, first=first, last=last, scale=dk ** -0.5, sink=s, gate=g, splits=splits)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("splits", [1, 2, 8])
def test_rows_anywhere_in_their_sequences(dtype, splits):
    """Several rows of one sequence, as a portion of a prompt has them: later tokens and pages are not seen."""
    S = Sequences([500, 260], 4, 2, 64, 64, dtype, seed=3)
    bounds = _bounds(S)
    positions, seqs = [499, 0, 15, 16, 170, 171, 259, 3], [0, 0, 1, 1, 0, 0, 1, 0]
    q = S.rows_of(8)
    for chunk in (None, 100, 32, 250):
        _check(S, q, positions, seqs, bounds, top=5, first=1, last=2, scale=0.3, chunk=chunk, splits=splits)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_the_pages_wanted_are_found(dtype):
    """Keys that a query looks for, on a few pages of a long sequence, decide the output as if all pages had been read."""
    from mojo_linuxperiments_b200.ops import attention as A
    from mojo_linuxperiments_b200.ops import sparse as SP
    S = Sequences([20011], 8, 2, 64, 64, dtype, seed=5, spread=0.1)
    q = S.rows_of(1)
    qh = q.view(2, 4, 64).float()
    for h, places in ((0, (70, 5003, 19000)), (1, (16, 9999))):
        for n, t in enumerate(places):
            x = qh[h, n % 4]
            S.cache.keys()[S.rows[0][t // 16], h, t % 16] = (x * (12.0 / x.norm())).to(S.dtype)
    bounds = _bounds(S)
    positions = torch.tensor([20010], dtype=torch.int32, device=DEV)
    out, full = (torch.empty((1, 8 * 64), dtype=S.dtype, device=DEV) for _ in range(2))
    spec = A.attn_spec(1.0)
    chosen = torch.empty((1, 2, 24), dtype=torch.int32, device=DEV)
    SP.attn_paged_sparse(q, 8, positions, None, S.cache, S.table, bounds, spec, out, top=24, chosen=chosen)
    A.attn_paged(q, 8, positions, None, S.cache, S.table, spec, full)
    status_ok()
    assert {70 // 16, 5003 // 16, 19000 // 16} <= set(chosen[0, 0].tolist()) and {1, 9999 // 16} <= set(chosen[0, 1].tolist())
    heads = [0, 1, 2, 4, 5]                             # those that look for something
    a, b = out.view(8, 64)[heads].float(), full.view(8, 64)[heads].float()
    # what the other pages weigh, 20,011 keys with products of a standard deviation of 0.8: less than 1e-5 of e^(12 |q|) with |q| about 8
    assert float((a - b).abs().max()) < 0.03


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("splits", [1, 2, 4, 8])
def test_equal_scores_take_the_lower_page(dtype, splits):
    """Small whole numbers: sums are exact, and many are equal."""
    from mojo_linuxperiments_b200.ops import attention as A
    from mojo_linuxperiments_b200.ops import sparse as SP
    S = Sequences([1600, 1599, 900], 4, 2, 16, 16, dtype, seed=9)
    g = torch.Generator(device=DEV).manual_seed(1)
    bounds = torch.randint(-1, 2, (S.cache.num_pages, 2, 2, 16), generator=g, device=DEV).sort(2).values.to(S.dtype)
    bounds[:, 1] = 1.0                                  # the second head's are all equal
    q = torch.randint(-1, 2, (3, 64), generator=g, device=DEV).to(S.dtype)
    for top, first, last in ((10, 1, 2), (40, 0, 1), (55, 3, 1), (2, 1, 1)):
        chosen = torch.empty((3, 2, top), dtype=torch.int32, device=DEV)
        out = torch.empty((3, 64), dtype=S.dtype, device=DEV)
        SP.attn_paged_sparse(q, 4, torch.tensor([n - 1 for n in S.lens], dtype=torch.int32, device=DEV), None, S.cache, S.table, bounds, A.attn_spec(0.1), out,
                             top=top, first=first, last=last, chosen=chosen, splits=splits)
        status_ok()
        for i, n in enumerate(S.lens):
            pages = -(-n // 16)
            score, _ = _scores(S, q, i, i, bounds, pages)
            for h in range(2):
                free = list(range(first, pages - last))
                best = sorted(free, key=lambda p: (-float(score[h, p]), p))[:top - first - last]
                assert chosen[i, h].tolist() == sorted(list(range(first)) + best + list(range(pages - last, pages)))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_bounds_that_are_not_finite(dtype):
    S = Sequences([640], 2, 1, 32, 32, dtype, seed=2)
    bounds = _bounds(S)
    q = S.rows_of(1)
    bounds[S.rows[0][7], 0, 0, 3] = float("nan")                    # taken rather than lost
    bounds[S.rows[0][9], 0, :, 4] = float("inf") * torch.sign(q[0, 4].float())
    _, chosen = None, None
    from mojo_linuxperiments_b200.ops import attention as A
    from mojo_linuxperiments_b200.ops import sparse as SP
    chosen, out = torch.empty((1, 1, 5), dtype=torch.int32, device=DEV), torch.empty((1, 64), dtype=S.dtype, device=DEV)
    SP.attn_paged_sparse(q, 2, torch.tensor([639], dtype=torch.int32, device=DEV), None, S.cache, S.table, bounds, A.attn_spec(0.2), out, top=5, chosen=chosen)
    got = set(chosen.flatten().tolist())
    assert {0, 7, 9, 38, 39} == got and torch.isfinite(out).all()


def test_empty_slots_bad_rows_and_their_status():
    S = Sequences([100, 100, 100], 4, 2, 64, 64, "bfloat16", seed=4)
    bounds, q = _bounds(S), S.rows_of(3)
    _check(S, q, [99, 0, 50], [0, 1, 2], bounds, top=4, first=1, last=2, scale=0.1, live=[100, 0, 51])
    from mojo_linuxperiments_b200.ops import attention as A
    from mojo_linuxperiments_b200.ops import sparse as SP
    for positions, seqs in (([99, -1, 5], [0, 1, 2]), ([99, 112, 5], [0, 1, 2]), ([99, 3, 5], [0, 3, 2]), ([99, 3, 5], [0, -1, 2])):
        out = torch.full((3, 256), float("nan"), dtype=S.dtype, device=DEV)
        ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
        SP.attn_paged_sparse(q, 4, ints(positions), ints(seqs), S.cache, S.table, bounds, A.attn_spec(0.1), out, top=4)
        with pytest.raises(RuntimeError, match="attn_paged_sparse"):
            status_ok()
        assert float(out[1].abs().max()) == 0 and torch.isfinite(out).all()


def test_a_captured_call_follows_its_positions():
    from mojo_linuxperiments_b200.ops import attention as A
    from mojo_linuxperiments_b200.ops import sparse as SP
    S = Sequences([900, 500], 8, 2, 128, 128, "bfloat16", seed=6)
    bounds, q = _bounds(S), S.rows_of(2)
    pos = torch.tensor([899, 499], dtype=torch.int32, device=DEV)
    out, other = (torch.empty((2, 1024), dtype=S.dtype, device=DEV) for _ in range(2))
    spec = A.attn_spec(0.1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        SP.attn_paged_sparse(q, 8, pos, None, S.cache, S.table, bounds, spec, out, top=6)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            SP.attn_paged_sparse(q, 8, pos, None, S.cache, S.table, bounds, spec, out, top=6)
    torch.cuda.current_stream().wait_stream(side)
    for p in ([899, 499], [16, 33], [700, 0]):
        pos.copy_(torch.tensor(p, dtype=torch.int32))
        out.fill_(float("nan"))
        g.replay()
        SP.attn_paged_sparse(q, 8, pos, None, S.cache, S.table, bounds, spec, other, top=6)
        assert torch.equal(out, other)
    status_ok()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_more_pages_than_a_selection_holds_at_once(dtype):
    """20,000 and 9,000 pages: whole numbers with many equal scores, whose order is known."""
    from mojo_linuxperiments_b200.ops import attention as A
    from mojo_linuxperiments_b200.ops import sparse as SP
    g = torch.Generator(device=DEV).manual_seed(3)
    n = [20000, 9000]
    cache = A.PagedKVCache(64, 1, 16, DEV, dk=16, dv=16, dtype=torch.float32 if dtype == "float32" else torch.bfloat16)
    cache.data.normal_(generator=g)
    table = torch.randint(0, 64, (2, n[0]), generator=g, device=DEV, dtype=torch.int32)            # pages seen many times over
    bounds = torch.randint(-2, 3, (64, 1, 2, 16), generator=g, device=DEV).sort(2).values.to(cache.data.dtype)
    q = torch.randint(-1, 2, (2, 32), generator=g, device=DEV).to(cache.data.dtype)
    pos = torch.tensor([16 * k - 3 for k in n], dtype=torch.int32, device=DEV)
    for top in (100, 1500, 3):
        chosen, out = torch.empty((2, 1, top), dtype=torch.int32, device=DEV), torch.empty((2, 32), dtype=cache.data.dtype, device=DEV)
        SP.attn_paged_sparse(q, 2, pos, None, cache, table, bounds, A.attn_spec(0.1), out, top=top, chosen=chosen)
        status_ok()
        for i, k in enumerate(n):
            x = q[i].double().view(2, 1, 16)
            b = bounds[:, 0].double()
            score = torch.maximum(x * b[:, 0], x * b[:, 1]).sum(-1).amax(0)[table[i, :k].long()]
            score[0], score[k - 2:] = 1e9, 1e9
            want = torch.sort(score, descending=True, stable=True).indices[:top].sort().values
            assert torch.equal(chosen[i, 0].long(), want), (top, i)


@pytest.mark.parametrize("sink", [True, False])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("hq,hkv,dk,dv", [(4, 2, 64, 64), (20, 1, 128, 128), (6, 2, 40, 56)])
def test_queries_that_are_not_numbers_give_none(hq, hkv, dk, dv, dtype, sink):
    from mojo_linuxperiments_b200.ops import attention as A
    from mojo_linuxperiments_b200.ops import sparse as SP
    S = Sequences([500, 40, 300], hq, hkv, dk, dv, dtype, seed=2)
    q = S.rows_of(3)
    q[0, :dk] = float("nan")
    q[1] = float("nan")
    s, _ = S.heads_of(3, sink, False)
    pos = torch.tensor([499, 39, 299], dtype=torch.int32, device=DEV)
    out = torch.empty((3, hq * dv), dtype=S.dtype, device=DEV)
    SP.attn_paged_sparse(q, hq, pos, None, S.cache, S.table, _bounds(S), A.attn_spec(0.1, sink=s), out, top=8)
    status_ok()
    assert torch.isnan(out[0, :dv]).all() and torch.isnan(out[1]).all() and torch.isfinite(out[0, dv:]).all() and torch.isfinite(out[2]).all()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_more_pages_than_a_chunk_has(dtype):
    """Room for all pages of a table of 140,000, which no row ever sees: a row's list is as long as its chunk."""
    S = Sequences([700, 300], 4, 2, 64, 64, dtype, seed=3)
    bounds, held = _bounds(S), S.table
    S.table = torch.full((2, 140000), S.rows[0][0], dtype=torch.int32, device=DEV)
    S.table[:, :held.shape[1]] = held
    q = S.rows_of(2)
    from mojo_linuxperiments_b200.ops import attention as A
    from mojo_linuxperiments_b200.ops import sparse as SP
    for chunk in (50, 200):
        for splits in (None, 1, 8):
            out = torch.empty((2, 4 * 64), dtype=S.dtype, device=DEV)
            positions = torch.tensor([699, 298], dtype=torch.int32, device=DEV)
            SP.attn_paged_sparse(q, 4, positions, None, S.cache, S.table, bounds, A.attn_spec(0.2, chunk=chunk), out, top=140000, splits=splits)
            status_ok()
            for i, pos in enumerate((699, 298)):
                want, tol = S.want(q, i, i, list(range(pos - pos % chunk, pos + 1)), 0.2, None, None)
                assert worst(out[i], want, tol) <= 1
