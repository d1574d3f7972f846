"""Copies of pages and bounds of their keys on the GPU: both are exact."""
import pytest
import torch

from paged_cases import DEV, DT, Sequences, status_ok

pytestmark = pytest.mark.gpu


def _records(shape, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randint(-2 ** 31, 2 ** 31 - 1, shape, generator=g, device=DEV, dtype=torch.int64).to(torch.int32).view(dtype)


@pytest.mark.parametrize("layers,pages,record,n", [(1, 2, 4, 1), (3, 9, 20, 4), (40, 30, 4096, 15), (70, 12, 1028, 5), (2, 9000, 16, 4400), (1, 700, 33000, 300)])
def test_copies_every_record_and_nothing_else(layers, pages, record, n):
    from mojo_linuxperiments_b200.ops import pages as PG
    # records of different lengths (in words of 4 bytes, multiples of 4), any bits
    arrays = [_records((pages, record + 8 * (i % 3)), torch.float32, i) for i in range(layers)]
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(n)).tolist()
    src, dst = order[:n], order[n:2 * n]
    src = (src * n)[:len(dst)] if n == 1 else [src[i // 2] for i in range(len(dst))]         # a page may be copied more than once
    want = [a.clone().view(torch.int32) for a in arrays]
    for w in want:
        w[torch.tensor(dst, device=DEV)] = w[torch.tensor(src, device=DEV)]
    PG.copy_pages(arrays, src, dst)
    assert all(torch.equal(a.view(torch.int32), w) for a, w in zip(arrays, want))


def test_copies_of_caches_of_several_types_and_of_odd_records():
    from mojo_linuxperiments_b200.ops import attention as A
    from mojo_linuxperiments_b200.ops import pages as PG
    caches = [A.PagedKVCache(7, 2, 16, DEV, dk=40, dv=24, dtype=torch.bfloat16), A.PagedKVCache(9, 1, 16, DEV, dk=8, dv=0, dtype=torch.float32)]
    bounds = PG.bounds_for(caches[0])
    for t in (caches[0].data, caches[1].data, bounds):
        t.normal_()
    before = [t.clone() for t in (caches[0].data, caches[1].data, bounds)]
    PG.copy_pages([*caches, bounds], torch.tensor([6, 0]), torch.tensor([1, 3]))
    for t, b in zip((caches[0].data, caches[1].data, bounds), before):
        assert torch.equal(t[1], b[6]) and torch.equal(t[3], b[0]) and torch.equal(t[[0, 2, 4, 5, 6]], b[[0, 2, 4, 5, 6]])


def test_offsets_beyond_32_bits():
    from mojo_linuxperiments_b200.ops import pages as PG
    a = torch.zeros((320, 1 << 23), dtype=torch.float16, device=DEV)              # records of 16 MB, 5 GB in all
    a[1].copy_(torch.arange(1 << 23, device=DEV) % 1021)
    PG.copy_pages(a, [1], [319])
    assert torch.equal(a[1], a[319]) and float(a[318].abs().max()) == 0


def test_a_captured_copy_and_another_stream():
    from mojo_linuxperiments_b200.ops import pages as PG
    a = _records((50, 64), torch.float32, 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        PG.copy_pages(a, [3], [4])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            PG.copy_pages(a, [1, 2], [40, 41])
            PG.copy_pages(a, [40], [42])
    torch.cuda.current_stream().wait_stream(side)
    a[1].copy_(a[9])
    g.replay()
    w = a.view(torch.int32)
    assert torch.equal(w[4], w[3]) and torch.equal(w[40], w[9]) and torch.equal(w[42], w[9]) and torch.equal(w[41], w[2])


def _bounds(S, spans):
    """the definition, at the pages that it touches"""
    out = {}
    for seq, (a, e) in spans:
        for place in range(a // S.ps, -(-e // S.ps)):
            page, n = S.rows[seq][place], min(S.ps, e - place * S.ps)
            k = S.cache.keys()[page, :, :n]
            out[page] = torch.stack([k.amin(1), k.amax(1)], 1)
    return out


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("hkv,dk,ps", [(2, 128, 16), (1, 8, 16), (3, 40, 16), (1, 300, 16), (5, 64, 16), (2, 24, 7), (1, 5, 16), (4, 128, 64)])
def test_bounds_of_every_page_that_a_portion_touches(hkv, dk, ps, dtype):
    from mojo_linuxperiments_b200.ops import pages as PG
    S = Sequences([1, ps, ps + 1, 5 * ps - 3, 900, 33], hkv, hkv, dk, 16, dtype, ps=ps)
    for spans in ([(i, (0, n)) for i, n in enumerate(S.lens)], [(4, (899, 900)), (0, (0, 1)), (3, (ps + 2, ps + 3))], [(4, (100, 700)), (2, (0, 0)), (1, (3, min(9, ps)))]):
        bounds = PG.bounds_for(S.cache).fill_(7.0)
        seqs = torch.tensor([s for s, _ in spans], dtype=torch.int32, device=DEV)
        ends = torch.tensor([x for _, x in spans], dtype=torch.int32, device=DEV)
        PG.page_bounds(S.cache, S.table, ends[:, 0].contiguous(), ends[:, 1].contiguous(), seqs, max(e - a for _, (a, e) in spans), bounds)
        status_ok()
        want = torch.full_like(bounds, 7.0)
        for page, b in _bounds(S, [x for x in spans if x[1][1] > x[1][0]]).items():
            want[page] = b
        assert torch.equal(bounds, want)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_bounds_of_keys_that_are_not_finite(dtype):
    from mojo_linuxperiments_b200.ops import pages as PG
    S = Sequences([64], 1, 1, 16, 8, dtype)
    K = S.cache.keys()
    K[S.rows[0][0], 0, 5, 3] = float("nan")
    K[S.rows[0][1], 0, 5, 3] = float("inf")
    K[S.rows[0][2], 0, 5, 3] = -float("inf")
    K[S.rows[0][3]] = torch.finfo(DT[dtype]).min
    bounds = PG.bounds_for(S.cache)
    z = torch.zeros(1, dtype=torch.int32, device=DEV)
    PG.page_bounds(S.cache, S.table, z, z + 64, None, 64, bounds)
    b = [bounds[p, 0, :, 3] for p in S.rows[0]]
    assert torch.isnan(b[0]).all() and b[1][1] == float("inf") and b[2][0] == -float("inf") and (b[3] == torch.finfo(DT[dtype]).min).all()
    assert torch.isfinite(bounds[S.rows[0][0], 0, :, :3]).all()


def test_pages_that_do_not_exist_are_told_and_left_out():
    from mojo_linuxperiments_b200.ops import pages as PG
    S = Sequences([40, 40], 1, 1, 16, 8, "bfloat16")
    bounds = PG.bounds_for(S.cache)
    z = torch.zeros(2, dtype=torch.int32, device=DEV)
    table = S.table.clone()
    table[0, 1] = S.cache.num_pages
    PG.page_bounds(S.cache, table, z, z + 40, None, 40, bounds)
    with pytest.raises(RuntimeError, match="page_bounds"):
        status_ok()
    assert torch.equal(bounds[S.rows[1][2]], _bounds(S, [(1, (0, 40))])[S.rows[1][2]])
    PG.page_bounds(S.cache, S.table, z, z + 49, None, 49, bounds)                  # longer than a row of the table
    with pytest.raises(RuntimeError, match="page_bounds"):
        status_ok()


def test_a_portion_longer_than_was_said_is_told_and_left_out():
    from mojo_linuxperiments_b200.ops import pages as PG
    S = Sequences([400], 1, 1, 16, 8, "bfloat16")
    bounds = PG.bounds_for(S.cache).fill_(7.0)
    z = torch.zeros(1, dtype=torch.int32, device=DEV)
    PG.page_bounds(S.cache, S.table, z, z + 400, None, 16, bounds)
    with pytest.raises(RuntimeError, match="page_bounds"):
        status_ok()
    assert (bounds == 7.0).all()
