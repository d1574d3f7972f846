"""Decode attention of sequences that share a prefix, against the definition in 64 bits."""
import pytest
import torch

from paged_cases import DEV, Sequences, status_ok, worst

pytestmark = pytest.mark.gpu
HEADS = [(4, 2, 64, 48), (6, 1, 40, 64), (8, 2, 128, 128), (3, 3, 24, 96), (20, 1, 64, 64), (2, 1, 200, 136), (160, 1, 64, 32), (8, 8, 128, 64), (6, 2, 104, 56)]


def _run(S, q, lens, plan, scale, sink, gate, chunk=None):
    from mojo_linuxperiments_b200.ops import attention as A
    from mojo_linuxperiments_b200.ops import shared as SH
    n = len(lens)
    out = torch.full((n, S.hq * S.dv + 8), float("nan"), dtype=S.dtype, device=DEV)
    spec = A.attn_spec(scale, chunk=chunk, sink=sink, gate=gate)
    SH.attn_decode_shared(q, S.hq, torch.tensor(lens, dtype=torch.int32, device=DEV), S.cache, S.table, plan, spec, out[:, :S.hq * S.dv])
    assert torch.isnan(out[:, S.hq * S.dv:]).all()
    return out[:, :S.hq * S.dv]


def _check(S, q, lens, groups, scale, sink=None, gate=None, chunk=None):
    from mojo_linuxperiments_b200.ops import shared as SH
    plan = SH.SharedPrefixes(len(lens), DEV)
    plan.set(groups)
    out = _run(S, q, lens, plan, scale, sink, gate, chunk)
    status_ok()
    for i, n in enumerate(lens):
        if n <= 0:
            assert float(out[i].abs().max()) == 0
            continue
        low = (n - 1) - (n - 1) % chunk if chunk else 0
        want, tol = S.want(q, i, i, list(range(low, n)), scale, sink, gate)
        assert worst(out[i], want, tol) <= 1, (i, n, worst(out[i], want, tol))
    return out


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("hq,hkv,dk,dv", HEADS)
def test_heads_groups_and_lengths(hq, hkv, dk, dv, dtype):
    for lens, groups in (([40, 33, 300, 17], [([0, 1, 2, 3], 16)]),
                         ([300, 257, 700, 256, 1, 20, 400], [([2, 0, 3, 1], 256), ([6], 384)]),
                         ([130, 129, 145], [([1, 2, 0], 128)]),
                         ([5, 64], [])):
        S = Sequences(lens, hq, hkv, dk, dv, dtype, groups=groups, seed=dk)
        q = S.rows_of(len(lens), 8)
        for sink, gate in ((True, True), (False, False)):
            s, g = S.heads_of(len(lens), sink, gate)
            _check(S, q, lens, groups, dk ** -0.5, s, g)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("chunk", [16, 50, 128, 200, 1000])
def test_chunks_that_end_inside_the_prefix_or_behind_it(chunk, dtype):
    groups = [([0, 2, 4], 320), ([3, 1], 144)]
    lens = [321, 150, 700, 144, 409]
    S = Sequences(lens, 8, 2, 64, 64, dtype, groups=groups, seed=chunk)
    q = S.rows_of(5)
    s, g = S.heads_of(5)
    _check(S, q, lens, groups, 0.2, s, g, chunk)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_sequences_that_end_inside_the_prefix_and_empty_slots(dtype):
    """A plan may say more than a sequence holds, or name a slot that has been emptied."""
    groups = [([0, 1, 2, 3, 4], 256)]
    S = Sequences([256, 300, 256, 256, 256], 4, 2, 64, 64, dtype, groups=groups, seed=1)
    q = S.rows_of(5)
    s, g = S.heads_of(5)
    for lens in ([100, 300, 0, 1, 256], [0, 0, 0, 0, 0], [16, 17, 255, 256, 129]):
        _check(S, q, lens, groups, 0.2, s, g)


def test_many_members_and_a_long_prefix():
    n = 70
    groups = [(list(range(n)), 4096), ]
    lens = [4096 + 1 + 7 * i for i in range(n)]
    S = Sequences(lens, 16, 4, 128, 128, "bfloat16", groups=groups, seed=8)
    _check(S, S.rows_of(n), lens, groups, 0.09)


def test_many_groups():
    groups = [([2 * i, 2 * i + 1], 16 * (1 + i % 5)) for i in range(40)]
    lens = [16 * (1 + (i // 2) % 5) + i % 23 for i in range(81)]
    S = Sequences(lens, 4, 2, 64, 64, "bfloat16", groups=groups, seed=8)
    _check(S, S.rows_of(81), lens, groups, 0.2)


def test_weights_far_apart():
    """Scores of hundreds: nothing overflows, whichever part holds the largest."""
    groups = [([0, 1, 2], 128)]
    S = Sequences([160, 128, 200], 4, 2, 64, 64, "bfloat16", groups=groups, seed=8, spread=6.0)
    _check(S, S.rows_of(3), S.lens, groups, 1.0)


def test_a_plan_that_changes_under_a_captured_call():
    from mojo_linuxperiments_b200.ops import attention as A
    from mojo_linuxperiments_b200.ops import shared as SH
    groups = [([0, 1, 2, 3], 512)]
    S = Sequences([600, 530, 513, 800], 8, 2, 128, 128, "bfloat16", groups=groups, seed=6)
    q = S.rows_of(4)
    lens = torch.tensor(S.lens, dtype=torch.int32, device=DEV)
    plan = SH.SharedPrefixes(4, DEV)
    plan.set(groups)
    out = torch.empty((4, 1024), dtype=S.dtype, device=DEV)
    spec = A.attn_spec(0.1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        SH.attn_decode_shared(q, 8, lens, S.cache, S.table, plan, spec, out)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            SH.attn_decode_shared(q, 8, lens, S.cache, S.table, plan, spec, out)
    torch.cuda.current_stream().wait_stream(side)
    for groups, n in (([([0, 1, 2, 3], 512)], S.lens), ([([0, 1], 256), ([3, 2], 512)], S.lens), ([], S.lens), ([([1, 3], 64)], [64, 300, 0, 700])):
        plan.set(groups)
        lens.copy_(torch.tensor(n, dtype=torch.int32))
        out.fill_(float("nan"))
        g.replay()
        status_ok()
        for i, k in enumerate(n):
            if k == 0:
                assert float(out[i].abs().max()) == 0
                continue
            want, tol = S.want(q, i, i, list(range(k)), 0.1, None, None)
            assert worst(out[i], want, tol) <= 1


def test_two_plans_on_two_streams():
    from mojo_linuxperiments_b200.ops import shared as SH
    groups = [([0, 1, 2, 3], 1024)]
    S = Sequences([1100, 1030, 1025, 1800], 8, 2, 128, 128, "bfloat16", groups=groups, seed=6)
    qs = [S.rows_of(4), S.rows_of(4)]
    plans, want = [], []
    for q in qs:
        plans.append(SH.SharedPrefixes(4, DEV))
        plans[-1].set(groups)
        want.append(_run(S, q, S.lens, plans[-1], 0.1, None, None).clone())
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = _run(S, qs[i], S.lens, plans[i], 0.1, None, None)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_the_same_call_gives_the_same_bits():
    groups = [([0, 1, 2, 3], 2048)]
    S = Sequences([2100, 2600, 2049, 2800], 32, 8, 128, 128, "bfloat16", groups=groups, seed=6)
    q = S.rows_of(4)
    first = _check(S, q, S.lens, groups, 0.09).clone()
    for _ in range(5):
        assert torch.equal(_check(S, q, S.lens, groups, 0.09), first)


@pytest.mark.parametrize("hq,hkv,dk,dv,n", [(16, 4, 128, 128, 170), (8, 8, 40, 64, 90), (40, 2, 64, 64, 120), (48, 4, 128, 96, 80)])
def test_more_slots_than_ctas(hq, hkv, dk, dv, n):
    """Empty slots, slots that share nothing and sequences of any length among them, in several waves; twice, and the same bits."""
    groups = [(list(range(0, n, 2)), 272), ([1, 3, 5, 7], 128)]
    lens = [0] * n
    for i in range(n):
        base = 272 if i % 2 == 0 else 128 if i in (1, 3, 5, 7) else 0
        lens[i] = 0 if i % 11 == 10 and base == 0 else base + (i * 37) % 200
    S = Sequences([max(1, x) for x in lens], hq, hkv, dk, dv, "bfloat16", groups=groups, seed=n)
    q = S.rows_of(n, 8)
    s, g = S.heads_of(n)
    first = _check(S, q, lens, groups, dk ** -0.5, s, g).clone()
    assert torch.equal(_check(S, q, lens, groups, dk ** -0.5, s, g), first)
    _check(S, q, lens, groups, dk ** -0.5, s, g, chunk=150)


@pytest.mark.parametrize("chunk", [None, 40, 100])
@pytest.mark.parametrize("hq,hkv,dk,dv", [(16, 4, 128, 128), (96, 4, 64, 80)])
def test_more_pieces_than_ctas(hq, hkv, dk, dv, chunk):
    """A CTA takes several pieces one after the other: of groups with one, two or some tiles, with rows for one unit or for both, seen in full, in part or not at all."""
    groups, lens, at = [], [], 0
    for i in range(70):
        members, tokens = 2 + (i % 7 == 3) * (12 if hq == 96 else 40), 16 * (1 + (i * 5) % 23)
        groups.append((list(range(at, at + members)), tokens))
        lens += [tokens + (i + j * 3) % 50 for j in range(members)]
        at += members
    S = Sequences(lens, hq, hkv, dk, dv, "bfloat16", groups=groups, seed=7)
    q = S.rows_of(len(lens))
    s, g = S.heads_of(len(lens))
    first = _check(S, q, lens, groups, dk ** -0.5, s, g, chunk).clone()
    assert torch.equal(_check(S, q, lens, groups, dk ** -0.5, s, g, chunk), first)


def test_groups_are_not_set_inside_a_capture():
    from mojo_linuxperiments_b200.ops import shared as SH
    groups = [([0, 1], 32)]
    S = Sequences([40, 40], 4, 2, 64, 64, "bfloat16", groups=groups)
    plan = SH.SharedPrefixes(2, DEV)
    q = S.rows_of(2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            with pytest.raises(RuntimeError, match="capture"):
                _run(S, q, [40, 40], plan, 0.1, None, None)            # the plan is not on the device yet
            torch.zeros(1, device=DEV).add_(1)
        _run(S, q, [40, 40], plan, 0.1, None, None)
        with torch.cuda.graph(g := torch.cuda.CUDAGraph(), stream=side):
            with pytest.raises(RuntimeError, match="captured"):
                plan.set(groups)
            torch.zeros(1, device=DEV).add_(1)
    torch.cuda.synchronize()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("chunk,lens,right", [(None, [320, 500, 100, 16, 0, 99], [2, 3, 4, 5]), (50, [320, 700, 321, 100, 319, 0], range(6)),
                                              (304, [320, 700, 321, 319, 100, 0], range(6)), (128, [320, 400, 500, 321, 50, 0], [1, 2, 4, 5])])
@pytest.mark.parametrize("hq", [8, 120])
def test_what_a_slot_does_not_see_may_be_anything(chunk, lens, right, hq, bad):
    """Positions 100 .. 299 of the prefix are not finite: rows that see none of them are as they would be without."""
    groups = [([2, 0, 1, 3, 4, 5], 320)]
    S = Sequences(lens, hq, 2, 64, 64, "bfloat16", groups=groups, seed=3)
    for at in range(100, 300):
        S.cache.keys()[S.rows[0][at // 16], :, at % 16] = bad
        S.cache.values()[S.rows[0][at // 16], :, at % 16] = bad
    q = S.rows_of(6)
    from mojo_linuxperiments_b200.ops import shared as SH
    plan = SH.SharedPrefixes(6, DEV)
    plan.set(groups)
    out = _run(S, q, lens, plan, 0.1, None, None, chunk)
    status_ok()
    for i in right:
        n = lens[i]
        low = (n - 1) - (n - 1) % chunk if chunk and n else 0
        assert not set(range(100, 300)) & set(range(low, n))
        want, tol = S.want(q, i, i, list(range(low, n)), 0.1, None, None)
        assert worst(out[i], want, tol) <= 1, (i, worst(out[i], want, tol))


@pytest.mark.parametrize("sink", [True, False])
@pytest.mark.parametrize("hq,hkv,dk,dv", [(4, 2, 64, 64), (160, 1, 64, 32), (40, 2, 128, 128), (6, 2, 40, 56)])
def test_queries_that_are_not_numbers_give_none(hq, hkv, dk, dv, sink):
    from mojo_linuxperiments_b200.ops import shared as SH
    lens, groups = [320, 400, 260, 272], [([0, 1, 2, 3], 256)]
    S = Sequences(lens, hq, hkv, dk, dv, "bfloat16", groups=groups, seed=2)
    q = S.rows_of(4)
    q[0, :dk] = float("nan")
    q[1, :hq * dk] = float("nan")
    s, _ = S.heads_of(4, sink, False)
    plan = SH.SharedPrefixes(4, DEV)
    plan.set(groups)
    out = _run(S, q, lens, plan, 0.1, s, None)
    status_ok()
    assert torch.isnan(out[0, :dv]).all() and torch.isnan(out[1]).all() and torch.isfinite(out[0, dv:]).all() and torch.isfinite(out[2:]).all()


@pytest.mark.parametrize("hq,hkv,dk,dv,n,tokens", [(32, 8, 128, 128, 24, 4096), (40, 2, 64, 64, 12, 2048), (6, 2, 104, 56, 30, 1024)])
def test_weights_add_up_to_the_denominator(hq, hkv, dk, dv, n, tokens):
    """All values are one, so every result is the sum of the weights over the denominator: exactly one, whatever the weights are rounded to.  Between
    the two stand fp32 sums of some thousand terms and a reciprocal, 2^-10 at most, where the bf16 number below one is 2^-8 away and what lies within half of that rounds to one."""
    groups = [(list(range(n)), tokens)]
    lens = [tokens + 1 + 5 * i for i in range(n)]
    S = Sequences(lens, hq, hkv, dk, dv, "bfloat16", groups=groups, seed=tokens, spread=3.0)
    S.cache.values().fill_(1.0)
    from mojo_linuxperiments_b200.ops import shared as SH
    plan = SH.SharedPrefixes(n, DEV)
    plan.set(groups)
    out = _run(S, S.rows_of(n), lens, plan, dk ** -0.5, None, None)
    status_ok()
    assert torch.equal(out, torch.ones_like(out)), (float(out.min()), float(out.max()))


def test_no_further_from_exact_than_decoding_alone():
    """A few keys decide each softmax (scores of a standard deviation of 3): the errors against 64 bits are those of the decode kernel that reads every
    sequence's keys by itself, whose weights are rounded as well, relative to the largest so far.  Errors of 4,096 independent rows: their mean square is known to
    sqrt(2 / 4096) = 2.2 %, its root to 1.1 %; 5 % are allowed.  (Weights relative to an older maximum: 12 % and more.)"""
    from mojo_linuxperiments_b200.ops import attention as A
    from mojo_linuxperiments_b200.ops import shared as SH
    n, hq, hkv, d, tokens, own = 128, 32, 8, 128, 4096, 16
    groups = [(list(range(n)), tokens)]
    S = Sequences([tokens + own] * n, hq, hkv, d, d, "bfloat16", groups=groups, seed=4, spread=3.0)
    q, per = S.rows_of(n), hq // hkv
    plan = SH.SharedPrefixes(n, DEV)
    plan.set(groups)
    got = _run(S, q, S.lens, plan, d ** -0.5, None, None)
    # the new token's key and value are in the cache already and are written there once more
    last = torch.tensor([r[-1] for r in S.rows], device=DEV)
    k, v = S.cache.keys()[last, :, own - 1].reshape(n, -1), S.cache.values()[last, :, own - 1].reshape(n, -1)
    lens = torch.tensor(S.lens, dtype=torch.int32, device=DEV)
    alone = torch.empty((n, hq * d), dtype=S.dtype, device=DEV)
    A.attn_decode_paged(torch.cat([q, k, v], 1), hq, lens - 1, lens, None, None, S.cache, S.table, A.attn_spec(d ** -0.5), alone)
    status_ok()
    want = torch.empty((n, hkv, per, d), dtype=torch.float64, device=DEV)
    for h in range(hkv):
        for i in range(0, n, 16):
            page = S.table[i:i + 16].long()
            K, V = (x()[page][:, :, h].flatten(1, 2).double() for x in (S.cache.keys, S.cache.values))
            want[i:i + 16, h] = torch.softmax(q[i:i + 16].view(-1, hkv, per, d)[:, h].double() @ K.transpose(1, 2) * d ** -0.5, -1) @ V
    off = [float((x.view_as(want).double() - want).norm() / want.norm()) for x in (got, alone)]
    assert off[0] <= 1.05 * off[1], off


def test_a_captured_call_has_the_clusters_that_sequences_without_groups_need(monkeypatch):
    """Captured while all share most of what they hold, replayed when none shares anything: as many CTAs per slot as a plan without groups would have had,
    and the same for page tables of any width that asks for as many."""
    from mojo_linuxperiments_b200.ops import attention as A
    from mojo_linuxperiments_b200.ops import shared as SH
    lens, groups = [4100, 4200, 4097, 4150], [([0, 1, 2, 3], 4096)]
    S = Sequences(lens, 8, 2, 128, 128, "bfloat16", groups=groups, seed=6)
    q, seq_lens, spec = S.rows_of(4), torch.tensor(lens, dtype=torch.int32, device=DEV), A.attn_spec(0.1)
    out, launched, run = torch.empty((4, 1024), dtype=S.dtype, device=DEV), [], SH._lib.on_device

    def on_device(device, fn, *args):
        launched.append(args[-3])
        return run(device, fn, *args)
    monkeypatch.setattr(SH._lib, "on_device", on_device)

    def call(plan, table=S.table):
        SH.attn_decode_shared(q, 8, seq_lens, S.cache, table, plan, spec, out)
    plan, other = SH.SharedPrefixes(4, DEV), SH.SharedPrefixes(4, DEV)
    plan.set(groups)
    call(other)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(plan)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            call(plan)
    torch.cuda.current_stream().wait_stream(side)
    plan.set([])
    call(plan)
    assert len(set(launched)) == 1 and launched[0] > 1, launched
    assert all(c.splits == launched[0] for c in plan._cuts.values())
    for groups in ([], [([0, 1, 2, 3], 4096)], [([3, 1], 64)]):
        plan.set(groups)
        out.fill_(float("nan"))
        g.replay()
        status_ok()
        for i, k in enumerate(lens):
            want, tol = S.want(q, i, i, list(range(k)), 0.1, None, None)
            assert worst(out[i], want, tol) <= 1
    for more in range(20):
        call(plan, torch.cat([S.table, S.table[:, :1].expand(-1, more)], 1).contiguous())
    assert len(plan._cuts) == 1
    with pytest.raises(ValueError):
        SH.attn_decode_shared(q, 8, seq_lens, S.cache, S.table, plan, spec, out, splits=9)


@pytest.mark.parametrize("bad", [-1, 1 << 30, "behind the last"])
@pytest.mark.parametrize("hq,hkv,dk,chunk", [(8, 2, 128, None), (160, 1, 64, None), (6, 2, 40, 300), (8, 2, 128, 1000)])
def test_pages_that_do_not_exist_are_left_out_and_told(hq, hkv, dk, chunk, bad):
    """In a prefix (single pages, a whole tile of eight, the last one) and among a sequence's own keys: as if the sequences did not have these tokens."""
    from mojo_linuxperiments_b200.ops import shared as SH
    lens, groups = [700, 641, 640, 655], [([2, 0, 1, 3], 640)]
    S = Sequences(lens, hq, hkv, dk, 64, "bfloat16", groups=groups, seed=5)
    q, (s, g) = S.rows_of(4), S.heads_of(4)
    plan = SH.SharedPrefixes(4, DEV)
    plan.set(groups)
    held = S.table.clone()
    for gone, slots in (([3], range(4)), ([0, 17, 39], range(4)), (list(range(16, 24)) + [31], range(4)), (list(range(40)), range(4)), ([40, 42], [0]), ([], [])):
        S.table.copy_(held)
        for t in gone:
            for i in slots:
                S.table[i, t] = S.cache.num_pages if bad == "behind the last" else bad
        out = _run(S, q, lens, plan, 0.2, s, g, chunk)
        low = [(n - 1) - (n - 1) % chunk if chunk else 0 for n in lens]
        if any(low[i] // 16 <= t <= (lens[i] - 1) // 16 for i in slots for t in gone):
            with pytest.raises(RuntimeError, match="bad argument|status 6"):
                status_ok()
        status_ok()
        for i, n in enumerate(lens):
            want, tol = S.want(q, i, i, [t for t in range(low[i], n) if i not in slots or t // 16 not in gone], 0.2, s, g)
            assert worst(out[i], want, tol) <= 1, (gone, i, worst(out[i], want, tol))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("scale", [0.0, -0.2])
def test_scales_that_are_not_positive(scale, dtype):
    """The largest product is not the largest score then: the same results in either type.  scale (q . k) is |scale| (-q . k): the definition is asked that
    way, because its bound on the sums' error, (dk + 8) 2^-24 scale sum |q k|, is one for scales that are not negative."""
    from mojo_linuxperiments_b200.ops import shared as SH
    lens, groups = [300, 257, 256, 0], [([2, 0, 1], 240)]
    S = Sequences([300, 257, 256, 1], 8, 2, 64, 64, dtype, groups=groups, seed=5)
    s, g = S.heads_of(4)
    q, plan = S.rows_of(4), SH.SharedPrefixes(4, DEV)
    plan.set(groups)
    out = _run(S, q, lens, plan, scale, s, g)
    status_ok()
    assert float(out[3].abs().max()) == 0
    for i in range(3):
        want, tol = S.want(-q, i, i, list(range(lens[i])), abs(scale), s, g)
        assert worst(out[i], want, tol) <= 1, (i, worst(out[i], want, tol))
