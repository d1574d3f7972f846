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
