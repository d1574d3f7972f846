"""Forked sequences through the engine: each must go on as if it had been run by itself, whatever is shared, moved or read once for all."""
import pytest
import torch

from mojo_linuxperiments_b200.models import config as C
from mojo_linuxperiments_b200.models import layered_config as LC

pytestmark = pytest.mark.gpu
CONFIGS = {"dense": (C.tiny_dense, "bfloat16"), "moe": (C.tiny_moe, "bfloat16"), "volonex": (LC.tiny_volonex, "bfloat16"), "volonex32": (LC.tiny_volonex, "float32"),
           "rakelorn": (LC.tiny_rakelorn, "bfloat16")}
# Between two kernels of the same attention: its output is rounded to bf16 (2^-9 of it in the mean) and, in the W8A8 models, to 8 bits of its largest
# element once more (about 1/254 of it), in each of a few layers; in 32 bits sums of up to 200 terms, 2e-5 as in the comparisons with the oracle
TOL = {"float32": 2e-5, "bfloat16": 4e-2}
PROMPT, STEPS, SLOTS = 70, 40, 4


def _engine(kind, weights=None, **rt):
    from mojo_linuxperiments_b200.engine.engine import Engine
    make, dtype = CONFIGS[kind]
    eng = Engine(make(), C.RuntimeConfig(max_seq_len=256, dtype=dtype, **rt), weights=weights, seed=3)
    eng.start_batch(SLOTS, 200)
    return eng


def _tokens(vocab):
    g = torch.Generator().manual_seed(11)
    return torch.randint(0, vocab, (PROMPT,), generator=g), torch.randint(0, vocab, (STEPS, SLOTS), generator=g)


def _alone(kind):
    """logits of every step and slot, no slot ever forked: slot 2 has the tokens of slot 1 until it parts from it at step 10"""
    eng = _engine(kind)
    prompt, toks = _tokens(eng.cfg.vocab)
    for s in range(SLOTS):
        eng.step([(s, prompt, [PROMPT - 1])])
    out = []
    for t in range(STEPS):
        row = toks[t].clone()
        if t < 10:
            row[2] = row[1]
        out.append(torch.stack([x[0] for x in eng.step([(s, row[s:s + 1], [0]) for s in range(SLOTS)])]))
    eng.check_status()
    return eng.model.w, out


def _forked(eng):
    prompt, toks = _tokens(eng.cfg.vocab)
    eng.step([(0, prompt, [PROMPT - 1])])
    eng.fork_sequence(0, [1, 3])
    out = []
    for t in range(STEPS):
        live = [0, 1, 3]
        if t == 10:
            eng.fork_sequence(1, [2])
        if t >= 10:
            live = [0, 1, 2, 3]
        if t in (5, 15, 33):
            eng.compact_cache()
            used = eng.kv.pages_in_use()
            assert all(p < used for pages in eng.kv.owned.values() for p in pages)
        out.append(dict(zip(live, (x[0] for x in eng.step([(s, toks[t][s:s + 1], [0]) for s in live])))))
    eng.check_status()
    return out


def _rel(a, b):
    return float((a.double() - b.double()).pow(2).mean().sqrt() / b.double().pow(2).mean().sqrt())


def _near(kind, got, want):
    """Every row within the tolerance.  With a router a row may differ by an expert: the random routers' fourth and fifth logit of sixteen lie 0.3 of their
    standard deviation apart in the mean, so what moves a logit by 0.01 of it sends about 2 x 0.01 / 0.3 = 7 % of the rows elsewhere in one of two layers: 13 %
    of 150 rows, 20 with a standard deviation of 4, so at most 40; such a row has another expert in the place of one of four, whose output
    is of the same size: off by sqrt(2) / 4 of the mixtures' part, less than half of all."""
    tol, off = TOL[CONFIGS[kind][1]], []
    for t, logits in enumerate(got):
        for s, x in logits.items():
            off.append(_rel(x, want[t][s]))
            assert off[-1] < (0.5 if kind == "moe" else tol), (t, s)
    assert sum(o > tol for o in off) <= 40


@pytest.fixture(scope="module")
def alone():
    kept = {}

    def get(kind):
        if kind not in kept:
            kept[kind] = _alone(kind)
        return kept[kind]
    return get


@pytest.mark.parametrize("kind", list(CONFIGS))
def test_forked_sequences_go_on_as_if_alone(kind, alone):
    """The same kernels over the same numbers, wherever their pages are."""
    weights, want = alone(kind)
    for t, got in enumerate(_forked(_engine(kind, weights))):
        for s, x in got.items():
            assert _rel(x, want[t][s]) < TOL[CONFIGS[kind][1]] / 4, (t, s)


@pytest.mark.parametrize("kind", list(CONFIGS))
def test_shared_prefixes_read_once(kind, alone):
    weights, want = alone(kind)
    eng = _engine(kind, weights, share_prefix=True)
    _near(kind, _forked(eng), want)
    if kind in ("dense", "moe"):
        # 70 tokens: four full pages for all; slots 1 and 2 have 80 tokens in common, five pages
        assert eng.kv.shared.groups == [([0, 1, 2, 3], 64)]
        eng.release_sequence(0), eng.release_sequence(3)
        eng.decode_step()
        assert eng.kv.shared.groups == [([1, 2], 80)]
        eng.release_sequence(1)
        eng.decode_step()
        assert eng.kv.shared.groups == []
        eng.check_status()


@pytest.mark.parametrize("kind", ["dense", "moe", "volonex", "volonex32"])
def test_as_many_selected_pages_as_there_are(kind, alone):
    """Pages selected with room for all of them: attention to every key, also of forked and moved sequences, through prompts, decoding and its graph."""
    weights, want = alone(kind)
    _near(kind, _forked(_engine(kind, weights, sparse_pages=16)), want)


@pytest.mark.parametrize("kind", ["dense", "volonex", "volonex32"])
def test_few_selected_pages_keep_their_bounds_up_to_date(kind):
    """The bounds that the engine keeps are those of the keys in its cache, through prompts in portions, decoding, forks and compaction."""
    eng = _engine(kind, sparse_pages=3)
    got = _forked(eng)
    assert all(torch.isfinite(x).all() for logits in got for x in logits.values())
    kv = eng.kv
    for run, bounds in enumerate(kv.bounds):
        if bounds is None:
            continue
        K = kv.layers[run].keys()
        for s, pages in kv.owned.items():
            for i, p in enumerate(pages):
                n = min(16, eng._lens[s] - 16 * i)
                if p < 0 or n <= 0:
                    continue
                k = K[p, :, :n]
                assert torch.equal(bounds[p], torch.stack([k.amin(1), k.amax(1)], 1)), (run, s, i)


def test_a_fork_of_everything_and_greedy_decoding():
    """Forks alone do not part: greedy decoding gives every copy the same tokens, as many steps as its source by itself."""
    eng = _engine("dense", share_prefix=True)
    prompt = torch.randint(0, eng.cfg.vocab, (1, 33), generator=torch.Generator().manual_seed(2))
    other = _engine("dense", eng.model.w, share_prefix=True)
    eng.step([(0, prompt[0], [32])]), other.step([(0, prompt[0], [32])])
    eng.fork_sequence(0, [1, 2, 3])
    for _ in range(20):
        toks = eng.decode_step().tolist()
        assert toks == [other.decode_step().tolist()[0]] * 4
    eng.check_status()
    with pytest.raises(ValueError):
        eng.fork_sequence(0, [0])
    with pytest.raises(ValueError):
        eng.fork_sequence(0, [1, 1])
    with pytest.raises(IndexError):
        eng.fork_sequence(0, [4])
    eng.release_sequence(2)
    with pytest.raises(ValueError):
        eng.fork_sequence(2, [1])


def _wide_heads():
    from dataclasses import replace
    cfg = LC.tiny_volonex()
    return replace(cfg, layers=tuple(replace(x, mixer=replace(x.mixer, dim=200, vdim=136)) for x in cfg.layers))


@pytest.mark.parametrize("kind,rt", [("wide", {}), ("volonex32", {}), ("dense", {"page_size": 32})])
def test_what_no_prefix_kernel_takes_decodes_as_without_the_option(kind, rt, monkeypatch):
    """Heads above 128, 32 bits, other pages: the same kernels in a step, and the same bits."""
    monkeypatch.setitem(CONFIGS, "wide", (_wide_heads, "bfloat16"))
    plain = _engine(kind, **rt)
    want = _forked(plain)
    eng = _engine(kind, plain.model.w, share_prefix=True, **rt)
    got = _forked(eng)
    assert eng.kernels_per_step == plain.kernels_per_step
    assert all(torch.equal(x, want[t][s]) for t, logits in enumerate(got) for s, x in logits.items())


def _open_chunks():
    """Layers that see everything, and one that sees up to seven pages."""
    from dataclasses import replace
    cfg = LC.tiny_volonex()
    return replace(cfg, layers=tuple(replace(x, mixer=replace(x.mixer, chunk=100 if x.mixer.chunk == 24 else None)) for x in cfg.layers))


def _select(eng, use_graph):
    """A prompt of 182 tokens, forks and compaction between the steps; logits per step and slot"""
    g = torch.Generator().manual_seed(12)
    prompt, toks = torch.randint(0, eng.cfg.vocab, (182,), generator=g), torch.randint(0, eng.cfg.vocab, (14, SLOTS), generator=g)
    eng.step([(0, prompt, [181])])
    eng.fork_sequence(0, [1, 3])
    out = []
    for t in range(len(toks)):
        if t == 6:
            eng.fork_sequence(1, [2])
        if t in (3, 9):
            eng.compact_cache()
        if t == 11:
            eng.release_sequence(0)
        live = [s for s in range(SLOTS) if (s != 2 or t >= 6) and (s != 0 or t < 11)]
        out += [x[0].clone() for x in eng.step([(s, toks[t][s:s + 1], [0]) for s in live], use_graph=use_graph)]
    eng.check_status()
    return out


@pytest.mark.parametrize("kind", ["dense", "open", "open32"])
def test_decoding_attends_to_the_pages_that_the_real_keys_select(kind, monkeypatch):
    """Four pages of up to thirteen, one of them by score.  Every call of an eager run is held against 64 bits: the bounds that the engine keeps are those of the keys in its
    cache, through prompts in portions of 24 tokens (16 and 24 are no multiples of one another: portions begin inside pages), decoding, forks and compaction; the pages are
    those of the largest scores by these keys; the result is the attention over them.  The captured step gives the same bits."""
    from mojo_linuxperiments_b200.models import decoder, mixers
    from mojo_linuxperiments_b200.ops.sparse import attn_paged_sparse
    from paged_cases import HALF_STEP
    monkeypatch.setitem(CONFIGS, "open", (_open_chunks, "bfloat16"))
    monkeypatch.setitem(CONFIGS, "open32", (_open_chunks, "float32"))
    rt = {} if kind == "dense" else {"max_prefill_tokens": 24}
    graphs = _engine(kind, sparse_pages=4, **rt)
    want = _select(graphs, True)

    top, first, last, by_score, asked = 4, 1, 2, [0], {}
    make = mixers.A.attn_spec

    def attn_spec(scale, *, chunk=None, sink=None, gate=None):
        asked.update(scale=scale, chunk=chunk, sink=sink, gate=gate)
        return make(scale, chunk=chunk, sink=sink, gate=gate)

    def checked(q, hq, positions, seq_ids, cache, table, bounds, spec, out, *, top, seq_lens):
        chosen = torch.empty((positions.numel(), cache.kv_heads, top), dtype=torch.int32, device=q.device)
        attn_paged_sparse(q, hq, positions, seq_ids, cache, table, bounds, spec, out, top=top, seq_lens=seq_lens, chosen=chosen)
        per, half, dk, dv = hq // cache.kv_heads, HALF_STEP[q.dtype], cache.dk, cache.dv
        for b, (pos, n) in enumerate(zip(positions.tolist(), seq_lens.tolist())):
            if n == 0:
                continue
            low = pos - pos % asked["chunk"] if asked["chunk"] else 0
            p0, p1 = low // 16, pos // 16 + 1
            pages = table[b, p0:p1].long()
            K, V = cache.keys()[pages].double(), cache.values()[pages].double()              # [pages][kv_heads][16][d]
            assert torch.equal(bounds[pages[:-1]], torch.stack([K[:-1].amin(2), K[:-1].amax(2)], 2).to(q.dtype))
            for h in range(cache.kv_heads):
                x = q[b, :hq * dk].double().view(hq, dk)[h * per:(h + 1) * per]
                got = [c - p0 for c in chosen[b, h].tolist() if c >= 0]
                if p1 - p0 <= top:
                    assert got == list(range(p1 - p0))
                else:
                    terms = torch.maximum(x[:, None] * K[:-1, h].amin(1), x[:, None] * K[:-1, h].amax(1))      # of every page but the last
                    score, off = terms.sum(-1).amax(0).tolist(), 2 * dk * 2.0 ** -24 * float(terms.abs().sum(-1).max())
                    free = range(first, p1 - p0 - last)
                    taken = [c for c in got if c in free]
                    assert len(got) == top and got[0] == 0 and got[-2:] == [p1 - p0 - 2, p1 - p0 - 1] and len(taken) == 1
                    assert score[taken[0]] >= max(score[c] for c in free) - 2 * off
                    by_score[0] += taken[0] != free[-1]
                at = torch.tensor([(c, r) for c in got for r in range(16) if low <= (p0 + c) * 16 + r <= pos], device=q.device)
                k, v = K[at[:, 0], h, at[:, 1]], V[at[:, 0], h, at[:, 1]]
                s = x @ k.t() * asked["scale"]
                off = (dk + 8) * 2.0 ** -24 * float((x.abs() @ k.abs().t() * asked["scale"]).max())
                if asked["sink"] is not None:
                    s = torch.cat([s, asked["sink"][h * per:(h + 1) * per].double()[:, None]], 1)
                w = torch.softmax(s, 1)[:, :len(at)]
                f = torch.sigmoid(asked["gate"][b, h * per:(h + 1) * per].double())[:, None] if asked["gate"] is not None else 1.0
                o, a = w @ v * f, w @ v.abs() * f
                # as in paged_cases: the weights' rounding in the numerator and the denominator, sums and exponentials, the result's rounding
                tol = half * o.abs() + ((2 * half if q.dtype != torch.float32 else 0.0) + 2 * off + 2.0 ** -18 + len(at) * 2.0 ** -23) * a + 1e-30
                err = (out[b, :hq * dv].double().view(hq, dv)[h * per:(h + 1) * per] - o).abs()
                assert bool((err <= tol).all()), (b, h, float((err / tol).max()))
        return out

    eager = _engine(kind, graphs.model.w, sparse_pages=4, **rt)
    for m in (decoder, mixers):
        monkeypatch.setattr(m, "attn_paged_sparse", checked)
    monkeypatch.setattr(mixers.A, "attn_spec", attn_spec)
    got = _select(eager, False)
    assert by_score[0] > 50                        # the page before the last two is not all that is ever taken
    assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))


def test_what_shared_prefixes_hold_is_reported():
    eng = _engine("volonex", share_prefix=True)
    assert eng.memory_report()["shared_prefixes"] == {"groups": 0, "bytes": 0}
    before = torch.cuda.memory_allocated()
    _forked(eng)
    rep, cuts = eng.memory_report()["shared_prefixes"], eng.kv.shared._cuts.values()
    assert rep["groups"] == len(eng.kv.shared.groups)
    assert 0 < rep["bytes"] == sum(c.plan.numel() * 4 + c.part.numel() * 4 for c in cuts) <= torch.cuda.memory_allocated() - before
    assert "shared_prefixes" not in _engine("volonex").memory_report()


@pytest.mark.parametrize("option", [{}, {"share_prefix": True}])
@pytest.mark.parametrize("kind", ["volonex", "volonex32", "rakelorn"])
def test_forked_slots_go_on_with_portions_of_their_own(kind, option, alone):
    """Behind a common beginning every slot has a portion of several tokens, of its own length, and then decodes: as if each had been run by itself, in the same portions."""
    weights, _ = alone(kind)
    one, eng = _engine(kind, weights, max_prefill_tokens=24), _engine(kind, weights, max_prefill_tokens=24, **option)
    prompt, toks = _tokens(eng.cfg.vocab)
    own = [(s, prompt[5 * s:5 * s + 7 + 9 * s], [6 + 9 * s]) for s in range(SLOTS)]
    for s in range(SLOTS):
        one.step([(s, prompt, [PROMPT - 1])])
    eng.step([(0, prompt, [PROMPT - 1])])
    eng.fork_sequence(0, [1, 2, 3])
    want, got = one.step(own), eng.step(own)
    assert all(_rel(a, b) < TOL[CONFIGS[kind][1]] / 4 for a, b in zip(got, want))
    for t in range(6):
        entries = [(s, toks[t][s:s + 1], [0]) for s in range(SLOTS)]
        want, got = one.step(entries), eng.step(entries)
        assert all(_rel(a, b) < TOL[CONFIGS[kind][1]] / (1 if option else 4) for a, b in zip(got, want)), t
    eng.check_status()
