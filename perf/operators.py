"""Operators of the paged cache measured one by one: copies of pages, bounds of the keys of a page, decode attention of sequences that
share a prefix, and attention over the pages that those bounds select.

``run`` computes an operator in elementary torch operations, or, where ``own`` is set, calls the framework.  The caches are those of a serving
program: records of 16 tokens, all heads' keys and then all heads' values, in pages that lie anywhere in the pool."""
from __future__ import annotations

import math
import zlib

import torch

own = False

DEVICE = "cuda"
PAGE = 16
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ---- cases --------------------------------------------------------------------------------------------------------------------
def copy(name, pages, layers, kv_heads, dk, dv, dtype="bf16"):
    return named(name, {"op": "copy", "pages": pages, "layers": layers, "kv_heads": kv_heads, "dk": dk, "dv": dv, "dtype": dtype})


def bounds(name, portions, tokens, before, kv_heads, dk, dtype="bf16"):
    return named(name, {"op": "bounds", "portions": portions, "tokens": tokens, "before": before, "kv_heads": kv_heads, "dk": dk, "dtype": dtype})


def shared(name, groups, members, prefix, rest, heads, kv_heads, dk=128, dv=128, chunk=0, sink=False, gate=False, dtype="bf16"):
    return named(name, {"op": "shared", "groups": groups, "members": members, "prefix": prefix, "rest": rest, "heads": heads, "kv_heads": kv_heads,
                        "dk": dk, "dv": dv, "chunk": chunk, "sink": sink, "gate": gate, "dtype": dtype})


def sparse(name, batch, tokens, top, heads, kv_heads, dk=128, dv=128, sink=False, gate=False, dtype="bf16"):
    return named(name, {"op": "sparse", "batch": batch, "tokens": tokens, "top": top, "first": 1, "last": 2, "heads": heads, "kv_heads": kv_heads,
                        "dk": dk, "dv": dv, "sink": sink, "gate": gate, "dtype": dtype})


def named(name, case):
    return {"name": name, **case} if name else case


def listed():
    return [
        # a sequence is forked: its last, partly filled page in all layers of the 8B shape
        copy("copy_fork", 1, 32, 8, 128, 128),
        # a pool is compacted after many sequences have ended
        copy("copy_compact", 1500, 16, 8, 128, 128),
        # a decode step of a batch: the page that each new token went to
        bounds("bounds_step", 32, 1, 2000, 8, 128),
        # long prompts of different lengths
        bounds("bounds_prompts", 8, 30001, 0, 8, 128),
        # a few answers to one short question
        shared("shared_few", 1, 4, 512, 40, 32, 8),
        # the benchmark's batch behind one system prompt
        shared("shared_batch", 1, 32, 2048, 300, 32, 8),
        # a wide batch that asks about one long document
        shared("shared_document", 1, 128, 32768, 1000, 32, 8),
        # several documents at once, of a model with chunked attention, sinks and gates
        shared("shared_groups", 6, 11, 1500, 700, 16, 8, chunk=1024, sink=True, gate=True),
        # two continuations of a trace in 32 bits
        shared("shared_trace", 1, 2, 96, 94, 16, 8, sink=True, gate=True, dtype="fp32"),
        # one user with a very long context
        sparse("sparse_long", 1, 131071, 128, 32, 8),
        # a batch of long contexts, eight query heads per KV head
        sparse("sparse_batch", 16, 16001, 64, 32, 4),
        # a trace in 32 bits
        sparse("sparse_trace", 2, 900, 16, 16, 8, sink=True, gate=True, dtype="fp32"),
    ]


HEADS = [(32, 8, 128, 128), (32, 8, 128, 128), (32, 4, 128, 128), (64, 4, 128, 128), (16, 8, 128, 128), (8, 1, 128, 128), (6, 2, 48, 80), (20, 2, 64, 64),
         (12, 4, 104, 56)]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["copy", "bounds", "shared", "shared", "shared", "sparse", "sparse"])
    hq, hkv, dk, dv = rng.choice(HEADS)
    if op == "copy":
        layers = log(1, 40)
        return copy(None, log(1, max(2, min(2000, 24000 * 32768 // (layers * hkv * PAGE * (dk + dv))))), layers, hkv, dk, dv, rng.choice(["bf16", "bf16", "fp32"]))
    if op == "bounds":
        portions = log(1, 128)
        return bounds(None, portions, rng.choice([1, log(1, 240000 // portions)]), rng.choice([0, log(1, 500)]), hkv, dk, rng.choice(["bf16", "bf16", "fp32"]))
    features = {"sink": rng.random() < 0.3, "gate": rng.random() < 0.3}
    if rng.random() < 0.15:             # 32 bits: traces, a few short sequences
        if op == "shared":
            return shared(None, 1, log(1, 4), log(16, 1000), log(1, 300), hq, hkv, dk, dv, dtype="fp32", **features)
        return sparse(None, log(1, 4), log(100, 2000), log(8, 32), hq, hkv, dk, dv, dtype="fp32", **features)
    if op == "shared":
        groups = rng.choice([1, 1, 1, log(2, 16)])
        members = log(1, max(2, 128 // groups))
        prefix = log(16, max(1000, min(32768, 131072 // groups)))
        return shared(None, groups, members, prefix, log(1, max(2, min(2000, 128000 // (groups * members)))), hq, hkv, dk, dv,
                      chunk=rng.choice([0, 0, 0, log(200, 8000)]), **features)
    batch = log(1, 64)
    return sparse(None, batch, log(100, max(2000, min(131072, 262144 // batch))), log(8, 256), hq, hkv, dk, dv, **features)


# ---- what the sizes of a case come to ---------------------------------------------------------------------------------------------
def spread(n, most, least=1, step=1):
    """n sizes from ``least`` to ``most`` in multiples of ``step``, in no order; the largest is among them."""
    span = max(0, most - least) // step
    return [least + step * (span - (i * 2654435761 % 4294967296) * (span + 1) // 4294967296 if i else span) for i in range(n)]


def pages_of(tokens):
    return -(-tokens // PAGE)


def members_of(c):
    """(slots of every group, tokens that they share, length of every slot): groups of different sizes whose members lie anywhere in the batch"""
    sizes = spread(c["groups"], c["members"], max(1, c["members"] // 2))
    prefix = [PAGE * p for p in spread(c["groups"], max(1, c["prefix"] // PAGE), max(1, c["prefix"] // (2 * PAGE)))]
    n = sum(sizes)
    order = sorted(range(n), key=lambda i: zlib.crc32(b"%d" % i))
    slots, at = [], 0
    for s in sizes:
        slots.append(order[at:at + s])
        at += s
    rest, lens = spread(n, c["rest"]), [0] * n
    for g, own_slots in enumerate(slots):
        for i in own_slots:
            lens[i] = prefix[g] + rest[i]
    return slots, prefix, lens


def spans_of(c):
    """first and end position of every portion"""
    sizes = spread(c["portions"], c["tokens"], max(1, c["tokens"] // 4))
    before = spread(c["portions"], c["before"], c["before"] // 2) if c["before"] else [0] * c["portions"]
    return before, [a + n for a, n in zip(before, sizes)]


def lens_of(c):
    return spread(c["batch"], c["tokens"], max(1, c["tokens"] // 2))


def item(c):
    return TYPES[c["dtype"]].itemsize


def work(c):
    op, size = c["op"], item(c)
    if op == "copy":
        record = c["kv_heads"] * PAGE * (c["dk"] + c["dv"]) * size
        return {"bytes": 2 * record * c["pages"] * c["layers"] + 8 * c["pages"], "flops": 0}
    if op == "bounds":
        first, end = spans_of(c)
        tokens = sum(e - a // PAGE * PAGE for a, e in zip(first, end))
        pages = sum(pages_of(e) - a // PAGE for a, e in zip(first, end))
        return {"bytes": (tokens + 2 * pages) * c["kv_heads"] * c["dk"] * size, "flops": 2 * tokens * c["kv_heads"] * c["dk"]}
    rows = c["heads"] * (c["dk"] + c["dv"]) * size + (c["heads"] * size if c["gate"] else 0)
    token = c["kv_heads"] * (c["dk"] + c["dv"]) * size
    if op == "shared":
        slots, prefix, lens = members_of(c)
        seen = [n - (n - 1) // c["chunk"] * c["chunk"] if c["chunk"] else n for n in lens]      # keys that each sequence sees
        first = [n - s for n, s in zip(lens, seen)]
        once = sum(max(0, p - min(first[i] for i in m)) for m, p in zip(slots, prefix))
        rest = sum(n - max(first[i], p) for m, p in zip(slots, prefix) for i, n in ((i, lens[i]) for i in m))
        return {"bytes": (once + rest) * token + len(lens) * rows, "flops": 2 * c["heads"] * (c["dk"] + c["dv"]) * sum(seen)}
    n_bytes = flops = 0
    for n in lens_of(c):
        n_pages = pages_of(n)
        taken = min(n_pages, c["top"])
        tokens = (taken - 1) * PAGE + (n - 1) % PAGE + 1
        scored = n_pages - min(n_pages, c["first"] + c["last"]) if n_pages > c["top"] else 0
        n_bytes += tokens * token + scored * 2 * c["kv_heads"] * c["dk"] * size + rows
        flops += 2 * c["heads"] * (c["dk"] + c["dv"]) * tokens + 4 * c["heads"] * c["dk"] * scored
    return {"bytes": n_bytes, "flops": flops}


# ---- inputs ----------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed((seed * 0x9E3779B1 + 12345) & 0x7FFFFFFF)
    state = {"copy": prepare_copy, "bounds": prepare_bounds, "shared": prepare_shared, "sparse": prepare_sparse}[case["op"]](case, g)
    state["case"] = case
    if own:
        keep(state)
    return state


def normal(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device=DEVICE, dtype=dtype)


def prepare_copy(c, g):
    n = 2 * c["pages"] + 5
    record = c["kv_heads"] * PAGE * (c["dk"] + c["dv"])
    layers = [normal(g, n, record, dtype=TYPES[c["dtype"]]) for _ in range(c["layers"])]
    order = torch.randperm(n, generator=g, device=DEVICE).to(torch.int32).cpu()
    return {"layers": layers, "src": order[:c["pages"]].tolist(), "dst": order[c["pages"]:2 * c["pages"]].tolist()}


def cache_of(c, g, counts, spare=3):
    """a cache of random records and the page table of sequences with ``counts`` pages; the rest of a row names the last page"""
    n = sum(counts) + spare
    data = normal(g, n, c["kv_heads"] * PAGE * (c["dk"] + c.get("dv", c["dk"])), dtype=TYPES[c["dtype"]])
    order = torch.randperm(n - 1, generator=g, device=DEVICE).to(torch.int32).cpu()
    table, at = torch.full((len(counts), max(counts)), n - 1, dtype=torch.int32), 0
    for i, k in enumerate(counts):
        table[i, :k] = order[at:at + k]
        at += k
    return data, table


def prepare_bounds(c, g):
    first, end = spans_of(c)
    data, table = cache_of(c, g, [pages_of(e) for e in end])
    ints = torch.tensor([first, end], dtype=torch.int32, device=DEVICE)
    out = torch.zeros((data.shape[0], c["kv_heads"], 2, c["dk"]), dtype=data.dtype, device=DEVICE)
    return {"data": data, "table": table.to(DEVICE), "starts": ints[0], "ends": ints[1], "longest": max(e - a for a, e in zip(first, end)), "bounds": out}


def rows_of(c, g, n):
    dt = TYPES[c["dtype"]]
    return {"sink": normal(g, c["heads"]) if c["sink"] else None, "gate": normal(g, n, c["heads"], dtype=dt) if c["gate"] else None,
            "scale": c["dk"] ** -0.5, "out": torch.empty((n, c["heads"] * c["dv"]), dtype=dt, device=DEVICE)}


def prepare_shared(c, g):
    slots, prefix, lens = members_of(c)
    group = {i: k for k, m in enumerate(slots) for i in m}
    data, table = cache_of(c, g, [prefix[k] // PAGE for k in range(len(slots))] + [pages_of(n - prefix[group[i]]) for i, n in enumerate(lens)])
    full = torch.full((len(lens), max(pages_of(n) for n in lens)), data.shape[0] - 1, dtype=torch.int32)
    for i, n in enumerate(lens):
        k = prefix[group[i]] // PAGE
        full[i, :k] = table[group[i], :k]
        full[i, k:pages_of(n)] = table[len(slots) + i, :pages_of(n) - k]
    return {"data": data, "table": full.to(DEVICE), "q": normal(g, len(lens), c["heads"] * c["dk"], dtype=data.dtype), "slots": slots, "prefix": prefix,
            "lens": torch.tensor(lens, dtype=torch.int32, device=DEVICE), "longest": max(lens), **rows_of(c, g, len(lens))}


def prepare_sparse(c, g):
    """Keys of a page resemble one another and a query looks for a few pages, as where leaving pages out is worth while."""
    lens = lens_of(c)
    data, table = cache_of(c, g, [pages_of(n) for n in lens])
    keys = keys_of(data, c)
    center = normal(g, keys.shape[0], c["kv_heads"], 1, c["dk"], dtype=data.dtype)
    keys.mul_(0.45).add_(center, alpha=0.9)
    n, per = len(lens), c["heads"] // c["kv_heads"]
    table = table.to(DEVICE)
    counts = torch.tensor([pages_of(k) for k in lens], device=DEVICE)
    places = (torch.rand((n, c["kv_heads"], 4), generator=g, device=DEVICE) * counts[:, None, None]).long()
    found = torch.gather(table[:, None].expand(-1, c["kv_heads"], -1), 2, places).long()
    wanted = center[found, torch.arange(c["kv_heads"], device=DEVICE)[None, :, None], 0].float().sum(2) / 2
    q = 3 * wanted[:, :, None] + normal(g, n, c["kv_heads"], per, c["dk"])
    kept = torch.stack([keys.amin(2), keys.amax(2)], 2)
    ints = torch.tensor([k - 1 for k in lens], dtype=torch.int32, device=DEVICE)
    return {"data": data, "table": table, "q": q.reshape(n, -1).to(data.dtype), "positions": ints, "bounds": kept, **rows_of(c, g, n)}


def keys_of(data, c):
    """[pages][kv_heads][16][dk] view of the records"""
    return data[:, :c["kv_heads"] * PAGE * c["dk"]].unflatten(1, (c["kv_heads"], PAGE, c["dk"]))


def values_of(data, c):
    return data[:, c["kv_heads"] * PAGE * c["dk"]:].unflatten(1, (c["kv_heads"], PAGE, c["dv"]))


# ---- one pass ----------------------------------------------------------------------------------------------------------------------
def run(state):
    if own:
        return call(state)
    return {"copy": plain_copy, "bounds": plain_bounds, "shared": plain_shared, "sparse": plain_sparse}[state["case"]["op"]](state, state["case"])


def keep(s):
    """What a serving program keeps from step to step: the description of its cache and the plan of who shares what."""
    from mojo_linuxperiments_b200.ops import attention as A
    c = s["case"]
    if c["op"] in ("copy",):
        return
    dv = c.get("dv", c["dk"])
    s["cache"] = A.PagedKVCache(s["data"].shape[0], c["kv_heads"], PAGE, DEVICE, storage=s["data"], dk=c["dk"], dv=dv)
    if c["op"] == "shared":
        from mojo_linuxperiments_b200.ops import shared as SH
        s["plan"] = SH.SharedPrefixes(s["lens"].numel(), DEVICE)
        s["plan"].set(list(zip(s["slots"], s["prefix"])))


def call(s):
    from mojo_linuxperiments_b200.ops import attention as A
    from mojo_linuxperiments_b200.ops import pages as PG
    c = s["case"]
    if c["op"] == "copy":
        PG.copy_pages(s["layers"], s["src"], s["dst"])
        return s["layers"]
    if c["op"] == "bounds":
        return PG.page_bounds(s["cache"], s["table"], s["starts"], s["ends"], None, s["longest"], s["bounds"])
    spec = A.attn_spec(s["scale"], chunk=c.get("chunk"), sink=s["sink"], gate=s["gate"])
    if c["op"] == "shared":
        from mojo_linuxperiments_b200.ops import shared as SH
        return SH.attn_decode_shared(s["q"], c["heads"], s["lens"], s["cache"], s["table"], s["plan"], spec, s["out"])
    from mojo_linuxperiments_b200.ops import sparse as SP
    return SP.attn_paged_sparse(s["q"], c["heads"], s["positions"], None, s["cache"], s["table"], s["bounds"], spec, s["out"], top=c["top"],
                                first=c["first"], last=c["last"])


def plain_copy(s, c):
    index = torch.tensor([s["src"], s["dst"]], device=DEVICE)
    for layer in s["layers"]:
        layer[index[1]] = layer[index[0]]
    return s["layers"]


def plain_bounds(s, c):
    first, ends = (s["starts"] // PAGE).long(), s["ends"].long()
    n = (s["longest"] + 2 * PAGE - 2) // PAGE
    place = first[:, None] + torch.arange(n, device=DEVICE)                                    # [portion][page]
    portion, at = torch.nonzero(place * PAGE < ends[:, None], as_tuple=True)
    place = place[portion, at]
    page = s["table"][portion, place].long()
    k = keys_of(s["data"], c)[page].float()
    gone = (place[:, None] * PAGE + torch.arange(PAGE, device=DEVICE) >= ends[portion, None])[:, None, :, None]
    s["bounds"][page] = torch.stack([k.masked_fill(gone, math.inf).amin(2), k.masked_fill(gone, -math.inf).amax(2)], 2).to(s["bounds"].dtype)
    return s["bounds"]


def softmax_parts(scores, sink, per):
    """weights of the pieces of a softmax over the last axis, [..., kv_heads, per, keys] each; ``sink``: one more exponent per head"""
    top = scores[0].amax(-1, keepdim=True)
    for x in scores[1:]:
        top = torch.maximum(top, x.amax(-1, keepdim=True))
    if sink is not None:
        sink = sink.reshape(-1, per, 1)
        top = torch.maximum(top, sink)
    e = [torch.exp(x - top) for x in scores]
    total = sum(x.sum(-1, keepdim=True) for x in e) + (torch.exp(sink - top) if sink is not None else 0)
    return [x / total for x in e]


def finish(o, s, n):
    """[n, kv_heads, per, dv] -> rows, behind the gate"""
    o = o.reshape(n, s["case"]["heads"], s["case"]["dv"])
    if s["gate"] is not None:
        o = o * torch.sigmoid(s["gate"].float())[..., None]
    return o.reshape(n, -1).to(s["out"].dtype)


def plain_shared(s, c):
    n, hkv, per = s["lens"].numel(), c["kv_heads"], c["heads"] // c["kv_heads"]
    widest, longest = max(len(m) for m in s["slots"]), max(s["prefix"])
    padded = torch.tensor([m + [m[0]] * (widest - len(m)) for m in s["slots"]], device=DEVICE)          # [group][member]
    place = torch.tensor([[g, i, b] for g, m in enumerate(s["slots"]) for i, b in enumerate(m)], device=DEVICE)
    group = torch.empty(n, dtype=torch.long, device=DEVICE)
    within = torch.empty(n, dtype=torch.long, device=DEVICE)
    group[place[:, 2]], within[place[:, 2]] = place[:, 0], place[:, 1]
    prefix = torch.tensor(s["prefix"], device=DEVICE)
    lens = s["lens"].long()
    q = s["q"].float().view(n, hkv, per, c["dk"]) * s["scale"]
    keys, values = keys_of(s["data"], c), values_of(s["data"], c)

    def gathered(x, table):             # [r][kv_heads][tokens][d]
        return x[table.long()].transpose(1, 2).flatten(2, 3).float()

    once = s["table"][padded[:, 0], :longest // PAGE]
    # prefixes: the rows of a group's members against its keys
    qg = q[padded].permute(0, 2, 1, 3, 4).flatten(2, 3)                                                # [group][kv_heads][member x per][dk]
    sg = (qg @ gathered(keys, once).transpose(2, 3)).unflatten(2, (widest, per)).transpose(1, 2)      # [group][member][kv_heads][per][key]
    s1 = sg[group, within]
    # what is a sequence's own
    most = pages_of(int(s["longest"]))
    at = (prefix[group] // PAGE)[:, None] + torch.arange(max(1, min(most, pages_of(c["rest"]))), device=DEVICE)
    rest = torch.gather(s["table"], 1, at.clamp(max=s["table"].shape[1] - 1))
    s2 = q @ gathered(keys, rest).transpose(2, 3)
    low = (lens - 1) // c["chunk"] * c["chunk"] if c["chunk"] else torch.zeros_like(lens)

    def hidden(pos, end):
        return ((pos < low[:, None]) | (pos >= end[:, None]))[:, None, None]
    pos1 = torch.arange(longest, device=DEVICE)[None].expand(n, -1)
    pos2 = prefix[group][:, None] + torch.arange(s2.shape[-1], device=DEVICE)
    s1 = s1.masked_fill(hidden(pos1, torch.minimum(prefix[group], lens)), -math.inf)
    s2 = s2.masked_fill(hidden(pos2, lens), -math.inf)
    p1, p2 = softmax_parts([s1, s2], s["sink"], per)
    pg = p1[padded].transpose(1, 2).flatten(2, 3)
    og = (pg @ gathered(values, once)).unflatten(2, (widest, per)).transpose(1, 2)[group, within]
    # a page behind the end may hold anything: its weight is zero, and so is its part
    v2 = gathered(values, rest).masked_fill((pos2 >= lens[:, None])[:, None, :, None], 0.0)
    return finish(og + p2 @ v2, s, n)


def plain_sparse(s, c):
    n, hkv, per = s["positions"].numel(), c["kv_heads"], c["heads"] // c["kv_heads"]
    pos = s["positions"].long()
    last = pos // PAGE
    q = s["q"].view(n, hkv, per, c["dk"])
    # the largest product that a key within the bounds could have, of any head of the group; in 64 bits, since a border may be narrow
    q64 = q.double()
    b = s["bounds"][s["table"].long()].permute(0, 2, 3, 4, 1).double()                       # [row][kv_heads][2][dk][page]
    score = (q64.clamp(min=0) @ b[:, :, 1] + q64.clamp(max=0) @ b[:, :, 0]).amax(2)
    at = torch.arange(score.shape[-1], device=DEVICE)
    always = (at < c["first"]) | (at > (last - c["last"])[:, None])
    score = torch.where(always[:, None], math.inf, score).masked_fill((at > last[:, None])[:, None], -math.inf)
    chosen = torch.sort(score, dim=-1, descending=True, stable=True)[1][..., :c["top"]]          # [row][kv_heads][pages taken]
    page = torch.gather(s["table"].long()[:, None].expand(-1, hkv, -1), 2, chosen)
    head = torch.arange(hkv, device=DEVICE)[None, :, None]
    seen = (chosen[..., None] * PAGE + torch.arange(PAGE, device=DEVICE) <= pos[:, None, None, None]).flatten(2)
    k = keys_of(s["data"], c)[page, head].flatten(2, 3).float()
    scores = (q.float() * s["scale"]) @ k.transpose(2, 3)
    p, = softmax_parts([scores.masked_fill(~seen[:, :, None], -math.inf)], s["sink"], per)
    v = values_of(s["data"], c)[page, head].flatten(2, 3).float().masked_fill(~seen[..., None], 0.0)
    return finish(p @ v, s, n)


# ---- the definition in 64 bits --------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["op"] == "copy":               # nothing is computed
        out = [x.clone() for x in s["layers"]]
        for x, y in zip(out, s["layers"]):
            for a, b in zip(s["src"], s["dst"]):
                x[b] = y[a]
        return out
    if c["op"] == "bounds":
        out = s["bounds"].double()
        table, data = s["table"].tolist(), keys_of(s["data"], c)
        for i, (a, e) in enumerate(zip(s["starts"].tolist(), s["ends"].tolist())):
            pages = torch.tensor(table[i][a // PAGE:pages_of(e)], device=DEVICE)
            k = data[pages].transpose(1, 2).flatten(0, 1)[:e - a // PAGE * PAGE].double()       # [token][head][dk]
            full = k.shape[0] // PAGE * PAGE
            if full:
                grouped = k[:full].unflatten(0, (-1, PAGE))
                out[pages[:full // PAGE], :, 0], out[pages[:full // PAGE], :, 1] = grouped.min(1).values, grouped.max(1).values
            if full < k.shape[0]:
                out[pages[-1], :, 0], out[pages[-1], :, 1] = k[full:].min(0).values, k[full:].max(0).values
        return out
    rows = []
    per = c["heads"] // c["kv_heads"]
    K, V = keys_of(s["data"], c), values_of(s["data"], c)
    lens = s["lens"].tolist() if c["op"] == "shared" else [p + 1 for p in s["positions"].tolist()]
    for i, n in enumerate(lens):
        pages = s["table"][i, :pages_of(n)].long()
        heads = []
        for h in range(c["kv_heads"]):
            q = s["q"][i].view(c["heads"], c["dk"])[h * per:(h + 1) * per].double()
            low, taken = 0, None
            if c["op"] == "shared":
                low = (n - 1) // c["chunk"] * c["chunk"] if c["chunk"] else 0
            else:
                lo, hi = s["bounds"][pages, h, 0].double(), s["bounds"][pages, h, 1].double()
                score = torch.maximum(q[:, None] * lo, q[:, None] * hi).sum(-1).max(0).values if len(pages) <= 2048 else torch.cat(
                    [torch.maximum(q[:, None] * x, q[:, None] * y).sum(-1).max(0).values for x, y in zip(lo.split(2048), hi.split(2048))])
                score[:c["first"]] = math.inf
                score[max(0, len(pages) - c["last"]):] = math.inf
                taken = torch.sort(score, descending=True, stable=True).indices[:c["top"]].sort().values
            token = torch.arange(low, n, device=DEVICE)
            if taken is not None:
                token = (taken[:, None] * PAGE + torch.arange(PAGE, device=DEVICE)).flatten()
                token = token[token < n]
            page, off = pages[token // PAGE], token % PAGE
            x = (q @ K[page, h, off].double().t()) * s["scale"]
            if s["sink"] is not None:
                x = torch.cat([x, s["sink"][h * per:(h + 1) * per].double()[:, None]], 1)
            w = torch.softmax(x, -1)[:, :len(token)]
            heads.append(w @ V[page, h, off].double())
        o = torch.cat(heads)
        if s["gate"] is not None:
            o = o / (1 + torch.exp(-s["gate"][i].double()))[:, None]
        rows.append(o.flatten())
    return torch.stack(rows)
