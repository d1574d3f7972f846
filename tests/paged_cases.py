"""Sequences in a paged cache for tests of what reads it, and the plain definitions in 64 bits.

Whatever a sequence does not hold is NaN, so that a key or value read from behind an end shows."""
import math

import torch

DEV = "cuda"
PAGE = 16
DT = {"float32": torch.float32, "bfloat16": torch.bfloat16}
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


class Sequences:
    """``lens`` tokens per slot; ``groups``: (slots, shared tokens) with the same pages in front."""

    def __init__(self, lens, hq, hkv, dk, dv, dtype, *, groups=(), seed=0, spread=1.0, spare=2, ps=PAGE):
        from mojo_linuxperiments_b200.ops import attention as A
        self.lens, self.hq, self.hkv, self.dk, self.dv, self.dtype, self.ps = list(lens), hq, hkv, dk, dv, DT[dtype], ps
        g = self.g = torch.Generator(device=DEV).manual_seed(seed)
        prefix = {s: (i, t) for i, (slots, t) in enumerate(groups) for s in slots}
        need = [max(0, -(-n // ps) - (prefix[i][1] // ps if i in prefix else 0)) for i, n in enumerate(lens)]
        total = sum(need) + sum(t // ps for _, t in groups)
        order = torch.randperm(total + spare, generator=torch.Generator().manual_seed(seed)).tolist()
        shared = [[order.pop() for _ in range(t // ps)] for _, t in groups]
        rows = [(shared[prefix[i][0]] if i in prefix else []) + [order.pop() for _ in range(k)] for i, k in enumerate(need)]
        self.rows = rows
        self.width = max(1, max(len(r) for r in rows))
        table = torch.full((len(lens), self.width), order[0], dtype=torch.int32)         # a page that nobody owns
        for i, r in enumerate(rows):
            table[i, :len(r)] = torch.tensor(r, dtype=torch.int32)
        self.table = table.to(DEV)
        self.cache = A.PagedKVCache(total + spare, hkv, ps, DEV, dk=dk, dv=dv, dtype=self.dtype)
        self.cache.data.fill_(float("nan"))
        held = {}
        for r, n in zip(rows, lens):
            for at, p in enumerate(r):
                held[p] = max(held.get(p, 0), min(ps, n - at * ps))
        for i, (slots, t) in enumerate(groups):
            for p in shared[i]:
                held[p] = ps
        K, V = self.cache.keys(), self.cache.values()
        for p, n in held.items():
            if n > 0:
                K[p, :, :n] = (torch.randn((hkv, n, dk), generator=g, device=DEV) * spread).to(self.dtype)
                V[p, :, :n] = torch.randn((hkv, n, dv), generator=g, device=DEV).to(self.dtype)

    def rows_of(self, n, pitch=0):
        """q rows with a pitch, whatever lies between them is NaN"""
        w = self.hq * self.dk
        q = torch.full((n, w + pitch), float("nan"), dtype=self.dtype, device=DEV)
        q[:, :w] = torch.randn((n, w), generator=self.g, device=DEV).to(self.dtype)
        return q

    def heads_of(self, n, sink=True, gate=True):
        s = torch.randn(self.hq, generator=self.g, device=DEV) if sink else None
        wide = torch.randn((n, self.hq + 3), generator=self.g, device=DEV).to(self.dtype)
        return s, wide[:, :self.hq] if gate else None

    def tokens(self, seq, places):
        """fp64 keys [hkv][n][dk] and values of the given positions"""
        pages = torch.tensor([self.rows[seq][p // self.ps] for p in places], device=DEV)
        at = torch.tensor([p % self.ps for p in places], device=DEV)
        return self.cache.keys()[pages, :, at].double().transpose(0, 1), self.cache.values()[pages, :, at].double().transpose(0, 1)

    def want(self, q, row, seq, places, scale, sink, gate, heads=None):
        """Output of one row over the keys at ``places`` (a list, or one per KV head), and how far off it may be.

        Scores: products are exact in fp32, their sum of dk terms is off by (dk + 8) 2^-24 of the terms' absolute sum, and so, doubled (numerator and
        denominator), are the weights.  Weights that are rounded to the type are off by its half step each, in the numerator and in the denominator; sums of
        n weights by n 2^-24 at most; exponentials and the gate by 2^-20; the result by another half step."""
        per, half = self.hq // self.hkv, HALF_STEP[self.dtype]
        out, tol = [], []
        for h in range(self.hkv):
            mine = places[h] if places and isinstance(places[0], list) else places
            qh = q[row, :self.hq * self.dk].double().view(self.hq, self.dk)[h * per:(h + 1) * per]
            k, v = (x[h] for x in self.tokens(seq, mine)) if mine else (qh.new_zeros((0, self.dk)), qh.new_zeros((0, self.dv)))
            s = qh @ k.t() * scale
            off = (self.dk + 8) * 2.0 ** -24 * float((qh.abs() @ k.abs().t() * scale).max()) if mine else 0.0
            if sink is not None:
                s = torch.cat([s, sink[h * per:(h + 1) * per].double()[:, None]], 1)
            w = torch.softmax(s, 1)[:, :len(mine)] if s.shape[1] else s
            o, a = w @ v, w @ v.abs()
            weights = 2 * half if self.dtype != torch.float32 else 0.0
            f = torch.sigmoid(gate[row, h * per:(h + 1) * per].double())[:, None] if gate is not None else 1.0
            out.append(o * f)
            tol.append((half * o.abs() + (weights + 2 * off + 2.0 ** -18 + len(mine) * 2.0 ** -24 * 2) * a) * f + 1e-30)
        return torch.cat(out).flatten(), torch.cat(tol).flatten()


def worst(got, want, tol):
    """largest error over what is allowed; infinite where a result is not finite"""
    got = got.double()
    if not torch.isfinite(got).all():
        return math.inf
    return float(((got - want).abs() / tol).max()) if got.numel() else 0.0


def status_ok():
    from mojo_linuxperiments_b200.ops.workspace import default_workspace
    default_workspace(torch.device(DEV)).check_status()
