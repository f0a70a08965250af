"""A paged cache and its operators written out in float64 with loops, and caches to test with."""
import math

import torch

F64 = torch.float64


class Cache:
    """Pages with every slot that is not in use, and every page that no table names, full of NaN."""

    def __init__(self, lens, n_kv_heads, dim, page, dtype, seed=0, layout="rows", spare=1, device="cuda", missing=()):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.page, self.hk, self.dim, self.dtype = list(lens), page, n_kv_heads, dim, dtype
        n = len(lens)
        self.wide = max([-(-x // page) for x in lens] + [0]) + spare
        pages = n * self.wide + 1
        order = torch.randperm(pages, generator=g)[:n * self.wide].reshape(n, self.wide)
        self.table = order.to(torch.int32)
        for s, i in missing:
            self.table[s, i] = -1 if (s + i) % 2 else pages + 5
        if layout == "rows":
            k, v = (torch.full((pages, page, n_kv_heads, dim), math.nan, dtype=dtype) for _ in range(2))
        elif layout == "interleaved":  # keys and values of a page in one tensor
            both = torch.full((pages, 2, page, n_kv_heads, dim), math.nan, dtype=dtype)
            k, v = both[:, 0], both[:, 1]
        else:  # heads ahead of slots, the values' rows wider than they need be
            k = torch.full((pages, n_kv_heads, page, dim), math.nan, dtype=dtype).transpose(1, 2)
            v = torch.full((pages, n_kv_heads, page, dim + 32), math.nan, dtype=dtype).transpose(1, 2)[..., :dim]
        for s, x in enumerate(self.lens):
            for j in range(x):
                p = int(self.table[s, j // page])
                if 0 <= p < pages:
                    k[p, j % page] = torch.randn(n_kv_heads, dim, generator=g).to(dtype)
                    v[p, j % page] = torch.randn(n_kv_heads, dim, generator=g).to(dtype)
        self.k, self.v = k, v
        self.pages = pages
        self.capacity = self.wide * page

    def cuda(self):
        import cera_b200 as cb
        if self.k.untyped_storage().data_ptr() == self.v.untyped_storage().data_ptr():
            n = self.k.shape
            both = torch.stack([self.k, self.v], 1).cuda()
            self.kd, self.vd = both[:, 0], both[:, 1]
            assert self.kd.shape == n
        else:
            self.kd, self.vd = self._same(self.k), self._same(self.v)
        self.td, self.ld = self.table.cuda(), torch.tensor(self.lens, dtype=torch.int32).cuda()
        return cb.PagedKv(self.kd, self.vd, self.td, self.ld)

    @staticmethod
    def _same(t):  # on the GPU in the same strides
        d = torch.full((t.untyped_storage().nbytes() // t.element_size(),), math.nan, dtype=t.dtype, device="cuda").as_strided(t.shape, t.stride())
        return d.copy_(t)

    def slot(self, s, j):
        """(page, row) of a slot; None where there is no page."""
        p = int(self.table[s, j // self.page])
        return (p, j % self.page) if 0 <= p < self.pages else None

    def seen(self, s, p, window, sink):
        return [j for j in range(p + 1) if (not window or j < sink or j > p - window) and self.slot(s, j) is not None]


def attend(c, s, p, q, scale, window=0, sink=0):
    """Query heads q [heads][dim] in slot p -> (result, bound on the sum of p |v|, largest scale * sum |q k|, probabilities {slot: [heads]})."""
    heads = q.shape[0]
    js = c.seen(s, p, window, sink)
    if not js:
        z = torch.zeros(heads, c.dim, dtype=F64)
        return z, z, 0.0, [], torch.zeros(heads, 0, dtype=F64)
    at = [c.slot(s, j) for j in js]
    pg, rw = torch.tensor([a[0] for a in at]), torch.tensor([a[1] for a in at])
    k, v = c.k[pg, rw].double(), c.v[pg, rw].double()  # [slots][kv heads][dim]
    g = heads // c.hk
    kk, vv = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    z = torch.einsum("hd,jhd->hj", q.double(), kk) * scale
    e = torch.exp(z - z.amax(-1, keepdim=True))
    w = e / e.sum(-1, keepdim=True)
    size = float((torch.einsum("hd,jhd->hj", q.double().abs(), kk.abs()) * abs(scale)).max())
    return torch.einsum("hj,jhd->hd", w, vv), torch.einsum("hj,jhd->hd", w, vv.abs()), size, js, w


def tolerance(want, p_v, size, n, dim, q_dtype, kv_dtype):
    """What f32 arithmetic may be off by, worst case.  u = 2^-24.  A score: dim products, each off by u of the sum of their sizes, and its scaling by two
    roundings; numerator and denominator each take that much, so twice.  The exponential: 2^-22 and the rounding of its argument (4 u of the score's
    size, counted there).  Sums over n slots, of the weights and of the weighted values: n u each, and the rescalings as much again.  Queries and weights in 16-bit
    parts: 2^-21.  With 16-bit queries the weight of a slot is rounded once to the cache's type.  The result is rounded to q's type."""
    u = 2.0 ** -24
    rel = 2 * (dim + 6) * u * max(size, 1.0) + 4 * n * u + 2.0 ** -22 + 2.0 ** -21
    if q_dtype != torch.float32:
        rel += torch.finfo(kv_dtype).eps / 2
    tiny = 0.0 if q_dtype == torch.float32 else float(torch.finfo(q_dtype).smallest_normal) * torch.finfo(q_dtype).eps
    return torch.finfo(q_dtype).eps / 2 * (want.abs() + rel * p_v) + rel * p_v + tiny


def check(got, want, tol, what):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (got.shape, want.shape)
    assert torch.isfinite(got).all(), f"{what}: not finite"
    off = (got - want).abs() - tol
    assert (off <= 0).all(), f"{what}: {int((off > 0).sum())} of {off.numel()} outside, by {float(off.max()):.3e}"


def evict(c, weights, positions, budget, n_sink, n_recent):
    """weights, positions [seqs][kv heads][slots] (lists are fine) -> kept [seqs][kv heads][budget]."""
    kept = torch.full((len(c.lens), c.hk, budget), -1, dtype=torch.int32)
    for s, x in enumerate(c.lens):
        for h in range(c.hk):
            w, pos = weights[s, h, :x].tolist(), positions[s, h, :x].tolist()
            row = list(range(min(x, budget)))
            if x > budget:
                newest = max(pos)
                safe = [p < n_sink or p > newest - n_recent for p in pos]
                rank = [math.inf if ok else (-math.inf if wt != wt else wt) for wt, ok in zip(w, safe)]
                nan_below = [0 if wt == wt or ok else 1 for wt, ok in zip(w, safe)]
                best = set(sorted(range(x), key=lambda j: (not safe[j], nan_below[j], -rank[j], j))[:budget])
                movers = iter(sorted(j for j in best if j >= budget))
                row = [j if j in best else next(movers) for j in range(budget)]
            kept[s, h, :len(row)] = torch.tensor(row, dtype=torch.int32)
    return kept
