"""The paged cache's operators against the formulas in float64."""
import math

import pytest
import torch

import paged_ref as R
from gpu_util import need_gpu

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [(F32, F32), (F32, F16), (F32, BF16), (F16, F16), (BF16, BF16)]  # queries, cache
SHAPES = [(8, 2, 128), (1, 1, 32), (15, 3, 64), (7, 1, 96), (40, 2, 64), (4, 4, 256), (12, 4, 160), (9, 1, 128)]


def _q(n, heads, dim, dtype, seed=1, size=1.5):
    return (torch.randn(n, heads, dim, generator=torch.Generator().manual_seed(seed)) * size).to(dtype)


def _decode_case(cb, c, heads, q_dtype, window=0, sink=0, weights=False, seed=1, size=1.5, **kw):
    cache = c.cuda()
    q = _q(len(c.lens), heads, c.dim, q_dtype, seed, size)
    scale = 1.0 / math.sqrt(c.dim)
    w = torch.rand(len(c.lens), c.hk, c.capacity) if weights else None
    wd = w.cuda() if weights else None
    got = cb.paged_decode_attention(cache, q.cuda(), scale, window=window, n_sink=sink, weights=wd, **kw)
    assert got.dtype == q_dtype
    for s, x in enumerate(c.lens):
        want, pv, size_s, js, p = R.attend(c, s, x - 1, q[s], scale, window, sink)
        tol = R.tolerance(want, pv, size_s, len(js), c.dim, q_dtype, c.dtype)
        R.check(got[s], want, tol, f"sequence {s} of {x}")
        if weights:
            add = torch.zeros(c.hk, c.capacity, dtype=R.F64)
            add[:, js] = p.reshape(c.hk, heads // c.hk, -1).sum(1)
            rel = 2 * (c.dim + 6) * 2.0 ** -24 * max(size_s, 1.0) + 4 * len(js) * 2.0 ** -24 + 2.0 ** -21 + heads // c.hk * 2.0 ** -24
            R.check(wd[s], w[s].double() + add, rel * add + 2.0 ** -24 * (w[s].double() + add) + 1e-30, f"weights of sequence {s}")


@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_decode(types, shape):
    need_gpu()
    import cera_b200 as cb
    heads, hk, dim = shape
    _decode_case(cb, R.Cache([5, 0, 1, 64, 65, 200, 31], hk, dim, 16, types[1], seed=heads), heads, types[0])


@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("window,sink", [(1, 0), (1, 3), (16, 4), (40, 0), (64, 64), (500, 4), (37, 1)])
def test_decode_window(types, window, sink):
    need_gpu()
    import cera_b200 as cb
    _decode_case(cb, R.Cache([1, 2, 0, 17, 100, 300, 41], 2, 64, 16, types[1], seed=window), 6, types[0], window, sink)


@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 64, 1000])
@pytest.mark.parametrize("layout", ["rows", "interleaved", "heads first"])
def test_decode_layouts(page, layout):
    need_gpu()
    import cera_b200 as cb
    for q, kv in [(F32, F32), (F32, F16), (BF16, BF16)]:
        _decode_case(cb, R.Cache([9, 130, 64, 200], 2, 64, page, kv, seed=page, layout=layout), 8, q)


@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("window,sink", [(0, 0), (50, 4)])
def test_decode_adds_weights(types, window, sink):
    need_gpu()
    import cera_b200 as cb
    _decode_case(cb, R.Cache([1, 90, 0, 700, 64, 33], 3, 64, 16, types[1], seed=5), 12, types[0], window, sink, weights=True)


@pytest.mark.parametrize("types", TYPES, ids=str)
def test_decode_long_and_split(types):
    """Few rows over many slots, and large scores: the parts of a sequence are joined."""
    need_gpu()
    import cera_b200 as cb
    _decode_case(cb, R.Cache([5000, 3], 1, 128, 16, types[1], seed=2), 4, types[0], weights=True)
    _decode_case(cb, R.Cache([2999], 2, 64, 32, types[1], seed=3), 16, types[0], size=30.0)


@pytest.mark.parametrize("types", TYPES, ids=str)
def test_missing_pages_are_not_seen(types):
    need_gpu()
    import cera_b200 as cb
    c = R.Cache([100, 40, 16, 200], 2, 64, 16, types[1], seed=4, missing=[(0, 1), (0, 6), (2, 0), (3, 4), (3, 5)])
    _decode_case(cb, c, 4, types[0], weights=True)
    _prefill_case(cb, c, 4, types[0], [30, 40, 16, 5])


def test_many_short_sequences():
    need_gpu()
    import cera_b200 as cb
    lens = [(7 * i) % 23 for i in range(300)]
    _decode_case(cb, R.Cache(lens, 2, 64, 8, F16, seed=6), 4, F16, weights=True)


def test_lengths_out_of_range_count_as_the_nearer_end():
    need_gpu()
    import cera_b200 as cb
    c = R.Cache([48, 20], 2, 64, 16, F16, seed=7, spare=0)
    cache = c.cuda()
    q = _q(2, 4, 64, F16).cuda()
    want = cb.paged_decode_attention(cache, q, 0.125)
    c.ld.copy_(torch.tensor([10 ** 6, -3]))
    got = cb.paged_decode_attention(cache, q, 0.125)
    assert torch.equal(got[0], want[0]) and not got[1].any()


def _prefill_case(cb, c, heads, q_dtype, new, window=0, sink=0, behind=3, seed=2, size=1.5):
    """The last new[s] slots of every sequence ask; `behind` rows of padding follow."""
    cache = c.cuda()
    n = sum(new)
    q = _q(n + behind, heads, c.dim, q_dtype, seed, size)
    starts = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32)
    scale = 1.0 / math.sqrt(c.dim)
    out = torch.full_like(q, 7.0).cuda()
    got = cb.paged_prefill_attention(cache, q.cuda(), starts.cuda(), scale, window=window, n_sink=sink, out=out)
    assert got is out and (out[n:] == 7.0).all()
    for s, (m, x) in enumerate(zip(new, c.lens)):
        for i in range(m):
            t = int(starts[s]) + i
            want, pv, size_s, js, _ = R.attend(c, s, x - m + i, q[t], scale, window, sink)
            R.check(got[t], want, R.tolerance(want, pv, size_s, len(js), c.dim, q_dtype, c.dtype), f"sequence {s}, query {i} of {m} at {x}")


@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_prefill(types, shape):
    need_gpu()
    import cera_b200 as cb
    heads, hk, dim = shape
    _prefill_case(cb, R.Cache([70, 1, 33, 0, 150, 200], hk, dim, 16, types[1], seed=heads), heads, types[0], [70, 1, 0, 0, 17, 3])


@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("window,sink", [(1, 0), (1, 2), (16, 4), (64, 0), (130, 70), (37, 1)])
def test_prefill_window(types, window, sink):
    need_gpu()
    import cera_b200 as cb
    _prefill_case(cb, R.Cache([160, 300, 5], 2, 64, 16, types[1], seed=window), 6, types[0], [160, 40, 5], window, sink)


@pytest.mark.parametrize("page", [1, 3, 24, 1000])
@pytest.mark.parametrize("layout", ["rows", "interleaved", "heads first"])
def test_prefill_layouts(page, layout):
    need_gpu()
    import cera_b200 as cb
    for q, kv in [(F32, F32), (F32, F16), (BF16, BF16)]:
        _prefill_case(cb, R.Cache([50, 130], 2, 64, page, kv, seed=page, layout=layout), 4, q, [50, 20])


@pytest.mark.parametrize("types", TYPES, ids=str)
def test_prefill_long_cache_few_queries(types):
    need_gpu()
    import cera_b200 as cb
    _prefill_case(cb, R.Cache([3000, 2500], 1, 128, 16, types[1], seed=8), 4, types[0], [5, 1])
    _prefill_case(cb, R.Cache([1500], 2, 64, 32, types[1], seed=9), 8, types[0], [40], size=30.0)


@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("dim", [64, 128, 160])
def test_prefill_several_tiles(types, dim):
    """More rows than any tile has, most keys seen by all of them."""
    need_gpu()
    import cera_b200 as cb
    c = R.Cache([700], 1, dim, 64, types[1], seed=10)
    _prefill_case(cb, c, 3, types[0], [300])
    _prefill_case(cb, c, 3, types[0], [300], window=190, sink=5)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=str)
@pytest.mark.parametrize("dim", [64, 128, 224])
@pytest.mark.parametrize("growing", [False, True])
def test_prefill_f32_over_many_slots(dtype, dim, growing):
    """Sums of many slots keep the precision of f32: with values of one sign, cutting a sum at each of its 2500 or 3750 steps by 2^-24 on average would add up to 1e-4.
    Bound, relative to the result's norm: scores of size 4 in dim / 16 <= 14 steps of 2^-23, which enter twice (above and below the line), 1.4e-5; sums of 128 slots in
    24 steps of 2^-23, 2.9e-6; 160 groups in steps of 2^-24 at random signs and parts of 2^-22, 1e-6.
    `growing`: scores that rise along the slots to 64 (2e-4 by the first term), so that the maximum is raised after sums were put aside."""
    need_gpu()
    import cera_b200 as cb
    n, heads, slots, page = 700, 16, 20000, 32
    g = torch.Generator("cuda").manual_seed(dim)
    k = torch.randn(slots // page, page, 2, dim, generator=g, device="cuda")
    if growing:
        k[..., 0] = torch.arange(slots, device="cuda").reshape(-1, page, 1) * (60.0 / slots)
    k, v = k.to(dtype), (torch.rand(slots // page, page, 2, dim, generator=g, device="cuda") + 0.5).to(dtype)
    q = torch.randn(n, heads, dim, generator=g, device="cuda")
    if growing:
        q[..., 0] = math.sqrt(dim)
    table = torch.randperm(slots // page, generator=torch.Generator().manual_seed(1)).to(torch.int32)[None].cuda()
    cache = cb.PagedKv(k, v, table, torch.tensor([slots], dtype=torch.int32, device="cuda"))
    got = cb.paged_prefill_attention(cache, q, torch.tensor([0, n], dtype=torch.int32, device="cuda"), 1.0 / math.sqrt(dim))
    kk, vv = (x[table[0].long()].reshape(slots, 2, dim).double() for x in (k, v))
    hidden = torch.arange(slots, device="cuda") > torch.arange(slots - n, slots, device="cuda")[:, None]
    for h in range(0, heads, 5):
        x = (q[:, h].double() @ kk[:, h // 8].T / math.sqrt(dim)).masked_fill_(hidden, -math.inf)
        want = torch.softmax(x, -1) @ vv[:, h // 8]
        assert float((got[:, h].double() - want).norm() / want.norm()) < (2.2e-4 if growing else 2e-5)


@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("window,sink", [(0, 0), (300, 4)])
def test_prefill_split_keys_of_several_sequences(types, window, sink):
    """Keys split by the capacity, which most sequences stay far below: parts without keys, and rows that see some of them only."""
    need_gpu()
    import cera_b200 as cb
    c = R.Cache([2100, 40, 700, 1, 0], 2, 64, 32, types[1], seed=12)
    _prefill_case(cb, c, 6, types[0], [9, 7, 30, 1, 0], window, sink)


def test_prefill_of_more_tokens_than_are_cached():
    """Queries whose place is before the first slot see nothing."""
    need_gpu()
    import cera_b200 as cb
    c = R.Cache([10], 1, 64, 16, F16, seed=11)
    cache = c.cuda()
    q = _q(14, 2, 64, F16)
    got = cb.paged_prefill_attention(cache, q.cuda(), torch.tensor([0, 14], dtype=torch.int32).cuda(), 0.125).cpu()
    assert not got[:4].any()
    for i in range(4, 14):
        want, pv, size, js, _ = R.attend(c, 0, i - 4, q[i], 0.125)
        R.check(got[i], want, R.tolerance(want, pv, size, len(js), 64, F16, F16), f"query {i}")


@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_values_that_are_not_finite_reach_only_who_sees_them(types, bad):
    need_gpu()
    import cera_b200 as cb
    for spoil_k, spoil_v in ((True, False), (False, True), (True, True)):
        c = R.Cache([200], 2, 64, 16, types[1], seed=12)
        p, r = c.slot(0, 150)
        if spoil_k:
            c.k[p, r, 0, 3] = bad
        if spoil_v:
            c.v[p, r, 0, 5] = bad
        cache = c.cuda()
        q = _q(90, 4, 64, types[0])
        starts = torch.tensor([0, 90], dtype=torch.int32).cuda()
        got = cb.paged_prefill_attention(cache, q.cuda(), starts, 0.125, window=20, n_sink=2).cpu()
        for i in range(90):
            at = 110 + i
            want, pv, size, js, w = R.attend(c, 0, at, q[i], 0.125, 20, 2)
            if 150 in js:
                fine = torch.isfinite(want)
                assert torch.equal(torch.isnan(got[i].double()), torch.isnan(want)), f"query {i}"
                assert torch.equal(got[i].double()[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)])
                got[i] = torch.where(fine, got[i], torch.zeros_like(got[i]))
                want, pv = torch.where(fine, want, 0.0), torch.where(torch.isfinite(pv), pv, 0.0)
                size = size if math.isfinite(size) else 10.0
            R.check(got[i], want, R.tolerance(want, pv, size, len(js), 64, types[0], types[1]), f"query {i}")
        d = cb.paged_decode_attention(cache, q[:1].cuda(), 0.125, window=20, n_sink=2)  # slot 199 does not see 150
        want, pv, size, js, _ = R.attend(c, 0, 199, q[0], 0.125, 20, 2)
        R.check(d[0], want, R.tolerance(want, pv, size, len(js), 64, types[0], types[1]), "decode")


# ---- storing -----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("page,layout,hk,dim", [(16, "rows", 2, 64), (3, "interleaved", 1, 128), (8, "heads first", 5, 96), (64, "rows", 300, 32)])
def test_append(types, page, layout, hk, dim):
    need_gpu()
    import cera_b200 as cb
    c = R.Cache([20, 0, 7, 33, 1], hk, dim, page, types[1], seed=1, layout=layout, missing=[(3, 0)])
    new = [5, 0, 7, 33, 1]
    cache = c.cuda()
    n = sum(new)
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(n + 2, hk, dim, generator=g).to(types[0]) for _ in range(2))
    starts = torch.tensor([0, 5, 5, 12, 45, 46], dtype=torch.int32)
    at = torch.arange(100, 100 + n + 2, dtype=torch.int32)
    w, pos = torch.ones(5, hk, c.capacity + 3), torch.full((5, hk, c.capacity + 3), -9, dtype=torch.int32)
    wd, pd = w.cuda(), pos.cuda()
    cb.paged_append(cache, k.cuda(), v.cuda(), starts.cuda(), weights=wd, positions=pd, token_positions=at.cuda())
    t = 0
    for s, m in enumerate(new):
        for i in range(m):
            j = c.lens[s] - m + i
            w[s, :, j], pos[s, :, j] = 0.0, at[t]
            if c.slot(s, j) is not None:
                p, r = c.slot(s, j)
                c.k[p, r], c.v[p, r] = k[t].to(types[1]), v[t].to(types[1])
            t += 1
    for got, want in ((c.kd, c.k), (c.vd, c.v), (wd, w), (pd, pos)):
        assert torch.equal(got.cpu().contiguous().view(torch.uint8), want.contiguous().view(torch.uint8))


def test_append_one_token_each():
    need_gpu()
    import cera_b200 as cb
    c = R.Cache([20, 0, 7], 2, 64, 16, F16, seed=1)
    cache = c.cuda()
    k, v = torch.randn(3, 2, 64), torch.randn(3, 2, 64)
    pd = torch.zeros(3, 2, c.capacity, dtype=torch.int32).cuda()
    cb.paged_append(cache, k.cuda(), v.cuda(), positions=pd)
    for s, x in enumerate(c.lens):
        if x:
            p, r = c.slot(s, x - 1)
            c.k[p, r], c.v[p, r] = k[s].half(), v[s].half()
            assert (pd[s, :, x - 1] == x - 1).all() and int(pd[s].abs().sum()) == 2 * (x - 1)
    assert torch.equal(c.kd.cpu().view(torch.int16), c.k.view(torch.int16)) and torch.equal(c.vd.cpu().view(torch.int16), c.v.view(torch.int16))


# ---- eviction ----------------------------------------------------------------------------------------------------------

def _evict_case(cb, c, weights, positions, budget, n_sink, n_recent, in_place):
    cache = c.cuda()
    wd, pd = weights.cuda(), positions.cuda()
    wo = po = None
    if not in_place:
        wo, po = torch.full((len(c.lens), c.hk, budget + 2), -5.0).cuda(), torch.full((len(c.lens), c.hk, budget + 2), -5, dtype=torch.int32).cuda()
    kept, lens = cb.paged_evict(cache, wd, pd, budget, n_sink, n_recent, weights_out=wo, positions_out=po, seq_lens_out=c.ld if in_place else None)
    want = R.evict(c, weights, positions, budget, n_sink, n_recent)
    assert torch.equal(kept.cpu(), want)
    assert lens.tolist() == [min(x, budget) for x in c.lens]
    w1, p1 = (weights.clone(), positions.clone()) if in_place else (wo.cpu() * 0 - 5, po.cpu() * 0 - 5)
    k1, v1 = c.k.clone(), c.v.clone()
    for s in range(len(c.lens)):
        for h in range(c.hk):
            for j, src in enumerate(want[s, h].tolist()):
                if src < 0:
                    continue
                w1[s, h, j], p1[s, h, j] = weights[s, h, src], positions[s, h, src]
                a, b = c.slot(s, j), c.slot(s, src)
                if a is not None and b is not None and src != j:
                    k1[a[0], a[1], h], v1[a[0], a[1], h] = c.k[b[0], b[1], h], c.v[b[0], b[1], h]
    got_w, got_p = (wd, pd) if in_place else (wo, po)
    assert torch.equal(got_w.cpu().view(torch.int32), w1.view(torch.int32)) and torch.equal(got_p.cpu(), p1)
    for got, ref in ((c.kd, k1), (c.vd, v1)):
        assert torch.equal(got.cpu().contiguous().view(torch.uint8), ref.contiguous().view(torch.uint8))


def _track(c, seed, ties=False, special=False, mixed=True):
    g = torch.Generator().manual_seed(seed)
    n = (len(c.lens), c.hk, c.capacity)
    w = torch.rand(n, generator=g) * 3
    if ties:
        w = (w * 2).floor()
    if special:
        pick = torch.randint(0, 12, n, generator=g)
        for i, x in enumerate((math.nan, math.inf, -math.inf, 0.0, -0.0, -1.5, 1e-42)):
            w[pick == i] = x
    pos = torch.arange(c.capacity, dtype=torch.int32).expand(n).contiguous()
    if mixed:
        for s, x in enumerate(c.lens):
            for h in range(c.hk):
                pos[s, h, :x] = torch.randperm(x, generator=g).to(torch.int32) * 3
    return w, pos


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=str)
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("ties,special,mixed", [(False, False, False), (True, False, True), (False, True, True)])
def test_evict(dtype, in_place, ties, special, mixed):
    need_gpu()
    import cera_b200 as cb
    for budget, sink, recent in ((16, 2, 5), (16, 0, 0), (16, 10, 6), (40, 4, 20), (1, 0, 1), (95, 4, 8), (200, 4, 8)):
        c = R.Cache([96, 17, 0, 16, 130, 1], 3, 32, 8, dtype, seed=budget, missing=[(4, 0), (4, 15)])
        _evict_case(cb, c, *_track(c, budget, ties, special, mixed), budget, sink, recent, in_place)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("length,budget", [(1025, 1024), (5000, 700), (31000, 4000), (70000, 66000), (70001, 500), (230001, 200000), (430001, 100000)])
def test_evict_long(length, budget, in_place):
    """One CTA, clusters, and lengths whose keys do not fit in their shared memory."""
    need_gpu()
    import cera_b200 as cb
    c = R.Cache([0], 1, 32, 64, F16)
    c.lens, c.wide = [length], -(-length // 64)
    c.pages, c.capacity = c.wide, c.wide * 64
    c.table = torch.randperm(c.wide, generator=torch.Generator().manual_seed(1)).to(torch.int32)[None]
    c.k, c.v = (torch.randn(c.pages, 64, 1, 32, generator=torch.Generator().manual_seed(i)).half() for i in (2, 3))
    _evict_case(cb, c, *_track(c, 5, ties=True), budget, 4, 30, in_place)


# ---- together, streams, graphs, far offsets -----------------------------------------------------------------------------

def _serve(cb, cache, parts, heads, window_layer):
    """A prompt, decode steps that weigh the slots, an eviction in place, more steps: what they return."""
    lens, starts, (qp, kp, vp), steps, weights, positions, budget = parts
    got = []
    lens += starts[1:] - starts[:-1]
    cb.paged_append(cache, kp, vp, starts, weights=weights, positions=positions)
    got.append(cb.paged_prefill_attention(cache, qp, starts, 0.125, window=window_layer, n_sink=2))
    at = lens.clone()
    for i, (q, k, v) in enumerate(steps):
        lens += 1
        cb.paged_append(cache, k, v, weights=weights, positions=positions, token_positions=at)
        got.append(cb.paged_decode_attention(cache, q, 0.125, weights=weights).clone())
        at += 1
        if i == 2:
            cb.paged_evict(cache, weights, positions, budget, n_sink=2, n_recent=8, seq_lens_out=lens)
    return got + [weights.clone(), positions.clone(), lens.clone()]


def _serve_parts(c, heads, q_dtype, seed):
    g = torch.Generator().manual_seed(seed)
    n, hk, dim = len(c.lens), c.hk, c.dim
    new = [60, 0, 33, 90][:n]
    starts = torch.tensor([sum(new[:i]) for i in range(n + 1)], dtype=torch.int32)
    rnd = lambda m, h: torch.randn(m, h, dim, generator=g).to(q_dtype)  # noqa: E731
    prompt = rnd(sum(new), heads), rnd(sum(new), hk), rnd(sum(new), hk)
    steps = [(rnd(n, heads), rnd(n, hk), rnd(n, hk)) for _ in range(6)]
    return new, starts, prompt, steps


def _serve_reference(c, new, starts, prompt, steps, heads, q_dtype, window, budget):
    """The same in float64; yields (result, tolerance) of every attention call."""
    n, hk = len(c.lens), c.hk
    weights, positions = torch.zeros(n, hk, c.capacity, dtype=R.F64), torch.zeros(n, hk, c.capacity, dtype=torch.int32)
    at = list(new)

    def store(s, k, v, pos):
        j = c.lens[s] - 1
        p, r = c.slot(s, j)
        c.k[p, r], c.v[p, r] = k.to(c.dtype), v.to(c.dtype)
        weights[s, :, j], positions[s, :, j] = 0.0, pos

    q, k, v = prompt
    rows = []
    for s, m in enumerate(new):
        for i in range(m):
            c.lens[s] += 1
            store(s, k[starts[s] + i], v[starts[s] + i], i)
            want, pv, size, js, _ = R.attend(c, s, c.lens[s] - 1, q[starts[s] + i], 0.125, window, 2)
            rows.append((want, R.tolerance(want, pv, size, len(js), c.dim, q_dtype, c.dtype)))
    yield torch.stack([r[0] for r in rows]), torch.stack([r[1] for r in rows])
    for i, (q, k, v) in enumerate(steps):
        rows = []
        for s in range(n):
            c.lens[s] += 1
            store(s, k[s], v[s], at[s])
            at[s] += 1
            want, pv, size, js, p = R.attend(c, s, c.lens[s] - 1, q[s], 0.125)
            weights[s][:, js] += p.reshape(hk, heads // hk, -1).sum(1)
            rows.append((want, R.tolerance(want, pv, size, len(js), c.dim, q_dtype, c.dtype)))
        yield torch.stack([r[0] for r in rows]), torch.stack([r[1] for r in rows])
        if i == 2:
            kept = R.evict(c, weights, positions, budget, 2, 8)
            for s in range(n):
                for h in range(hk):
                    src = [x for x in kept[s, h].tolist() if x >= 0]
                    moved = [(j, x) for j, x in enumerate(src) if j != x]
                    for j, x in moved:
                        a, b = c.slot(s, j), c.slot(s, x)
                        c.k[a[0], a[1], h], c.v[a[0], a[1], h] = c.k[b[0], b[1], h], c.v[b[0], b[1], h]
                    weights[s, h, :len(src)], positions[s, h, :len(src)] = weights[s, h, src], positions[s, h, src]
                c.lens[s] = min(c.lens[s], budget)


@pytest.mark.parametrize("types", [(F32, F32), (F32, F16), (BF16, BF16)], ids=str)
def test_a_conversation(types):
    need_gpu()
    import cera_b200 as cb
    heads, budget = 8, 48
    c = R.Cache([0, 0, 0, 0], 2, 64, 16, types[1], seed=20, spare=7)
    new, starts, prompt, steps = _serve_parts(c, heads, types[0], 21)
    cache = c.cuda()
    up = lambda t: tuple(x.cuda() for x in t)  # noqa: E731
    w, p = torch.zeros(4, 2, c.capacity).cuda(), torch.zeros(4, 2, c.capacity, dtype=torch.int32).cuda()
    got = _serve(cb, cache, (c.ld, starts.cuda(), up(prompt), [up(x) for x in steps], w, p, budget), heads, 24)
    for i, (want, tol) in enumerate(_serve_reference(c, new, starts, prompt, steps, heads, types[0], 24, budget)):
        R.check(got[i], want, tol, f"call {i}")
    assert got[-1].tolist() == c.lens


def test_on_a_side_stream_and_in_a_graph():
    """Captured once, replayed with other lengths, tables and queries in the same tensors."""
    need_gpu()
    import cera_b200 as cb
    c = R.Cache([100, 7], 2, 64, 16, F16, seed=30, spare=4)
    cache = c.cuda()
    q = _q(2, 8, 64, F16).cuda()
    starts = torch.tensor([0, 2, 4], dtype=torch.int32).cuda()
    qp = _q(4, 8, 64, F16, seed=9).cuda()
    w = torch.zeros(2, 2, c.capacity).cuda()

    def step():
        return cb.paged_decode_attention(cache, q, 0.125, weights=w), cb.paged_prefill_attention(cache, qp, starts, 0.125)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for turn in range(3):
        c.ld.copy_(torch.tensor([[100, 7], [3, 2], [64, 5]][turn]))
        if turn == 2:
            c.td.copy_(c.td.flip(1).contiguous())
            c.kd.copy_(torch.randn_like(c.kd.float()).half())
            c.vd.copy_(torch.randn_like(c.vd.float()).half())
        q.copy_(_q(2, 8, 64, F16, seed=turn + 40))
        w.zero_()
        want = [x.clone() for x in step()] + [w.clone()]
        for g, out in graphs:
            w.zero_()
            for x in out:
                x.fill_(9)
            g.replay()
            for a, b in zip([*out, w], want):
                assert torch.equal(a, b)


def test_calls_on_two_streams():
    need_gpu()
    import cera_b200 as cb
    cs = [R.Cache([900 + 300 * i, 40], 2, 64, 16, F16, seed=50 + i) for i in range(2)]
    caches = [c.cuda() for c in cs]
    qs = [_q(2, 8, 64, F16, seed=60 + i).cuda() for i in range(2)]
    want = [cb.paged_decode_attention(a, q, 0.125) for a, q in zip(caches, qs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(20):
        for a, q, st in zip(caches, qs, streams):
            with torch.cuda.stream(st):
                got.append(cb.paged_decode_attention(a, q, 0.125))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i % 2]) for i, g in enumerate(got))


@pytest.mark.parametrize("q_dtype,dtype", [(F32, F32), (F16, F16)], ids=str)
def test_pages_past_four_gigabytes(q_dtype, dtype):
    need_gpu()
    import cera_b200 as cb
    page, hk, dim, e = 64, 8, 128, torch.finfo(dtype).bits // 8
    pages = (5 << 30) // (page * hk * dim * e)
    k, v = (torch.empty(pages, page, hk, dim, dtype=dtype, device="cuda") for _ in range(2))
    c = R.Cache([130], hk, dim, page, dtype, seed=70, spare=0)
    c.cuda()
    far = torch.tensor([[pages - 1, pages // 2, pages - 3]], dtype=torch.int32)
    for i in range(3):
        k[far[0, i]], v[far[0, i]] = c.kd[c.table[0, i]], c.vd[c.table[0, i]]
    cache = cb.PagedKv(k, v, far.cuda(), c.ld)
    q = _q(1, 8, dim, q_dtype).cuda()
    want = cb.paged_decode_attention(c.cuda(), q, 0.1)
    assert torch.equal(cb.paged_decode_attention(cache, q, 0.1), want)
    starts = torch.tensor([0, 1], dtype=torch.int32).cuda()
    assert torch.equal(cb.paged_prefill_attention(cache, q, starts, 0.1), cb.paged_prefill_attention(c.cuda(), q, starts, 0.1))
    new = torch.randn(1, hk, dim, device="cuda")
    cb.paged_append(cache, new, new)
    assert torch.equal(k[pages - 3, 1], new[0].to(dtype)) and torch.equal(v[pages - 3, 1], new[0].to(dtype))
    w, pos = torch.rand(1, hk, 192).cuda(), torch.arange(192, dtype=torch.int32).cuda().expand(1, hk, 192).contiguous()
    w[..., 128] = 50.0
    kept, _ = cb.paged_evict(cache, w, pos, 1, 0, 0)
    assert (kept == 128).all() and torch.equal(k[pages - 1, 0], k[pages - 3, 0])


@pytest.mark.parametrize("types", TYPES, ids=str)
def test_sequences_that_share_their_beginning(types):
    """Pages in several tables, and twice in one: what is seen is as if they were copies."""
    need_gpu()
    import cera_b200 as cb
    c = R.Cache([100, 90, 160], 2, 64, 16, types[1], seed=85)
    c.table[1, :4] = c.table[0, :4]
    c.table[2, 5:8] = c.table[2, 1:4]
    _decode_case(cb, c, 8, types[0], weights=True)
    _prefill_case(cb, c, 8, types[0], [20, 1, 70])


def test_the_same_call_gives_the_same_bits():
    need_gpu()
    import cera_b200 as cb
    c = R.Cache([3000, 70, 500], 2, 64, 16, BF16, seed=80)
    cache, q = c.cuda(), _q(3, 8, 64, BF16).cuda()
    runs = []
    for _ in range(5):
        w = torch.zeros(3, 2, c.capacity).cuda()
        runs.append((cb.paged_decode_attention(cache, q, 0.125, weights=w), w))
    assert all(torch.equal(a, runs[0][0]) and torch.equal(b, runs[0][1]) for a, b in runs)
