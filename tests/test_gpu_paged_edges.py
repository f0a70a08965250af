"""The paged cache's operators where they are easily wrong: bits of weights, sums of very many slots, scores and scales that are not ordinary numbers, a result over its
queries, and forms that only larger groups or several sequences reach."""
import math

import pytest
import torch

import paged_ref as R
from gpu_util import need_gpu
from test_gpu_paged import TYPES, _decode_case, _evict_case, _q, _track

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ---- prompts of 16 bits ---------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F16, BF16], ids=str)
@pytest.mark.parametrize("dim,length,new,window", [(64, 40, 40, 9), (128, 310, 300, 9), (256, 12, 7, 0), (96, 3000, 2, 11)])
def test_weights_of_16_bit_prompts_keep_more_bits_than_the_result(dtype, dim, length, new, window):
    """Few slots with weights that are nearly alike, and values that nearly cancel.  Bound: what f32 arithmetic may be off by, weights in two parts of the type (f16 2^-21,
    which R.tolerance has; bf16 2^-8 of 2^-8), the result rounded once.  A weight rounded once would be off by 2^-11 or 2^-8."""
    need_gpu()
    import cera_b200 as cb
    c = R.Cache([length], 2, dim, 16, dtype, seed=dim)
    q = _q(new, 6, dim, dtype, size=0.2)
    scale = 1.0 / math.sqrt(dim)
    got = cb.paged_prefill_attention(c.cuda(), q.cuda(), _i32([0, new]), scale, window=window)
    for i in range(new):
        want, pv, size, js, _ = R.attend(c, 0, length - new + i, q[i], scale, window)
        f32 = R.tolerance(want, pv, size, len(js), dim, F32, dtype) + (2.0 ** -16 * pv if dtype == BF16 else 0.0)
        R.check(got[i], want, f32 + torch.finfo(dtype).eps / 2 * (want.abs() + f32) + 2.0 ** -24, f"query {i}")


@pytest.mark.parametrize("types", TYPES, ids=str)
def test_a_step_without_tokens(types):
    need_gpu()
    import cera_b200 as cb
    c = R.Cache([20, 3], 2, 64, 16, types[1], seed=3)
    cache = c.cuda()
    q = torch.empty(0, 4, 64, dtype=types[0], device="cuda")
    assert cb.paged_prefill_attention(cache, q, _i32([0, 0, 0]), 0.125).shape == (0, 4, 64)
    cb.paged_append(cache, torch.empty(0, 2, 64, dtype=types[0], device="cuda"), torch.empty(0, 2, 64, dtype=types[0], device="cuda"), _i32([0, 0, 0]))
    none = cb.PagedKv(cache.k_pages, cache.v_pages, cache.page_table[:0], cache.seq_lens[:0])
    assert cb.paged_decode_attention(none, q, 0.125).shape == (0, 4, 64)
    assert cb.paged_prefill_attention(none, q, _i32([0]), 0.125).shape == (0, 4, 64)
    assert torch.equal(c.kd.cpu().view(torch.uint8), c.k.contiguous().view(torch.uint8))


def _shared(cb, n, slots, heads, dim, dtype, page=64):
    """n sequences over the same pages, values of one sign -> cache, keys and values [slots][heads][dim]."""
    g = torch.Generator("cuda").manual_seed(dim)
    k = torch.randn(slots // page, page, heads, dim, generator=g, device="cuda").to(dtype)
    v = (torch.rand(slots // page, page, heads, dim, generator=g, device="cuda") + 0.5).to(dtype)
    table = torch.arange(slots // page, dtype=torch.int32, device="cuda").expand(n, -1).contiguous()
    return cb.PagedKv(k, v, table, _i32([slots] * n)), k.reshape(slots, heads, dim), v.reshape(slots, heads, dim)


# ---- one token each -------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("slots", [40960, 131072])
def test_decode_over_very_many_slots(types, slots):
    """64 sequences of 8 heads, so that a CTA has whole units.  Bound, relative to the result's norm: 8 steps (16 with a third part) that the tensor cores cut by 2^-23 at most, 1.9e-6; the
    sums of those, and of the weights, in f32: up to 2048 roundings of 2^-25 at random signs, 1.4e-6; scores of size 0.05, exponentials and parts 2^-20, 1e-6.  16-bit queries: every number, 64 steps
    (7.6e-6), sums of those in f32, weights in two parts (bf16 2^-16) and the rounding of the result.  (A unit in one sum: 5.4e-5 at 40 960 slots, 1.6e-4 at 131 072.)"""
    need_gpu()
    import cera_b200 as cb
    dim = 128
    cache, k, v = _shared(cb, 64, slots, 8, dim, types[1])
    q = (torch.randn(64, 8, dim, generator=torch.Generator("cuda").manual_seed(1), device="cuda") * 0.01).to(types[0])
    got = cb.paged_decode_attention(cache, q, 1.0 / math.sqrt(dim))
    for h in (0, 5):
        want = torch.softmax(q[:, h].double() @ k[:, h].double().T / math.sqrt(dim), -1) @ v[:, h].double()
        off = (got[:, h].double() - want).abs()
        if types[0] == F32:
            assert float(off.norm() / want.norm()) < 8e-6
        else:
            assert float((off / want).max()) < torch.finfo(types[0]).eps / 2 + (2e-5 if types[0] == F16 else 5e-5)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=str)
def test_16_bit_prompts_over_very_many_slots(dtype):
    """10 240 queries over 131 072 slots of one sign, unsplit.  Bound: 4096 slots (bf16: 32 768) in one sum are 512 (4096) steps that the tensor cores cut by 2^-23 at most, 6.1e-5
    (4.9e-4), and 32 of those sums in f32 2e-6; scores of size 0.05 and two parts of a weight 2^-16 (bf16) or 2^-21; the result rounded once.  In one sum with one part a weight 131 072 slots lose
    1.5e-4 on average, a third of f16's rounding."""
    need_gpu()
    import cera_b200 as cb
    n, slots, dim = 10240, 131072, 64
    cache, k, v = _shared(cb, 1, slots, 1, dim, dtype)
    q = (torch.randn(n, 4, dim, generator=torch.Generator("cuda").manual_seed(1), device="cuda") * 0.01).to(dtype)
    got = cb.paged_prefill_attention(cache, q, _i32([0, n]), 0.125)
    rows = torch.arange(0, n, 97, device="cuda")
    hidden = torch.arange(slots, device="cuda") > (slots - n + rows)[:, None]
    for h in (0, 3):
        x = (q[rows, h].double() @ k[:, 0].double().T * 0.125).masked_fill_(hidden, -math.inf)
        want = torch.softmax(x, -1) @ v[:, 0].double()
        off = (got[rows, h].double() - want).abs() / want
        assert float(off.max()) < torch.finfo(dtype).eps / 2 + (8e-5 if dtype == F16 else 5.2e-4)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=str)
@pytest.mark.parametrize("dim", [64, 128, 224])
def test_a_maximum_that_rises_after_sums_were_put_aside(dtype, dim):
    """Scores that rise along 40 000 slots to 64, 16-bit queries, unsplit.  Bound: scores in dim / 16 <= 14 steps of 2^-23 of 64, which enter twice, 2.2e-4; sums as in
    test_16_bit_prompts_over_very_many_slots."""
    need_gpu()
    import cera_b200 as cb
    n, heads, slots, page = 2400, 16, 40000, 32
    g = torch.Generator("cuda").manual_seed(dim)
    k = torch.randn(slots // page, page, 2, dim, generator=g, device="cuda")
    k[..., 0] = torch.arange(slots, device="cuda").reshape(-1, page, 1) * (60.0 / slots)
    k, v = k.to(dtype), (torch.rand(slots // page, page, 2, dim, generator=g, device="cuda") + 0.5).to(dtype)
    q = torch.randn(n, heads, dim, generator=g, device="cuda") * 0.5
    q[..., 0] = math.sqrt(dim)
    q = q.to(dtype)
    table = torch.randperm(slots // page, generator=torch.Generator().manual_seed(1)).to(torch.int32)[None].cuda()
    cache = cb.PagedKv(k, v, table, _i32([slots]))
    got = cb.paged_prefill_attention(cache, q, _i32([0, n]), 1.0 / math.sqrt(dim))
    rows = torch.arange(0, n, 7, device="cuda")
    kk, vv = (x[table[0].long()].reshape(slots, 2, dim).double() for x in (k, v))
    hidden = torch.arange(slots, device="cuda") > (slots - n + rows)[:, None]
    for h in (0, 13):
        x = (q[rows, h].double() @ kk[:, h // 8].T / math.sqrt(dim)).masked_fill_(hidden, -math.inf)
        want = torch.softmax(x, -1) @ vv[:, h // 8]
        off = (got[rows, h].double() - want).abs() / want
        assert float(off.max()) < torch.finfo(dtype).eps / 2 + (3.2e-4 if dtype == F16 else 8e-4)


def _newest_slot(types, length, bad, where):
    """The newest slot's key or value is not finite; at 33, 65 and 129 slots it has a part of the call to itself.  A NaN or infinite score makes the result NaN, one of minus infinity weighs
    nothing; values reach their own number of the result."""
    import cera_b200 as cb
    c = R.Cache([length], 1, 64, 16, types[1], seed=length)
    p, r = c.slot(0, length - 1)
    (c.k if where == "key" else c.v)[p, r, 0, 7] = bad
    q = _q(1, 6, 64, types[0])
    cache = c.cuda()
    w = torch.zeros(1, 1, c.capacity).cuda()
    want, pv, size, js, pr = R.attend(c, 0, length - 1, q[0], 0.125)
    fine = torch.isfinite(want)
    want, pv = want.nan_to_num(0.0, 1.0, -1.0), torch.where(torch.isfinite(pv), pv, 0.0)
    nan, sign = torch.isnan(R.attend(c, 0, length - 1, q[0], 0.125)[0]), torch.where(fine, 0.0, want)
    tol = R.tolerance(want, pv, size if math.isfinite(size) else 10.0, len(js), 64, types[0], types[1])
    for got in (cb.paged_decode_attention(cache, q.cuda(), 0.125), cb.paged_decode_attention(cache, q.cuda(), 0.125, weights=w),
                cb.paged_prefill_attention(cache, q.cuda(), _i32([0, 1]), 0.125)):
        got = got[0].cpu().double()
        assert torch.equal(torch.isnan(got), nan)
        assert torch.equal(torch.where(fine | nan, 0.0, got.nan_to_num(0.0, 1.0, -1.0)), sign)
        R.check(torch.where(fine, got, 0.0), torch.where(fine, want, 0.0), tol, "what is finite")


@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("length", [65, 129, 33, 200])
def test_the_newest_key_is_no_number(types, length):
    need_gpu()
    _newest_slot(types, length, math.nan, "key")


@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("length", [65, 129, 33, 200])
@pytest.mark.parametrize("bad,where", [(math.inf, "key"), (-math.inf, "key"), (math.inf, "value"), (-math.inf, "value"), (math.nan, "value")])
def test_the_newest_slot_is_infinite(types, length, bad, where):
    need_gpu()
    _newest_slot(types, length, bad, where)


@pytest.mark.parametrize("types", [(F32, F32), (F32, BF16), (BF16, BF16)], ids=str)
def test_scores_next_to_the_lowest_number(types):
    """All scores alike at about -3.2e38 in the exponent's units: the mean of the values."""
    need_gpu()
    import cera_b200 as cb
    k = torch.full((3, 64, 1, 64), 2.0 ** 60).to(types[1])
    v = torch.randn(3, 64, 1, 64, generator=torch.Generator().manual_seed(1)).to(types[1])
    q = torch.full((1, 2, 64), -3.2e38 / 1.4427 / 64 / 2.0 ** 60).to(types[0])
    cache = cb.PagedKv(k.cuda(), v.cuda(), _i32([[0, 1, 2]]), _i32([150]))
    want = v.reshape(-1, 64)[:150].double().mean(0).expand(2, 64)
    pv = v.reshape(-1, 64)[:150].double().abs().mean(0).expand(2, 64)
    tol = R.tolerance(want, pv, 0.0, 150, 64, types[0], types[1])
    w = torch.zeros(1, 1, 192).cuda()
    R.check(cb.paged_decode_attention(cache, q.cuda(), 1.0, weights=w)[0], want, tol, "decode")
    assert float((w[0, 0, :150] * 75 - 1).abs().max()) < 1e-5 and not w[0, 0, 150:].any()
    R.check(cb.paged_prefill_attention(cache, q.cuda(), _i32([0, 1]), 1.0)[0], want, tol, "prompt")


# ---- scales ---------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("scale", [0.0, -0.0, -0.125, 1e-39, -1e-39])
def test_scales(types, scale):
    need_gpu()
    import cera_b200 as cb
    c = R.Cache([200], 2, 64, 16, types[1], seed=3)
    q = _q(30, 4, 64, types[0])
    got = cb.paged_prefill_attention(c.cuda(), q.cuda(), _i32([0, 30]), scale, window=50, n_sink=3)
    one = cb.paged_decode_attention(c.cuda(), q[29:].cuda(), scale, window=50, n_sink=3)
    for i in range(30):
        want, pv, size, js, _ = R.attend(c, 0, 170 + i, q[i], scale, 50, 3)
        tol = R.tolerance(want, pv, size, len(js), 64, types[0], types[1])
        R.check(got[i], want, tol, f"query {i}")
        if i == 29:
            R.check(one[0], want, tol, "decode")


@pytest.mark.parametrize("types", TYPES, ids=str)
def test_a_scale_that_is_no_number(types):
    """Every row that sees a slot is NaN; one that sees none is zero."""
    need_gpu()
    import cera_b200 as cb
    c = R.Cache([20], 2, 64, 16, types[1], seed=3)
    q = _q(25, 4, 64, types[0]).cuda()
    got = cb.paged_prefill_attention(c.cuda(), q, _i32([0, 25]), math.nan)
    assert not got[:5].any() and torch.isnan(got[5:]).all()
    assert torch.isnan(cb.paged_decode_attention(c.cuda(), q[:1], math.nan)).all()


@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("in_query", [False, True])
def test_a_scale_of_zero_times_what_is_not_finite(types, bad, in_query):
    """Zero times infinity is NaN, for those who see it."""
    need_gpu()
    import cera_b200 as cb
    c = R.Cache([90], 1, 64, 16, types[1], seed=3)
    q = _q(90, 2, 64, types[0])
    if in_query:
        q[60:, :, 5] = bad
    else:
        p, r = c.slot(0, 60)
        c.k[p, r, 0, 5] = bad
    got = cb.paged_prefill_attention(c.cuda(), q.cuda(), _i32([0, 90]), 0.0)
    assert torch.isfinite(got[:60]).all() and torch.isnan(got[60:]).all()
    assert torch.isnan(cb.paged_decode_attention(c.cuda(), q[89:].cuda(), 0.0)).all()


# ---- a result over its queries --------------------------------------------------------------------------------------

@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("new,length", [(90, 200), (3, 1000), (300, 400)])
def test_a_result_may_go_where_its_queries_are(types, new, length):
    """With an infinite value that some rows do not see: those are computed a second time, from the queries."""
    need_gpu()
    import cera_b200 as cb
    c = R.Cache([length], 2, 64, 16, types[1], seed=3)
    p, r = c.slot(0, length - new // 2 - 1)
    c.v[p, r, 0, 5] = math.inf
    q = _q(new, 4, 64, types[0]).cuda()
    starts = _i32([0, new])
    want = cb.paged_prefill_attention(c.cuda(), q, starts, 0.125)
    over = q.clone()
    assert cb.paged_prefill_attention(c.cuda(), over, starts, 0.125, out=over) is over
    assert torch.equal(over.isnan(), want.isnan()) and torch.equal(over.nan_to_num(0.0), want.nan_to_num(0.0))
    want = cb.paged_decode_attention(c.cuda(), q[:1], 0.125)
    over = q[:1].clone()
    cb.paged_decode_attention(c.cuda(), over, 0.125, out=over)
    assert torch.equal(over.isnan(), want.isnan()) and torch.equal(over.nan_to_num(0.0), want.nan_to_num(0.0))


# ---- forms that only some calls reach -------------------------------------------------------------------------------

@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("heads,hk,dim", [(8, 1, 64), (5, 1, 128), (24, 2, 64), (17, 1, 96), (20, 1, 160), (6, 1, 256)])
def test_weights_of_large_groups(types, heads, hk, dim):
    """Five to eight heads a KV head, more than eight, and wide heads."""
    need_gpu()
    import cera_b200 as cb
    for window, sink in ((0, 0), (90, 4)):
        _decode_case(cb, R.Cache([1, 300, 0, 64, 130], hk, dim, 16, types[1], seed=heads), heads, types[0], window, sink, weights=True)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("longest,budget", [(9000, 900), (9000, 8500), (20000, 3000), (20000, 19500)])
def test_clusters_evict_several_sequences(longest, budget, in_place):
    """Clusters of four and eight CTAs a pair, ragged lengths, some within the budget; rows moved by a second launch and by the first."""
    need_gpu()
    import cera_b200 as cb
    c = R.Cache([0, 0, 0, 0], 2, 32, 64, F16)
    c.lens, c.wide = [longest, 5, 0, longest - 400], -(-longest // 64)
    c.pages, c.capacity = 4 * c.wide, c.wide * 64
    c.table = torch.randperm(c.pages, generator=torch.Generator().manual_seed(1)).to(torch.int32).reshape(4, c.wide)
    c.k, c.v = (torch.randn(c.pages, 64, 2, 32, generator=torch.Generator().manual_seed(i)).half() for i in (2, 3))
    _evict_case(cb, c, *_track(c, 5, ties=True), budget, 4, 30, in_place)


@pytest.mark.parametrize("types", TYPES, ids=str)
def test_a_workspace_of_ones_own(types):
    """Filled with NaN, used by one call after the other, of the size that is asked for and not a byte less."""
    need_gpu()
    import ctypes as C
    import cera_b200 as cb
    from cera_b200._lib import lib
    c = R.Cache([3000, 70, 0], 2, 64, 16, types[1], seed=80)
    cache = c.cuda()
    q, starts = _q(9, 8, 64, types[0]).cuda(), _i32([0, 4, 9, 9])
    w = [torch.zeros(3, 2, c.capacity).cuda() for _ in range(2)]
    ref = C.byref(cache._desc)
    calls = [(lambda **kw: cb.paged_decode_attention(cache, q[:3].contiguous(), 0.125, **kw), lib.cera_cuda_paged_decode_attention_workspace_bytes(ref, 8, 0)),
             (lambda **kw: cb.paged_decode_attention(cache, q[:3].contiguous(), 0.125, weights=w["workspace" in kw], **kw),
              lib.cera_cuda_paged_decode_attention_workspace_bytes(ref, 8, 1)),
             (lambda **kw: cb.paged_prefill_attention(cache, q, starts, 0.125, **kw), lib.cera_cuda_paged_prefill_attention_workspace_bytes(ref, 8, 9))]
    ws = torch.full((max(n for _, n in calls) + 64,), 255, dtype=torch.uint8, device="cuda")
    for _ in range(2):
        for call, need in calls:
            want = call()
            out = torch.full_like(want, 9.0)
            assert call(workspace=ws[:need], out=out) is out and torch.equal(out, want)
            with pytest.raises(ValueError, match="workspace"):
                call(workspace=ws[:need - 1])
    assert torch.equal(w[0], w[1])


def test_no_wait_of_these_kernels_ran_out():
    need_gpu()
    from cera_b200._lib import kernel_status
    torch.cuda.synchronize()
    assert kernel_status() == 0


@pytest.mark.parametrize("starts", [[0, 9, 2, 2], [0, 2, 9, 1], [0, 12, 12, 12], [5, 5, 5, 12], [0, -4, 3, 3], [3, 2, 1, 0]])
def test_starts_that_do_not_ascend_touch_nothing_else(starts):
    """They are not allowed, and what they give is not said; what lies beside the sequences' slots stays as it was."""
    need_gpu()
    import cera_b200 as cb
    c = R.Cache([48, 48, 48], 2, 64, 16, F16, seed=7, spare=0)
    cache = c.cuda()
    spare = next(p for p in range(c.pages) if p not in set(c.table.flatten().tolist()))
    table = torch.full((5, 3), spare, dtype=torch.int32)  # a slot past the capacity would find the page that no sequence has
    table[1:4] = c.table
    whole = table.cuda()
    cache = cb.PagedKv(cache.k_pages, cache.v_pages, whole[1:4], cache.seq_lens)
    k = torch.ones(9, 2, 64, dtype=F16, device="cuda")
    w, p = torch.full((5, 2, 48), 3.0).cuda(), torch.full((5, 2, 48), 3, dtype=torch.int32).cuda()
    cb.paged_append(cache, k, k, _i32(starts), weights=w[1:4], positions=p[1:4])
    for x in (w, p):
        assert (x[0] == 3).all() and (x[4] == 3).all()
    assert torch.isnan(c.kd[spare]).all() and torch.isnan(c.vd[spare]).all()
    q = torch.full((11, 4, 64), 5.0, dtype=F16, device="cuda")
    out = torch.full_like(q, 7.0)
    cb.paged_prefill_attention(cache, q[:9], _i32(starts), 0.125, out=out[:9])
    assert (out[9:] == 7.0).all() and (whole[0] == spare).all() and (whole[4] == spare).all()


def test_as_many_sequences_as_there_may_be():
    need_gpu()
    import cera_b200 as cb
    lens = [(7 * i) % 5 + (200 if i % 1000 == 999 else 0) for i in range(4096)]
    c = R.Cache([0], 2, 32, 8, F16)
    c.lens, c.wide = lens, 26
    c.pages, c.capacity = sum(-(-x // 8) for x in lens), 26 * 8
    c.table, at = torch.full((4096, 26), -1, dtype=torch.int32), 0
    for s, x in enumerate(lens):
        n = -(-x // 8)
        c.table[s, :n] = torch.arange(at, at + n)
        at += n
    c.k, c.v = (torch.randn(c.pages, 8, 2, 32, generator=torch.Generator().manual_seed(i)).half() for i in (2, 3))
    cache = c.cuda()
    q = _q(4096, 4, 32, F16)
    w = torch.zeros(4096, 2, 208).cuda()
    got = cb.paged_decode_attention(cache, q.cuda(), 0.2, weights=w).cpu()
    last = [i for i, x in enumerate(lens) if x]
    starts = torch.zeros(4097, dtype=torch.int32)
    starts[1:] = torch.tensor([int(x > 0) for x in lens]).cumsum(0)
    again = cb.paged_prefill_attention(cache, q[last].contiguous().cuda(), starts.cuda(), 0.2).cpu()
    for n, s in enumerate(last):
        if s % 37 and lens[s] < 100:
            continue
        want, pv, size, js, p = R.attend(c, s, lens[s] - 1, q[s], 0.2)
        tol = R.tolerance(want, pv, size, len(js), 32, F16, F16)
        R.check(got[s], want, tol, f"sequence {s}")
        R.check(again[n], want, tol, f"sequence {s} as a prompt")
    assert not got[[i for i, x in enumerate(lens) if not x]].any()
    assert float((w.sum(-1).cpu() - 2.0 * torch.tensor([[float(x > 0)] for x in lens])).abs().max()) < 1e-4
    new = torch.randn(4096, 2, 32).half()
    pos = torch.full((4096, 2, 208), -1, dtype=torch.int32).cuda()
    cb.paged_append(cache, new.cuda(), new.cuda(), positions=pos)
    kept, lens_out = cb.paged_evict(cache, w, torch.arange(208, dtype=torch.int32).expand(4096, 2, 208).contiguous().cuda(), 3, 1, 1)
    assert torch.equal(lens_out.cpu(), torch.tensor([min(x, 3) for x in lens], dtype=torch.int32))
    assert torch.equal((kept >= 0).sum(-1).cpu(), torch.tensor([[min(x, 3)] * 2 for x in lens]))
    assert torch.equal((pos >= 0).sum(-1).cpu(), torch.tensor([[int(x > 0)] * 2 for x in lens]))


@pytest.mark.parametrize("types", TYPES, ids=str)
def test_no_room_and_no_pages(types):
    """Tables without columns, and caches without a page: nothing is seen, stored or kept that is not there."""
    need_gpu()
    import cera_b200 as cb
    q, starts = _q(5, 4, 64, types[0]).cuda(), _i32([0, 2, 5])
    new = _q(5, 2, 64, types[0]).cuda()
    for pages, wide in ((4, 0), (0, 3), (0, 0)):
        k, v = (torch.zeros(pages, 16, 2, 64, dtype=types[1], device="cuda") for _ in range(2))
        lens = _i32([9, 40])
        cache = cb.PagedKv(k, v, torch.zeros(2, wide, dtype=torch.int32, device="cuda"), lens)
        cap = 16 * wide
        w, p = torch.ones(2, 2, cap, device="cuda"), torch.arange(cap, dtype=torch.int32, device="cuda").expand(2, 2, cap).contiguous()
        assert not cb.paged_decode_attention(cache, q[:2].contiguous(), 0.125).any()
        assert not cb.paged_decode_attention(cache, q[:2].contiguous(), 0.125, weights=w, window=3, n_sink=1).any() and (w == 1).all()
        assert not cb.paged_prefill_attention(cache, q, starts, 0.125).any()
        cb.paged_append(cache, new, new, starts, weights=w, positions=p)
        kept, lens_out = cb.paged_evict(cache, w, p, 4, 1, 1)
        assert lens_out.tolist() == [min(x, cap, 4) for x in (9, 40)] and torch.equal((kept >= 0).sum(-1), lens_out[:, None].expand(2, 2).long())
        assert not k.any() and not v.any()
