"""A paged key/value cache and what reads and writes it, as cases that can be timed and checked.

Families: storing new tokens' keys and values in the cache's pages (`append`), attention of one new token per sequence over the cache
(`decode`), attention of ragged portions of prompt tokens over it, with a sliding window and a few first tokens that stay visible
(`prompt`), and dropping the positions with the least accumulated attention weight (`evict`).

The cache is pages of `page` rows of kv_heads x dim numbers, a table of page numbers per sequence and the sequences' lengths; sequence s keeps
slot j in row j % page of page table[s][j / page].  With `own` unset, `run` evaluates the operators with elementary torch operations in 32
bits; `exact` evaluates the same formulas in 64 bits, sequence by sequence."""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # the smallest call: one decode step's keys and values of 64 conversations, f32 activations into an f16 cache, whose slots are weighed for eviction
        dict(name="append_step_64", kind="append", seqs=64, new=1, context=700, ragged=True, kv_heads=8, dim=128, page=16, q="f32", kv="f16", track=True),
        # prompts of several users that arrive together, bf16 throughout
        dict(name="append_prompts_6", kind="append", seqs=6, new=1900, context=0, ragged=True, kv_heads=8, dim=128, page=64, q="bf16", kv="bf16", track=False),
        # one conversation at the context of the package's benchmark: the latency a chat user waits for
        dict(name="decode_one_513", kind="decode", seqs=1, context=513, ragged=False, heads=32, kv_heads=8, dim=128, page=16, q="f32", kv="f16", window=0,
             sink=0, track=False),
        # a serving batch of conversations of all ages
        dict(name="decode_batch_24", kind="decode", seqs=24, context=9000, ragged=True, heads=40, kv_heads=8, dim=128, page=16, q="bf16", kv="bf16", window=0,
             sink=0, track=False),
        # one question about a very long document
        dict(name="decode_long_65537", kind="decode", seqs=1, context=65537, ragged=False, heads=32, kv_heads=8, dim=128, page=128, q="f16", kv="f16",
             window=0, sink=0, track=False),
        # a step that also adds up the attention weight of every slot, over the f32 cache that models have by default
        dict(name="decode_weights_4", kind="decode", seqs=4, context=4001, ragged=True, heads=32, kv_heads=8, dim=64, page=32, q="f32", kv="f32", window=0,
             sink=0, track=True),
        # a prompt of one chunk, f32 activations over an f16 cache
        dict(name="prompt_512", kind="prompt", seqs=1, new=512, context=0, ragged=False, heads=32, kv_heads=8, dim=128, page=16, q="f32", kv="f16", window=0,
             sink=0),
        # a document of 8000 tokens through a layer whose window is 4096
        dict(name="prompt_window_8000", kind="prompt", seqs=1, new=8000, context=0, ragged=False, heads=32, kv_heads=8, dim=128, page=64, q="bf16", kv="bf16",
             window=4096, sink=4),
        # the next turn of long conversations: a short question, or drafted tokens, over what is cached
        dict(name="prompt_turn_17", kind="prompt", seqs=2, new=17, context=30000, ragged=True, heads=32, kv_heads=8, dim=128, page=32, q="f16", kv="f16",
             window=0, sink=0),
        # small prompts of a small model, f32 throughout, with a short window
        dict(name="prompt_f32_3", kind="prompt", seqs=3, new=700, context=100, ragged=True, heads=14, kv_heads=2, dim=64, page=16, q="f32", kv="f32",
             window=256, sink=4),
        # one step of generation at a full budget: every sequence and head drops one slot for the token that came
        dict(name="evict_step_8", kind="evict", seqs=8, context=2049, kv_heads=8, dim=128, page=16, kv="f16", budget=2048, sink=4, recent=128, mixed=True),
        # a long prompt is cut down to its heaviest slots
        dict(name="evict_prompt_2", kind="evict", seqs=2, context=32000, kv_heads=8, dim=128, page=64, kv="bf16", budget=4096, sink=4, recent=512, mixed=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "decode", "decode", "prompt", "prompt", "evict"])
    kv = rng.choice(["f32", "f16", "bf16"])
    c = dict(kind=kind, kv_heads=rng.choice([1, 2, 4, 8]), dim=rng.choice([64, 64, 96, 128, 128, 128]), page=rng.choice([8, 16, 16, 24, 32, 64, 128]), kv=kv)
    if kind == "evict":
        context = _log(rng, 64, 32000)
        budget = max(16, int(context * rng.choice([0.1, 0.25, 0.5, 0.9])))
        c.update(seqs=_log(rng, 1, max(2, min(16, 64000 // context))), context=context, budget=budget, sink=rng.choice([0, 1, 4]),
                 recent=rng.randint(1, budget // 3), mixed=rng.random() < 0.5)
        return c
    c.update(q=kv if rng.random() < 0.5 else "f32", ragged=rng.random() < 0.7)
    if kind == "append":
        new = _log(rng, 1, 2000)
        c.update(seqs=_log(rng, 1, max(2, min(96, 8000 // new))), new=new, context=rng.randint(0, 1000), track=rng.random() < 0.5)
        return c
    c.update(heads=c["kv_heads"] * rng.choice([1, 2, 3, 4, 4, 5, 7, 8]), window=rng.choice([0, 0, 0, 1]) * _log(rng, 16, 2048), sink=0)
    if c["window"]:
        c["sink"] = rng.choice([0, 1, 4, 4])
    if kind == "decode":
        context = _log(rng, 1, 40000)
        c.update(seqs=_log(rng, 1, max(2, min(64, 100000 // context))), context=context, track=rng.random() < 0.3)
        return c
    new = _log(rng, 1, 700 if kv == "f32" else 1500)
    c.update(seqs=_log(rng, 1, max(2, min(16, 2000 // new))), new=new, context=_log(rng, 1, 4000) - 1)
    return c


# ---- inputs ----------------------------------------------------------------------------------------------------------

def _shares(case, n, most, least):
    """Lengths of the case's sequences: all alike, or spread over the range's logarithm (the longest is always there)."""
    if not case.get("ragged"):
        return [most] * n
    rng = random.Random(n * 1000003 + most)
    return [most] + [_log(rng, max(1, least), most) if most else 0 for _ in range(n - 1)]


def _lens(case):
    """(new tokens, all tokens) of each sequence; the cache holds the new tokens' slots last."""
    if case["kind"] in ("decode", "evict"):
        return [1] * case["seqs"], _shares(case, case["seqs"], case["context"], 1)
    new = _shares(case, case["seqs"], case["new"], max(1, case["new"] // 16))
    old = _shares(case, case["seqs"], case["context"], max(1, case["context"] // 16))
    return new, [a + b for a, b in zip(new, old)]


def _normal(shape, seed, what, dtype=torch.float32):
    return torch.randn(shape, device="cuda", dtype=dtype, generator=torch.Generator("cuda").manual_seed((seed * 1000003 + what) & 0x7FFFFFFFFFFFFFFF))


def _uniform(shape, seed, what):
    return torch.rand(shape, device="cuda", generator=torch.Generator("cuda").manual_seed((seed * 1000003 + what) & 0x7FFFFFFFFFFFFFFF))


def prepare(case, seed):
    new, lens = _lens(case)
    n, page, hk, dim, kv = case["seqs"], case["page"], case["kv_heads"], case["dim"], TYPES[case["kv"]]
    wide = max(-(-x // page) for x in lens)
    pages = n * wide + 1
    # pages as an allocator that has served for a while hands them out: in no order
    table = torch.argsort(_uniform((pages,), seed, 1))[:n * wide].reshape(n, wide).to(torch.int32).contiguous()
    s = dict(case=case, table=table, lens=torch.tensor(lens, dtype=torch.int32, device="cuda"), k=_normal((pages, page, hk, dim), seed, 2, kv),
             v=_normal((pages, page, hk, dim), seed, 3, kv), longest=max(new))
    if case["kind"] != "decode":
        s["starts"] = torch.tensor([0] + [sum(new[:i + 1]) for i in range(n)], dtype=torch.int32, device="cuda")
    if case["kind"] == "append":
        s["new_k"] = _normal((sum(new), hk, dim), seed, 4, TYPES[case["q"]])
        s["new_v"] = _normal((sum(new), hk, dim), seed, 5, TYPES[case["q"]])
        # a conversation that lost slots before: its next position is past its length
        s["at"] = torch.cat([torch.arange(x - m, x, device="cuda", dtype=torch.int32) + 64 for m, x in zip(new, lens)])
    elif case["kind"] != "evict":
        shape = (n if case["kind"] == "decode" else sum(new), case["heads"], dim)
        s["q"] = _normal(shape, seed, 6).mul_(1.5).to(TYPES[case["q"]])
        s["scale"] = 1.0 / math.sqrt(dim)
    if case.get("track") or case["kind"] == "evict":
        cap = wide * page
        heavy = torch.exp(2.0 * _normal((n, hk, cap), seed, 7))
        s["weights"] = torch.where(_uniform((n, hk, cap), seed, 8) < 0.02, torch.zeros_like(heavy), heavy)  # some slots are new, and weigh nothing yet
        s["positions"] = torch.arange(cap, device="cuda", dtype=torch.int32).expand(n, hk, cap).contiguous()
        if case.get("mixed"):  # earlier evictions left the slots in no order; the newest token is in the last one
            old = torch.argsort(_uniform((n, hk, max(lens) - 1), seed, 9)).to(torch.int32)
            s["positions"][..., :max(lens) - 1] = old
        if case["kind"] == "evict":
            s["weights_out"] = torch.zeros((n, hk, case["budget"]), device="cuda")
            s["positions_out"] = torch.zeros((n, hk, case["budget"]), dtype=torch.int32, device="cuda")
    return s


def work(case):
    new, lens = _lens(case)
    n, hk, dim, e = case["seqs"], case["kv_heads"], case["dim"], BYTES[case["kv"]]
    row = hk * dim
    if case["kind"] == "append":
        return {"bytes": sum(new) * (2 * row * (e + BYTES[case["q"]]) + (hk * 8 + 4 if case["track"] else 0)) + 8 * n, "flops": 0}
    if case["kind"] == "evict":
        kept = sum(min(x, case["budget"]) for x in lens)
        # a slot's weight and position are read, the kept ones' written; at least what is kept beyond the budget's share of slots moves
        moved = sum(max(0, x - case["budget"]) for x in lens)
        moved = max(n, moved * case["budget"] // max(lens)) if max(lens) > case["budget"] else 0
        return {"bytes": hk * (8 * sum(lens) + 12 * kept) + moved * 4 * row * e, "flops": 0}
    w, k0, heads = case["window"], case["sink"], case["heads"]
    pairs = rows = 0
    for m, x in zip(new, lens):
        if not w:
            pairs += m * x - m * (m - 1) // 2
            rows += x
        else:
            for p in range(x - m, x):
                pairs += min(p + 1, w + min(k0, max(0, p + 1 - w)))
            lo = max(0, x - m + 1 - w)
            rows += x - lo + min(k0, lo)
    bytes_ = rows * 2 * row * e + 2 * sum(new) * heads * dim * BYTES[case["q"]]
    if case.get("track"):
        bytes_ += rows * hk * 8
    return {"bytes": bytes_, "flops": 4 * pairs * heads * dim}


# ---- plain forms -----------------------------------------------------------------------------------------------------

def _gathered(s, pages):
    """[seqs][slots][kv_heads][dim] of a paged tensor, in 32 bits."""
    x = pages[s["table"].long()]
    return x.reshape(x.shape[0], -1, *x.shape[3:]).float()


def _attention(s, q, seen):
    """q [seqs][queries][heads][dim] over the cache where seen [seqs][queries][slots]: (result, probabilities [seqs][kv_heads][group][queries][slots])."""
    n, m, heads, dim = q.shape
    k, v = _gathered(s, s["k"]), _gathered(s, s["v"])
    hk = k.shape[2]
    qg = q.float().reshape(n, m, hk, heads // hk, dim).permute(0, 2, 3, 1, 4).reshape(n, hk, -1, dim)
    x = (qg @ k.permute(0, 2, 3, 1)).mul_(s["scale"]).reshape(n, hk, heads // hk, m, -1)
    x.masked_fill_(~seen[:, None, None], -math.inf)
    x -= x.amax(-1, keepdim=True)
    p = torch.exp_(x)
    p /= p.sum(-1, keepdim=True)
    out = p.reshape(n, hk, -1, p.shape[-1]) @ v.transpose(1, 2)
    return out.reshape(n, hk, heads // hk, m, dim).permute(0, 3, 1, 2, 4).reshape(n, m, heads, dim), p


def _seen(case, at, slots):
    """Whether the query at slot `at` [seqs][queries] sees each of `slots` slots."""
    j, p = torch.arange(slots, device=at.device), at[..., None]
    seen = j <= p
    if case["window"]:
        seen = seen & ((j < case["sink"]) | (j > p - case["window"]))
    return seen


def _plain_append(s):
    case, table, page = s["case"], s["table"].long(), s["case"]["page"]
    t = torch.arange(s["new_k"].shape[0], device="cuda")
    seq = torch.searchsorted(s["starts"].long(), t, right=True) - 1
    slot = s["lens"].long()[seq] - s["starts"].long()[seq + 1] + t
    at = table[seq, slot // page], slot % page
    s["k"][at] = s["new_k"].to(s["k"].dtype)
    s["v"][at] = s["new_v"].to(s["v"].dtype)
    if not case["track"]:
        return [s["k"], s["v"]]
    s["weights"][seq, :, slot] = 0.0
    s["positions"][seq, :, slot] = s["at"][:, None].expand(-1, case["kv_heads"])
    return [s["k"], s["v"], s["weights"], s["positions"]]


def _plain_decode(s):
    case = s["case"]
    slots = s["table"].shape[1] * case["page"]
    out, p = _attention(s, s["q"][:, None], _seen(case, s["lens"].long()[:, None] - 1, slots))
    out = out[:, 0].to(s["q"].dtype)
    if not case["track"]:
        return out
    s["weights"] += p[..., 0, :].sum(2)
    return [out, s["weights"]]


def _plain_prompt(s):
    case = s["case"]
    starts, m = s["starts"].long(), torch.arange(s["longest"], device="cuda")
    new = starts[1:] - starts[:-1]
    live = m < new[:, None]
    row = torch.where(live, starts[:-1, None] + m, 0)
    at = torch.where(live, (s["lens"].long() - new)[:, None] + m, 0)
    out, _ = _attention(s, s["q"][row], _seen(case, at, s["table"].shape[1] * case["page"]))
    return out[live].to(s["q"].dtype)


def _plain_evict(s):
    case, budget = s["case"], s["case"]["budget"]
    cap = s["weights"].shape[-1]
    j = torch.arange(cap, device="cuda")
    valid = (j < s["lens"][:, None])[:, None].expand_as(s["weights"])
    pos = torch.where(valid, s["positions"], -1)
    kept_anyway = (pos < case["sink"]) | (pos > pos.amax(-1, keepdim=True) - case["recent"])
    order = torch.where(kept_anyway, math.inf, s["weights"])
    order = torch.sort(torch.where(valid, order, -1.0), dim=-1, descending=True, stable=True).indices
    rank = torch.zeros_like(order).scatter_(-1, order, j.expand_as(order).contiguous())
    chosen = (rank < budget) & valid
    hole, mover = (valid & ~chosen & (j < budget)).nonzero(as_tuple=True), (chosen & (j >= budget)).nonzero(as_tuple=True)
    kept = torch.where(valid, j, -1)[..., :budget].to(torch.int32)
    kept[hole] = mover[2].to(torch.int32)
    src = kept.long().clamp(min=0)
    live = kept >= 0
    s["weights_out"].copy_(torch.where(live, s["weights"].gather(-1, src), s["weights_out"]))
    s["positions_out"].copy_(torch.where(live, s["positions"].gather(-1, src), s["positions_out"]))
    table, page = s["table"].long(), case["page"]
    to = table[hole[0], hole[2] // page], hole[2] % page, hole[1]
    fr = table[mover[0], mover[2] // page], mover[2] % page, mover[1]
    s["k"][to] = s["k"][fr]
    s["v"][to] = s["v"][fr]
    return [s["k"], s["v"], s["weights_out"], s["positions_out"], kept, s["lens"].clamp(max=budget)]


def run(s):
    case = s["case"]
    if not own:
        return {"append": _plain_append, "decode": _plain_decode, "prompt": _plain_prompt, "evict": _plain_evict}[case["kind"]](s)
    import cera_b200 as cb
    if "cache" not in s:  # the handle that a program keeps for a layer's cache
        s["cache"] = cb.PagedKv(s["k"], s["v"], s["table"], s["lens"])
    cache = s["cache"]
    if case["kind"] == "append":
        if not case["track"]:
            cb.paged_append(cache, s["new_k"], s["new_v"], s["starts"])
            return [s["k"], s["v"]]
        cb.paged_append(cache, s["new_k"], s["new_v"], s["starts"], weights=s["weights"], positions=s["positions"], token_positions=s["at"])
        return [s["k"], s["v"], s["weights"], s["positions"]]
    if case["kind"] == "decode":
        if not case["track"]:
            return cb.paged_decode_attention(cache, s["q"], s["scale"], window=case["window"], n_sink=case["sink"])
        return [cb.paged_decode_attention(cache, s["q"], s["scale"], window=case["window"], n_sink=case["sink"], weights=s["weights"]), s["weights"]]
    if case["kind"] == "prompt":
        return cb.paged_prefill_attention(cache, s["q"], s["starts"], s["scale"], window=case["window"], n_sink=case["sink"])
    kept, lens = cb.paged_evict(cache, s["weights"], s["positions"], case["budget"], n_sink=case["sink"], n_recent=case["recent"],
                                weights_out=s["weights_out"], positions_out=s["positions_out"])
    return [s["k"], s["v"], s["weights_out"], s["positions_out"], kept, lens]


# ---- the definitions, in 64 bits -------------------------------------------------------------------------------------

def _rows(s, pages, i, count):
    """Slots [0, count) of sequence i, [count][kv_heads][dim]."""
    need = -(-count // s["case"]["page"])
    return torch.cat(list(pages[s["table"][i, :need].long()].double()))[:count]


def _exact_attention(s, i, q, first, p_sum):
    """Queries q [m][heads][dim] of sequence i, the first at slot `first`; p_sum [kv_heads][slots] takes the probabilities."""
    case, m, heads = s["case"], q.shape[0], q.shape[1]
    hk, count = case["kv_heads"], first + q.shape[0]
    k, v = _rows(s, s["k"], i, count), _rows(s, s["v"], i, count)
    j, p = torch.arange(count, device="cuda")[None], torch.arange(first, count, device="cuda")[:, None]
    hidden = j > p
    if case["window"]:
        hidden |= (j >= case["sink"]) & (p - j >= case["window"])
    out = torch.empty(m, heads, case["dim"], dtype=torch.float64, device="cuda")
    for h in range(heads):
        g = h // (heads // hk)
        e = torch.einsum("md,jd->mj", q[:, h].double(), k[:, g]) * s["scale"]
        e[hidden] = -math.inf
        w = torch.softmax(e, -1)
        out[:, h] = torch.einsum("mj,jd->md", w, v[:, g])
        if p_sum is not None:
            p_sum[g, :count] += w.sum(0)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    new, lens = _lens(case)
    page = case["page"]
    if case["kind"] == "append":
        k, v, t = s["k"].double(), s["v"].double(), 0
        w = s["weights"].double() if case["track"] else None
        for i, (m, x) in enumerate(zip(new, lens)):
            slot = torch.arange(x - m, x, device="cuda")
            at = s["table"][i].long()[slot // page], slot % page
            k[at], v[at] = s["new_k"][t:t + m].double(), s["new_v"][t:t + m].double()
            if w is not None:
                w[i, :, x - m:x] = 0
            t += m
        return [k, v] if w is None else [k, v, w, None]
    if case["kind"] == "decode":
        w = s["weights"].double() if case["track"] else None
        out = torch.cat([_exact_attention(s, i, s["q"][i:i + 1], x - 1, None if w is None else w[i]) for i, x in enumerate(lens)])
        return out if w is None else [out, w]
    if case["kind"] == "prompt":
        at = [0] + [sum(new[:i + 1]) for i in range(len(new))]
        return torch.cat([_exact_attention(s, i, s["q"][at[i]:at[i + 1]], x - m, None) for i, (m, x) in enumerate(zip(new, lens))])
    k, v, budget = s["k"].double(), s["v"].double(), case["budget"]
    w_out, weights, positions = s["weights_out"].double(), s["weights"].cpu().tolist(), s["positions"].cpu().tolist()
    for i, x in enumerate(lens):
        if x <= budget:
            w_out[i, :, :x] = s["weights"][i, :, :x].double()
            continue
        for h in range(case["kv_heads"]):
            pos, wt = positions[i][h][:x], weights[i][h][:x]
            newest = max(pos)
            safe = [p < case["sink"] or newest - p < case["recent"] for p in pos]
            best = sorted(range(x), key=lambda j: (not safe[j], 0.0 if safe[j] else -wt[j], j))[:budget]
            stay = set(best)
            holes, movers = [j for j in range(budget) if j not in stay], sorted(j for j in best if j >= budget)
            w_out[i, h] = s["weights"][i, h, :budget].double()
            if not holes:
                continue
            a, b = torch.tensor(holes, device="cuda"), torch.tensor(movers, device="cuda")
            w_out[i, h, a] = s["weights"][i, h, b].double()
            row = s["table"][i].long()
            k[row[a // page], a % page, h] = s["k"][row[b // page], b % page, h].double()
            v[row[a // page], a % page, h] = s["v"][row[b // page], b % page, h].double()
    return [k, v, w_out, None, None, None]
