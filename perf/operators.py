"""What is timed of the paged 4-bit key / value cache: its tables, its store and load, the attention that reads it,
and one whole step of them. Cases, inputs, the plain forms in elementary torch operations, and 64-bit results.

The cache holds n_pages pages of P token rows. q: uint8 [n_pages][2][kv_heads][P][head_dim / 2], two 4-bit codes per
byte, low one first; d: f16 [n_pages][2][kv_heads][head_dim / 32][P], one scale per 32 channels of a row; plane 0 holds
keys, plane 1 values. A code c stands for d (c - 8). Slot s is row s % P of page s / P.
"""
import math
import os
import random
import sys

import torch

own = False

DEV = "cuda"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "f32": 4}


# ---------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # one planning session, one new row over two observed frames of 258 rows: latency
        dict(name="attention_one_row", op="attention", dtype="f16", reqs=1, heads=16, kv_heads=16, dim=64, page=16,
             len_min=516, len_max=516, new_min=1, new_max=1, frame=0),
        # a batch of sessions of ragged lengths, one new row each, grouped heads
        dict(name="attention_rows_batch", op="attention", dtype="bf16", reqs=64, heads=32, kv_heads=8, dim=128, page=64,
             len_min=1000, len_max=8190, new_min=1, new_max=1, frame=1),
        # one very long context: few rows, the work has to be split along the keys
        dict(name="attention_long", op="attention", dtype="f16", reqs=1, heads=32, kv_heads=8, dim=128, page=64,
             len_min=131071, len_max=131071, new_min=1, new_max=1, frame=1),
        # candidates' rollouts: a new frame of 258 rows over three frames, block-causal by frame
        dict(name="attention_frames", op="attention", dtype="f16", reqs=96, heads=16, kv_heads=16, dim=64, page=32,
             len_min=774, len_max=774, new_min=258, new_max=258, frame=258),
        # prompt chunks of ragged sizes behind cached rows, causal
        dict(name="attention_chunks", op="attention", dtype="bf16", reqs=4, heads=32, kv_heads=8, dim=128, page=128,
             len_min=4100, len_max=8191, new_min=700, new_max=2047, frame=1),
        # a handful of sessions, one token each: the bookkeeping of a step, latency
        dict(name="tables_step", op="tables", reqs=8, page=16, cached_min=200, cached_max=800, new_min=1, new_max=1, pad=0),
        # thousands of sessions, idle ones, single rows and whole frames mixed
        dict(name="tables_large", op="tables", reqs=4000, page=64, cached_min=0, cached_max=4000, new_min=0, new_max=258,
             pad=1000),
        # the rows of one step of 64 sessions
        dict(name="store_step", op="store", dtype="f16", tokens=64, kv_heads=16, dim=64, page=16, pool=96),
        # whole prompts: 65,000 rows of 8 heads of 128
        dict(name="store_prompts", op="store", dtype="bf16", tokens=65000, kv_heads=8, dim=128, page=64, pool=66048),
        # cached rows of one session read back
        dict(name="load_session", op="load", dtype="f16", tokens=516, kv_heads=16, dim=64, page=16, pool=2048),
        # cached rows of many sessions read back, in f32
        dict(name="load_prompts", op="load", dtype="f32", tokens=50001, kv_heads=8, dim=128, page=64, pool=65536),
        # a whole step: tables, store of the new frames' rows, their attention
        dict(name="step_frames", op="step", dtype="f16", reqs=16, heads=16, kv_heads=16, dim=64, page=32,
             len_min=258, len_max=774, new_min=1, new_max=258, frame=258),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the ranges the listed ones stand for."""
    op = rng.choice(["attention", "attention", "attention", "tables", "store", "load", "step"])
    page = rng.choice([16, 32, 64, 128, 256])
    dim = rng.choice([32, 64, 96, 128])
    if op == "tables":
        lo = rng.randint(0, 300)
        new_lo = rng.randint(0, 3)
        return dict(op=op, reqs=_log(rng, 1, 4000), page=page, cached_min=lo, cached_max=lo + _log(rng, 1, 4000),
                    new_min=new_lo, new_max=new_lo + _log(rng, 1, 255), pad=_log(rng, 1, 1000) - 1)
    if op in ("store", "load"):
        kv_heads = rng.choice([1, 2, 3, 4, 8, 16])
        tokens = min(_log(rng, 1, 60000), 60000 * 8 * 128 // (kv_heads * dim))
        return dict(op=op, dtype=rng.choice(["f16", "bf16", "f32"]), tokens=tokens, kv_heads=kv_heads, dim=dim, page=page,
                    pool=tokens + _log(rng, 1, 300))
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 2, 3, 4, 7, 8, 16])
    heads = kv_heads * group
    kind = rng.choice(["rows", "draft", "chunk"]) if op == "attention" else "chunk"
    if kind == "rows":
        reqs, new_lo, new_hi, len_hi = _log(rng, 1, 64), 1, 1, _log(rng, 16, 30000)
    elif kind == "draft":
        reqs, new_lo, new_hi, len_hi = _log(rng, 1, 48), 1, rng.randint(2, 9), _log(rng, 16, 8000)
    else:
        reqs, new_lo, new_hi, len_hi = _log(rng, 1, 16), rng.randint(0, 16), _log(rng, 20, 900), _log(rng, 900, 4000)
    # never dearer than the largest listed ones: cached values, and score pairs
    reqs = max(1, min(reqs, 60 * 8190 * 8 * 128 // (len_hi * kv_heads * dim), 4 * 2047 * 8191 * 32 // (2 * heads * new_hi * len_hi)))
    return dict(op=op, dtype=rng.choice(["f16", "bf16"]), reqs=reqs, heads=heads, kv_heads=kv_heads, dim=dim, page=page,
                len_min=rng.randint(0, max(1, len_hi // 2)), len_max=len_hi, new_min=new_lo, new_max=new_hi,
                frame=rng.choice([0, 1, 1, 16, 258]))


# ---------------------------------------------------------------------------------------------- inputs

def _lengths(case, seed):
    """Host lengths of the case: (tokens in the cache before the step, new tokens) of each request. The case fixes
    the pairs, so that shapes do not change with the seed; the seed deals them out to the requests."""
    rng = random.Random(repr(sorted(case.items())))
    lo, hi = (case["cached_min"], case["cached_max"]) if case["op"] == "tables" else (case["len_min"], case["len_max"])
    new = [rng.randint(case["new_min"], case["new_max"]) for _ in range(case["reqs"])]
    total = [rng.randint(lo, hi) for _ in range(case["reqs"])]
    if case["op"] != "tables" and case["reqs"] > 8:
        total[rng.randrange(case["reqs"])] = 0          # a session that holds nothing
    if case["op"] == "attention":                       # the new rows are among the cached ones
        total = [t - n for t, n in zip(total, new)]
    pairs = list(zip(total, new))
    random.Random(1000003 * seed + 17).shuffle(pairs)
    return [c for c, _ in pairs], [n for _, n in pairs]


def _quantise(x):
    """f32 [..., hd] -> codes int [..., hd], scales f16 [..., hd / 32]."""
    g = x.float().unflatten(-1, (-1, 32))
    hi, lo = g.amax(-1), g.amin(-1)
    m = torch.where(hi >= -lo, hi, lo)
    d = (m / -8).to(torch.bfloat16).float().clamp(-8160, 8160).to(torch.float16)
    dd = d.double().unsqueeze(-1)
    c = torch.where(dd == 0, torch.full_like(dd, 8), torch.floor(g.double() / dd + 0.5) + 8).clamp(0, 15)
    return c.to(torch.uint8).flatten(-2), d


def _pack(codes, values):
    """codes [..., hd] -> bytes [..., hd / 2]. Value rows keep their channels in order. A key row is a sequence of
    8-channel words of which word t NG + g holds channels 32 g + 8 t .. + 7 (NG = hd / 32)."""
    if not values:
        codes = codes.unflatten(-1, (-1, 4, 8)).transpose(-3, -2).flatten(-3)
    pair = codes.unflatten(-1, (-1, 2))
    return pair[..., 0] | (pair[..., 1] << 4)


def _unpack(q, d, values):
    """bytes [..., hd / 2] and scales [..., hd / 32] -> f32 [..., hd]."""
    codes = torch.stack((q & 15, q >> 4), -1).flatten(-2)
    if not values:
        codes = codes.unflatten(-1, (4, -1, 8)).transpose(-3, -2).flatten(-3)
    v = (codes.float() - 8).unflatten(-1, (-1, 32)) * d.float().unsqueeze(-1)
    return v.flatten(-2)


def _rows(g, n, heads, dim, dtype, keys):
    x = torch.randn(n, heads, dim, generator=g, device=DEV)
    if keys:                                            # keys have a few channels far above the others
        gain = 1 + 4 * (torch.rand(heads, dim, generator=g, device=DEV) > 0.95)
        x = x * gain
    return x.to(dtype)


def _pool(g, n_pages, page, heads, dim):
    """A filled pool, made in parts of about 2^26 values."""
    q = torch.empty(n_pages, 2, heads, page, dim // 2, dtype=torch.uint8, device=DEV)
    d = torch.empty(n_pages, 2, heads, dim // 32, page, dtype=torch.float16, device=DEV)
    part = max(1, (1 << 26) // (page * heads * dim))
    for p in range(0, n_pages, part):
        n = min(part, n_pages - p)
        for plane in range(2):
            x = _rows(g, n * page, heads, dim, torch.float32, plane == 0)
            c, s = _quantise(x.view(n, page, heads, dim).transpose(1, 2))
            q[p:p + n, plane] = _pack(c, plane == 1)
            d[p:p + n, plane] = s.transpose(-1, -2)
    return q, d


def _tables_inputs(case, g, cached, new, spare):
    """Lengths, block table (-1 where no page is held) and free list on the GPU; pages in random order."""
    page = case["page"]
    held = [-(-c // page) for c in cached]
    need = [-(-(c + n) // page) - h for c, n, h in zip(cached, new, held)]
    width = max(1, max(h + n for h, n in zip(held, need)))
    n_pages = sum(held) + sum(need) + spare
    perm = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)
    h = torch.tensor(held, device=DEV)
    col = torch.arange(width, device=DEV)
    take = (torch.cumsum(h, 0) - h).unsqueeze(1) + col
    table = torch.where(col < h.unsqueeze(1), perm[take.clamp(max=n_pages - 1)], -1).to(torch.int32)
    free = perm[sum(held):].contiguous()
    return table, free, n_pages


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = _inputs(case, seed, g)
    if own:
        root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "jepa.cpp_b200")
        if root not in sys.path:
            sys.path.insert(0, root)
        from jepa_b200 import kv4
        s["kv4"] = kv4
        if "q_pool" in s:
            s["cache"] = kv4.KV4Cache.wrap(s["q_pool"], s["d_pool"])
    return s


def _inputs(case, seed, g):
    op = case["op"]
    s = dict(case=case)
    if op in ("store", "load"):
        dt = TYPES[case["dtype"]]
        n_pages = -(-case["pool"] // case["page"])
        n_slots = n_pages * case["page"]
        s["q_pool"], s["d_pool"] = _pool(g, n_pages, case["page"], case["kv_heads"], case["dim"])
        # rows of requests: runs of whole pages in random order, the first rows of each taken
        slots = torch.randperm(n_pages, generator=g, device=DEV).unsqueeze(1) * case["page"] + torch.arange(case["page"], device=DEV)
        s["slots"] = slots.flatten()[:case["tokens"]].contiguous()
        s["slots"][case["tokens"] // 2:case["tokens"] // 2 + 1] = -1 if case["tokens"] > 8 else s["slots"][case["tokens"] // 2]
        s["all_slots"] = torch.arange(n_slots, device=DEV)
        if op == "store":
            s["k"] = _rows(g, case["tokens"], case["kv_heads"], case["dim"], dt, True)
            s["v"] = _rows(g, case["tokens"], case["kv_heads"], case["dim"], dt, False)
        return s
    cached, new = _lengths(case, seed)
    if op == "attention":
        lens = [c + n for c, n in zip(cached, new)]
        s["table"], _, n_pages = _tables_inputs(case, g, lens, [0] * len(lens), 1)
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    else:
        s["table"], s["free"], n_pages = _tables_inputs(case, g, cached, new, 5)
        s["cached"] = torch.tensor(cached, dtype=torch.int32, device=DEV)
        s["added"] = torch.tensor(new, dtype=torch.int32, device=DEV)
        s["n_slots"] = max(1, sum(new) + case.get("pad", 3))
    if op == "tables":
        return s
    dt = TYPES[case["dtype"]]
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    if op == "attention":
        s["q_start"] = torch.tensor(start, dtype=torch.int32, device=DEV)
        s["q"] = _rows(g, max(1, start[-1]), case["heads"], case["dim"], dt, False)
    else:
        s["q"] = _rows(g, s["n_slots"], case["heads"], case["dim"], dt, False)
        s["k"] = _rows(g, s["n_slots"], case["kv_heads"], case["dim"], dt, True)
        s["v"] = _rows(g, s["n_slots"], case["kv_heads"], case["dim"], dt, False)
        s["all_slots"] = torch.arange(n_pages * case["page"], device=DEV)
    s["out"] = torch.zeros_like(s["q"])
    s["q_pool"], s["d_pool"] = _pool(g, n_pages, case["page"], case["kv_heads"], case["dim"])
    if op == "attention":
        # rows that no request holds: scales that are not numbers, as freed pages may leave them
        rows = torch.ones(n_pages, case["page"], dtype=torch.bool, device=DEV)
        col = torch.arange(s["table"].shape[1] * case["page"], device=DEV)
        have = col < s["lens"].unsqueeze(1)
        page = s["table"].repeat_interleave(case["page"], 1)
        rows[page[have].long(), (col % case["page"]).expand_as(have)[have]] = False
        s["d_pool"].masked_fill_(rows[:, None, None, None, :], float("nan"))
    s["max_len"] = max(1, max(c + n for c, n in zip(cached, new)))
    s["max_new"] = max(1, max(new))
    return s


# ---------------------------------------------------------------------------------------------- plain forms

def _plain_tables(s):
    page = s["case"]["page"]
    table, free, cached, added = s["table"], s["free"], s["cached"].long(), s["added"].long()
    held = (cached + page - 1) // page
    need = (cached + added + page - 1) // page - held
    start = torch.cat((torch.zeros_like(added[:1]), torch.cumsum(added, 0)))
    first = torch.cumsum(need, 0) - need
    col = torch.arange(table.shape[1], device=DEV)
    fresh = (col >= held.unsqueeze(1)) & (col < (held + need).unsqueeze(1))
    pick = (first.unsqueeze(1) + col - held.unsqueeze(1)).clamp(0, max(0, free.numel() - 1))
    full = torch.where(fresh, free[pick], table)
    table.copy_(full)
    i = torch.arange(s["n_slots"], device=DEV)
    r = torch.searchsorted(start[1:], i, right=True).clamp(max=added.numel() - 1)
    pos = cached[r] + i - start[r]
    idx = (pos // page).clamp(0, table.shape[1] - 1)
    slots = torch.where(i < start[-1], full[r, idx].long() * page + pos % page, -1)
    state = torch.stack((torch.zeros_like(need[0]), need.sum())).to(torch.int32)
    return (cached + added).to(torch.int32), start.to(torch.int32), slots, state


def _plain_store(q_pool, d_pool, k, v, slots):
    page = q_pool.shape[3]
    # a row without a slot takes its place in a spare row behind the pool's
    n = q_pool.shape[0]
    s = torch.where(slots < 0, n * page, slots)
    for plane, x in ((0, k), (1, v)):
        c, d = _quantise(x)
        qp = torch.cat((q_pool[:, plane].transpose(1, 2).flatten(0, 1), torch.zeros_like(q_pool[:1, 0, :, 0])))
        dp = torch.cat((d_pool[:, plane].permute(0, 3, 1, 2).flatten(0, 1), torch.zeros_like(d_pool[:1, 0, :, :, 0])))
        qp[s] = _pack(c, plane == 1)
        dp[s] = d
        q_pool[:, plane] = qp[:-1].unflatten(0, (n, page)).transpose(1, 2)
        d_pool[:, plane] = dp[:-1].unflatten(0, (n, page)).permute(0, 2, 3, 1)


def _plain_load(q_pool, d_pool, slots, dtype):
    page = q_pool.shape[3]
    s = slots.clamp(min=0)
    out = []
    for plane in range(2):
        q = q_pool[s // page, plane, :, s % page]
        d = d_pool[s // page, plane, :, :, s % page]
        x = _unpack(q, d, plane == 1)
        out.append(torch.where((slots < 0)[:, None, None], 0.0, x).to(dtype))
    return out


def _plain_attention(s, lens, q_start):
    case, q, table = s["case"], s["q"], s["table"]
    page, group = case["page"], case["heads"] // case["kv_heads"]
    n_len, n_new = s["max_len"], s["max_new"]
    lens, q_start = lens.long(), q_start.long()
    n = q_start[1:] - q_start[:-1]
    # queries and keys padded to the longest request
    i = torch.arange(n_new, device=DEV)
    there = i < n.unsqueeze(1)
    rows = torch.where(there, q_start[:-1].unsqueeze(1) + i, 0)
    qs = q.float()[rows].unflatten(2, (-1, group))                       # [R, n, Hkv, G, hd]
    j = torch.arange(n_len, device=DEV)
    held = j < lens.unsqueeze(1)
    pg = torch.where(held, table[:, j // page].long(), 0)
    k = _unpack(s["q_pool"][pg, 0, :, j % page], s["d_pool"][pg, 0, :, :, j % page], False)   # [R, L, Hkv, hd]
    v = _unpack(s["q_pool"][pg, 1, :, j % page], s["d_pool"][pg, 1, :, :, j % page], True)
    k = torch.where(held[..., None, None], k, 0.0)
    v = torch.where(held[..., None, None], v, 0.0)
    sc = torch.matmul(qs.permute(0, 2, 3, 1, 4).flatten(2, 3), k.permute(0, 2, 3, 1))         # [R, Hkv, G n, L]
    sc = sc * (1.0 / math.sqrt(case["dim"]))
    pos = (lens - n).unsqueeze(1) + i
    limit = lens.unsqueeze(1).expand_as(pos)
    if case["frame"]:
        limit = torch.minimum(limit, (torch.div(pos, case["frame"], rounding_mode="floor") + 1) * case["frame"])
        limit = torch.where(pos < 0, 0, limit)
    see = (j < limit.unsqueeze(2))[:, None, None].expand(-1, 1, group, -1, -1).flatten(2, 3)   # [R, 1, G n, L]
    sc = sc.masked_fill(~see, float("-inf"))
    top = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(top == float("-inf"), 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v.transpose(1, 2)) / torch.where(total == 0, 1.0, total)
    o = o.unflatten(2, (group, n_new)).permute(0, 3, 1, 2, 4).flatten(2, 3)                   # [R, n, H, hd]
    out = s["out"]
    out[rows[there]] = o[there].to(out.dtype)
    return out


def run(s):
    case, op = s["case"], s["case"]["op"]
    if own:
        return _run_own(s, case, op)
    if op == "tables":
        lens, start, slots, state = _plain_tables(s)
        return lens, start, slots, state, s["table"]
    if op == "store":
        _plain_store(s["q_pool"], s["d_pool"], s["k"], s["v"], s["slots"])
        return tuple(_plain_load(s["q_pool"], s["d_pool"], s["all_slots"], torch.float16))
    if op == "load":
        return tuple(_plain_load(s["q_pool"], s["d_pool"], s["slots"], TYPES[case["dtype"]]))
    if op == "attention":
        return _plain_attention(s, s["lens"], s["q_start"])
    lens, start, slots, state = _plain_tables(s)
    _plain_store(s["q_pool"], s["d_pool"], s["k"], s["v"], slots)
    out = _plain_attention(s, lens, start)
    k, v = _plain_load(s["q_pool"], s["d_pool"], s["all_slots"], torch.float16)
    return out, lens, start, slots, state, s["table"], k, v


def _run_own(s, case, op):
    if op == "tables":
        t = s["kv4"].build_tables(s["cached"], s["added"], s["table"], s["free"], case["page"], s["n_slots"])
        return t.lens, t.q_start, t.slots, t.state, s["table"]
    cache = s["cache"]
    if op == "store":
        cache.store(s["k"], s["v"], s["slots"])
        return cache.load(s["all_slots"], torch.float16)
    if op == "load":
        return cache.load(s["slots"], TYPES[case["dtype"]])
    if op == "attention":
        return cache.attention(s["q"], s["q_start"], s["lens"], s["table"], frame=case["frame"], max_len=s["max_len"],
                               max_new=s["max_new"], out=s["out"])
    t = s["kv4"].build_tables(s["cached"], s["added"], s["table"], s["free"], case["page"], s["n_slots"])
    cache.store(s["k"], s["v"], t.slots)
    out = cache.attention(s["q"], t.q_start, t.lens, s["table"], frame=case["frame"], max_len=s["max_len"],
                          max_new=s["max_new"], out=s["out"])
    k, v = cache.load(s["all_slots"], torch.float16)
    return out, t.lens, t.q_start, t.slots, t.state, s["table"], k, v


# ---------------------------------------------------------------------------------------------- 64-bit results

def _exact_values(x):
    """f64 [..., hd] -> the values its 4-bit codes stand for, group by group from the definition."""
    x = x.double().reshape(*x.shape[:-1], -1, 32)
    big = x.abs().amax(-1, keepdim=True)
    m = torch.where((x == big).any(-1, keepdim=True), big, -big)          # the positive one of two of equal size
    d = -m / 8
    man, ex = torch.frexp(d)
    d = torch.ldexp(torch.round(man * 256) / 256, ex)                     # 8 significant bits, ties to even
    d = d.clamp(-8160, 8160)
    tiny = 2.0 ** -24
    d = torch.where(d.abs() < 2.0 ** -14, torch.round(d / tiny) * tiny, d)
    code = torch.floor(x / torch.where(d == 0, 1.0, d) + 0.5).clamp(-8, 7)
    return (torch.where(d == 0, 0.0, code) * d).flatten(-2)


def _exact_pool(q, d, slots, plane):
    """f64 values [n, heads, hd] of rows of the pool, channel by channel from the layout's formula."""
    page, dim = q.shape[3], 2 * q.shape[4]
    pg, row = slots // page, slots % page
    bytes_ = q[pg, plane, :, row].long()
    scale = d[pg, plane, :, :, row].double()
    c = torch.arange(dim, device=DEV)
    at = c if plane else ((c % 32) // 8 * (dim // 32) + c // 32) * 8 + c % 8
    code = (bytes_[..., at // 2] >> (4 * (at % 2))) & 15
    return (code - 8).double() * scale[..., c // 32]


def exact(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = _inputs(case, seed, g)
    op = case["op"]
    if op in ("store", "load"):
        if op == "load":
            ok = s["slots"] >= 0
            out = []
            for plane in range(2):
                x = _exact_pool(s["q_pool"], s["d_pool"], s["slots"].clamp(min=0), plane)
                out.append(torch.where(ok[:, None, None], x, 0.0))
            return tuple(out)
        out = []
        for plane, x in ((0, s["k"]), (1, s["v"])):
            pool = _exact_pool(s["q_pool"], s["d_pool"], s["all_slots"], plane)
            ok = s["slots"] >= 0
            pool[s["slots"][ok]] = _exact_values(x[ok])
            out.append(pool)
        return tuple(out)
    cached, new = _lengths(case, seed)
    lens = [c + n for c, n in zip(cached, new)]
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    table = s["table"].tolist()
    ints = ()
    if op in ("tables", "step"):
        page, free, taken, slots = case["page"], s["free"].tolist(), 0, []
        for r, (c, n) in enumerate(zip(cached, new)):
            for i in range(-(-c // page), -(-(c + n) // page)):
                table[r][i] = free[taken]
                taken += 1
            slots += [table[r][p // page] * page + p % page for p in range(c, c + n)]
        slots += [-1] * (s["n_slots"] - len(slots))
        ints = (torch.tensor(lens, dtype=torch.int32), torch.tensor(start, dtype=torch.int32), torch.tensor(slots),
                torch.tensor([0, taken], dtype=torch.int32), torch.tensor(table, dtype=torch.int32))
        if op == "tables":
            return ints
    k = v = None
    if op == "step":
        k, v = (_exact_pool(s["q_pool"], s["d_pool"], s["all_slots"], plane) for plane in range(2))
        n = start[-1]
        at = ints[2][:n].to(DEV)
        k[at] = _exact_values(s["k"][:n])
        v[at] = _exact_values(s["v"][:n])
    out = s["out"].double()
    page, group = case["page"], case["heads"] // case["kv_heads"]
    for r in range(case["reqs"]):
        n, ln = new[r], lens[r]
        if not n or ln <= 0:
            continue
        at = torch.tensor([table[r][p // page] * page + p % page for p in range(ln)], device=DEV)
        kk = k[at] if k is not None else _exact_pool(s["q_pool"], s["d_pool"], at, 0)
        vv = v[at] if v is not None else _exact_pool(s["q_pool"], s["d_pool"], at, 1)
        pos = torch.arange(ln - n, ln, device=DEV)
        lim = torch.full_like(pos, ln)
        if case["frame"]:
            lim = torch.where(pos < 0, 0, ((pos // case["frame"]) + 1) * case["frame"]).clamp(max=ln)
        see = torch.arange(ln, device=DEV) < lim.unsqueeze(1)
        for h in range(case["heads"]):
            x = s["q"][start[r]:start[r + 1], h].double() @ kk[:, h // group].T / math.sqrt(case["dim"])
            x = torch.where(see, x, -torch.inf)
            m = x.amax(1, keepdim=True)
            p = torch.where(see, torch.exp(x - torch.where(m == -torch.inf, 0.0, m)), 0.0)
            z = p.sum(1, keepdim=True)
            out[start[r]:start[r + 1], h] = (p @ vv[:, h // group]) / torch.where(z == 0, 1.0, z)
    return (out,) + ints + (k, v) if op == "step" else out


# ---------------------------------------------------------------------------------------------- work

def work(case):
    """Each input read once, each output written once; lengths by their middle where they are drawn."""
    op = case["op"]
    if op in ("store", "load"):
        row = 2 * case["kv_heads"] * case["dim"]
        held = row * 0.5625
        if op == "load":
            return {"bytes": case["tokens"] * (held + row * SIZE[case["dtype"]] + 8), "flops": case["tokens"] * row}
        return {"bytes": case["tokens"] * (row * SIZE[case["dtype"]] + held + 8) + case["pool"] * (held + row * 2 + 8),
                "flops": 2 * case["tokens"] * row + case["pool"] * row}
    new = (case["new_min"] + case["new_max"]) / 2 * case["reqs"]
    if op == "tables":
        pages = new / case["page"]
        return {"bytes": case["reqs"] * 16 + new * 8 + case["pad"] * 8 + pages * 8, "flops": 0}
    mid = (case["len_min"] + case["len_max"]) / 2
    keys = mid * case["reqs"]
    row = 2 * case["kv_heads"] * case["dim"]
    size = SIZE[case["dtype"]]
    n = (case["new_min"] + case["new_max"]) / 2
    pairs = new * mid
    if op == "step":
        keys += new
        pairs = new * (mid + n)
    elif case["frame"] and case["frame"] < n:
        pairs = new * max(mid - n / 2, mid / 2)
    total = {"bytes": keys * row * 0.5625 + 2 * new * case["heads"] * case["dim"] * size, "flops": 4.0 * case["heads"] * case["dim"] * pairs}
    if op == "step":
        total["bytes"] += new * (row * (size + 0.5625) + 16) + keys * row * (0.5625 + 2)
    return total
