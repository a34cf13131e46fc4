"""The operators of the 8-bit paged KV cache (`jev.KvPages`), as cases that can be timed and checked.

Many requests share one pool of pages; a key or value element takes a byte, with a scale for each
block of 16 tokens and KV head.  A case's `kind` names the operator:

plan    a step's bookkeeping from the requests' lengths: pages beyond what each request keeps are
        given back, the missing ones taken (lowest-numbered free page first, in batch order), and
        every new token gets its slot, position and batch row
rotate  rotary positions on a batch's queries: interleaved or half layout, the whole head or a part
        of it, frequencies scaled for long contexts
store   the same rotation on queries and keys, the keys and values into their pages, and the touched
        blocks read back as the values they stand for
attend  attention of a batch's queries over their requests' pages: one token a request, or prompts

`run` computes them in plain torch operations, or with `own` through the package.  The geometries
are the package's model (32 / 8 heads of 128, rotary base 1e6) and generic ones.
"""
import math
import os
import sys

import numpy as np
import torch

own = False  # set from outside: run() calls the package's operators

BLOCK = 16  # tokens that share a scale
GROUPS = {(32, 8, 128), (16, 2, 64), (8, 8, 128), (28, 4, 128), (24, 8, 64), (12, 1, 128)}


def listed():
    return [
        # a step of twelve reasoning rows: the smallest plan
        {"name": "plan_rows_12", "kind": "plan", "requests": 12, "others": 0, "past_lo": 250, "past_hi": 1100, "over": 0,
         "fresh_lo": 1, "fresh_hi": 1, "page": 16, "pad": 0, "mix": 1},
        # a busy server's step: prompts and single tokens, some requests cut back to a shared start first
        {"name": "plan_batch_700", "kind": "plan", "requests": 700, "others": 211, "past_lo": 1, "past_hi": 4096, "over": 90,
         "fresh_lo": 1, "fresh_hi": 150, "page": 32, "pad": 37, "mix": 2},
        # one decoded token's queries
        {"name": "rotate_token", "kind": "rotate", "heads": 32, "kv_heads": 8, "dim": 128, "rope": 128, "half": False,
         "factor": 1.0, "yarn": False, "requests": 1, "past_lo": 700, "past_hi": 700, "fresh_lo": 1, "fresh_hi": 1, "mix": 3},
        # prompts far into long contexts, the half layout over part of the head, scaled frequencies
        {"name": "rotate_long_half", "kind": "rotate", "heads": 32, "kv_heads": 8, "dim": 128, "rope": 96, "half": True,
         "factor": 8.0, "yarn": True, "requests": 9, "past_lo": 3000, "past_hi": 120000, "fresh_lo": 500, "fresh_hi": 1500, "mix": 4},
        # a decode step of 64 requests: most blocks are begun, some scales grow
        {"name": "store_rows_64", "kind": "store", "heads": 32, "kv_heads": 8, "dim": 128, "rope": 128, "half": False,
         "factor": 1.0, "yarn": False, "page": 16, "requests": 64, "past_lo": 100, "past_hi": 9000, "fresh_lo": 1, "fresh_hi": 1, "mix": 5},
        # prompts of uneven lengths behind cached ones
        {"name": "store_prompts", "kind": "store", "heads": 32, "kv_heads": 8, "dim": 128, "rope": 128, "half": False,
         "factor": 1.0, "yarn": False, "page": 64, "requests": 11, "past_lo": 1, "past_hi": 1000, "fresh_lo": 90, "fresh_hi": 2000, "mix": 6},
        # one short conversation's next token: the smallest attention
        {"name": "attend_token", "kind": "attend", "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "requests": 1,
         "past_lo": 299, "past_hi": 299, "fresh_lo": 1, "fresh_hi": 1, "mix": 7},
        # one token over a very long document
        {"name": "attend_token_long", "kind": "attend", "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "requests": 1,
         "past_lo": 120001, "past_hi": 120001, "fresh_lo": 1, "fresh_hi": 1, "mix": 8},
        # a decode step of sixty-four requests of all lengths
        {"name": "attend_rows_64", "kind": "attend", "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "requests": 64,
         "past_lo": 500, "past_hi": 12000, "fresh_lo": 1, "fresh_hi": 1, "mix": 9},
        # the same with narrow heads, eight queries to a KV head
        {"name": "attend_rows_64_narrow", "kind": "attend", "heads": 16, "kv_heads": 2, "dim": 64, "page": 32, "requests": 200,
         "past_lo": 30, "past_hi": 5000, "fresh_lo": 1, "fresh_hi": 1, "mix": 10},
        # nine options of a decision behind their cached policy
        {"name": "attend_options_9x48", "kind": "attend", "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "requests": 9,
         "past_lo": 4096, "past_hi": 4096, "fresh_lo": 48, "fresh_hi": 48, "mix": 11},
        # prompts being read, short ones beside long ones
        {"name": "attend_prompts", "kind": "attend", "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "requests": 4,
         "past_lo": 1, "past_hi": 700, "fresh_lo": 300, "fresh_hi": 4000, "mix": 12},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["plan", "rotate", "store", "attend", "attend"])
    c = {"kind": kind, "page": rng.choice([16, 32, 64, 128]), "mix": rng.randrange(1 << 20)}
    if kind == "plan":
        c.update(requests=_log_int(rng, 1, 700), others=_log_int(rng, 2, 300), past_lo=_log_int(rng, 1, 60),
                 past_hi=_log_int(rng, 60, 4096), over=rng.choice([0, 1, 40, 90]), fresh_lo=1,
                 fresh_hi=rng.choice([1, 1, _log_int(rng, 2, 150)]), pad=rng.choice([0, 1, 37]))
        return c
    heads, kv, dim = rng.choice(sorted(GROUPS))
    c.update(heads=heads, kv_heads=kv, dim=dim)
    if kind == "rotate":
        del c["page"]
    if kind in ("rotate", "store"):
        c.update(rope=rng.choice([dim, dim // 2, 3 * dim // 4, 20]), half=rng.random() < 0.5,
                 factor=rng.choice([1.0, 4.0, 8.0]))
        c.update(yarn=c["factor"] > 1 and rng.random() < 0.5, requests=_log_int(rng, 1, 64))
        most = 9000 // c["requests"]
        c.update(past_lo=_log_int(rng, 1, 300), past_hi=_log_int(rng, 300, 100000 if kind == "rotate" else 6000),
                 fresh_lo=1, fresh_hi=rng.choice([1, _log_int(rng, 2, max(3, most))]))
        if c["requests"] * c["past_hi"] > 2000000:
            c["past_hi"] = max(c["past_lo"], 2000000 // c["requests"])
        return c
    if rng.random() < 0.5:  # one token a request
        c.update(requests=_log_int(rng, 1, 200), fresh_lo=1, fresh_hi=1)
        most = min(120000, 400000 // c["requests"])
        c.update(past_lo=_log_int(rng, 1, 200), past_hi=_log_int(rng, 200, max(201, most)))
    else:  # prompts
        c.update(requests=_log_int(rng, 1, 12))
        c.update(fresh_lo=_log_int(rng, 1, 40), fresh_hi=_log_int(rng, 40, max(41, 4000 // c["requests"])),
                 past_lo=1, past_hi=_log_int(rng, 1, 5000))
    return c


def lengths(case):
    """Tokens each request has and gets, spread over the logarithm; the same for every seed."""
    r = np.random.RandomState(case["mix"])

    def spread(lo, hi):
        return np.exp(r.uniform(math.log(lo), math.log(hi), case["requests"])).round().astype(np.int64).clip(lo, hi)

    return spread(case["past_lo"], case["past_hi"]), spread(case["fresh_lo"], case["fresh_hi"])


def _ints(a):
    return torch.as_tensor(np.ascontiguousarray(a), dtype=torch.int32, device="cuda")


def _pages(n, page):
    return -(-n // page)


# ---------------------------------------------------------------- what a program has in hand


def _package():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llm-shield_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import jev

    return jev


def _cache(case, n_pages, requests, context, tokens):
    """The package's cache for a case."""
    jev = _package()
    dim = case.get("dim", 64)
    cfg = jev.ModelConfig(n_layers=1, n_heads=case.get("heads", 1), n_kv_heads=case.get("kv_heads", 1), head_dim=dim,
                          rope_dim=case.get("rope", 0), rope_scale_factor=case.get("factor", 1.0),
                          rope_scaling_yarn=int(case.get("yarn", False)), rope_original_context=4096 if case.get("yarn") else 0)
    return jev.KvPages(cfg, n_pages, page_tokens=case.get("page", 16), max_requests=requests, max_context=context,
                       max_tokens=tokens, rope_half=case.get("half", False))


def prepare(case, seed):
    rs = np.random.RandomState(seed % (1 << 32))
    gen = torch.Generator(device="cuda").manual_seed(seed)
    past, fresh = lengths(case)
    s = {"case": case, "past": past, "fresh": fresh}
    (_prepare_plan if case["kind"] == "plan" else _prepare_rows)(case, s, rs, gen)
    torch.cuda.synchronize()
    return s


def _prepare_plan(case, s, rs, gen):
    """Requests hold up to `over` tokens more than they keep; others hold pages and are not in the batch."""
    page, n = case["page"], case["requests"] + case["others"]
    held = np.concatenate([s["past"] + rs.randint(0, case["over"] + 1, case["requests"]), rs.randint(1, 900, case["others"])])
    ids = rs.permutation(n)  # batch row b (then the others) is request ids[b]
    context = int(case["past_hi"] + case["over"] + case["fresh_hi"]) + 900
    n_pages = int(_pages(held + case["fresh_hi"], page).sum()) + 64
    owned = _pages(held, page)
    table = np.full((n, _pages(context, page)), -1, np.int32)
    b = case["requests"]
    order = np.concatenate([np.arange(b, n), rs.permutation(b)])
    begin = np.concatenate([[0], owned[order].cumsum()])
    for i, r in enumerate(order):  # the first plan of an empty cache: lowest pages, in its batch's order
        table[r, :owned[r]] = np.arange(begin[i], begin[i + 1])
    s.update(n_pages=n_pages, tokens=int(s["fresh"].sum()) + case["pad"], request=_ints(ids[:b]), n_past=_ints(s["past"]),
             n_fresh=_ints(s["fresh"]))
    if own:
        cache = _cache(case, n_pages, n, context, int(max(held.sum(), s["tokens"])))
        ids, held = _ints(ids[order]), _ints(held[order])
        cache.plan_device(ids.data_ptr(), 0, held.data_ptr(), n, int(held.sum()))
        cache.sync()
        out = {"table": torch.empty((b, table.shape[1]), dtype=torch.int32, device="cuda")}
        for name in ("slot", "position", "row"):
            out[name] = torch.empty(s["tokens"], dtype=torch.int32, device="cuda")
        out["start"] = torch.empty(b + 1, dtype=torch.int32, device="cuda")
        s.update(cache=cache, out=out)
    else:
        s["table"] = _ints(table)


def _values(shape, gen, outliers=False):
    """Normal values; keys have a few channels that are several times larger, as trained models' keys do."""
    x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    if outliers:
        c = torch.randn(shape[-2:], generator=gen, device="cuda", dtype=torch.float32)
        x *= 0.5 + c * c
    return x


def _prepare_rows(case, s, rs, gen):
    page, past, fresh = case.get("page", 16), s["past"], s["fresh"]
    n, tokens, total = case["requests"], int(fresh.sum()), past + fresh
    q = _values((tokens, case["heads"], case["dim"]), gen)
    s.update(q=q, tokens=tokens)
    kv = (case["kv_heads"], case["dim"])
    context, n_pages = int(total.max()), int(_pages(total, page).sum()) + 8
    if case["kind"] != "rotate":
        s["k"], s["v"] = _values((tokens, *kv), gen, True), _values((tokens, *kv), gen)
    # what the requests' pages hold already: for `store` the begun blocks alone are read
    if case["kind"] == "store":
        begun = past % BLOCK
    elif case["kind"] == "attend":
        begun = past
    else:
        begun = past * 0
    old = int(begun.sum())
    old_k, old_v = _values((max(old, 1), *kv), gen, True)[:old], _values((max(old, 1), *kv), gen)[:old]
    s["scale"] = 1.0 / math.sqrt(case["dim"])
    if own:
        _fill_cache(case, s, past, begun, fresh, old_k, old_v, n_pages, context)
    else:
        _fill_plain(case, s, rs, begun, old_k, old_v, n_pages, context)


def _touched(slot_of, past, fresh):
    """Slots of every stored token of the blocks that the new tokens touch, request by request."""
    parts = [slot_of(r, np.arange(p // BLOCK * BLOCK, p + f)) for r, (p, f) in enumerate(zip(past, fresh))]
    return _ints(np.concatenate(parts))


def _fill_cache(case, s, past, begun, fresh, old_k, old_v, n_pages, context):
    """The package's cache with every request's `past` tokens, the last `begun` of them stored, and the batch planned."""
    n, tokens = case["requests"], s["tokens"]
    step = max(BLOCK, 16384 // n // BLOCK * BLOCK)  # the requests grow together, so their pages interleave
    cache = _cache(case, n_pages, n, context, max(tokens, n * step))
    ids, width = _ints(np.arange(n)), case["kv_heads"] * case["dim"]
    first, base, at = np.concatenate([[0], begun.cumsum()]), past - begun, past * 0
    while (at < past).any():
        goal = np.where(at < base, base, past)
        part = np.minimum(step, goal - at)
        kept, more = _ints(at), _ints(part)
        cache.plan_device(ids.data_ptr(), kept.data_ptr(), more.data_ptr(), n, int(part.sum()))
        if begun.any():
            lo = np.maximum(at - base, 0) + first[:-1]
            pick = torch.as_tensor(np.concatenate([np.arange(i, i + p) for i, p in zip(lo, part)]), device="cuda")
            pick = pick.clamp(max=len(old_k) - 1)  # tokens before the begun block hold whatever
            k, v = old_k[pick], old_v[pick]
            cache.store_device(0, 0, 0, k.data_ptr(), v.data_ptr(), width, 0)
            cache.sync()
        at = at + part
    table = torch.empty((n, _pages(context, case.get("page", 16))), dtype=torch.int32, device="cuda")
    kept, more = _ints(past), _ints(fresh)
    cache.plan_device(ids.data_ptr(), kept.data_ptr(), more.data_ptr(), n, tokens, table=table.data_ptr())
    if case["kind"] == "attend":
        cache.store_device(0, 0, 0, s["k"].data_ptr(), s["v"].data_ptr(), width, 0)
    cache.sync()
    s.update(cache=cache, out=torch.empty_like(s["q"]))
    if case["kind"] == "store":
        t, page = table.cpu().numpy().astype(np.int64), case["page"]
        s["read"] = _touched(lambda r, p: t[r, p // page] * page + p % page, past, fresh)
        shape = (len(s["read"]), case["kv_heads"], case["dim"])
        s["read_k"], s["read_v"] = torch.empty(shape, device="cuda"), torch.empty(shape, device="cuda")


def _fill_plain(case, s, rs, begun, old_k, old_v, n_pages, context):
    page, past, fresh = case.get("page", 16), s["past"], s["fresh"]
    n, total = case["requests"], s["past"] + s["fresh"]
    mp = _pages(context, page)
    table = np.full((n, mp), -1, np.int64)
    order, at = rs.permutation(n_pages), 0
    for r in range(n):
        need = _pages(total[r], page)
        table[r, :need] = order[at:at + need]
        at += need

    def slots(lo, hi):
        p = np.concatenate([np.arange(a, b) for a, b in zip(lo, hi)]) if n else np.zeros(0, np.int64)
        r = np.repeat(np.arange(n), hi - lo)
        return torch.as_tensor(table[r, p // page] * page + p % page, device="cuda"), torch.as_tensor(p, device="cuda"), torch.as_tensor(r, device="cuda")

    s["slot"], s["position"], s["row"] = slots(past, total)
    s["table"] = torch.as_tensor(table, device="cuda")
    if case["kind"] == "rotate":
        return
    shape = (n_pages * page // BLOCK, case["kv_heads"], BLOCK, case["dim"])
    s["pool"] = {name: (torch.zeros(shape, dtype=torch.int8, device="cuda"), torch.zeros(shape[:2], device="cuda")) for name in "kv"}
    if begun.sum():
        slot, position, _ = slots(past - begun, past)
        plan = _units(slot, position)
        if case["kind"] == "store":
            old_k = _rotate(case, old_k, position)
        _store(s["pool"]["k"], old_k, plan)
        _store(s["pool"]["v"], old_v, plan)
    s["units"] = _units(s["slot"], s["position"])
    if case["kind"] == "attend":
        _store(s["pool"]["k"], s["k"], s["units"])
        _store(s["pool"]["v"], s["v"], s["units"])
    else:
        s["read"] = _touched(lambda r, p: table[r, p // page] * page + p % page, past, fresh).long()


def _units(slot, position):
    """The blocks that tokens go to, the token in each of their places (-1: none), and whether a block was begun before."""
    block, unit = torch.unique(slot // BLOCK, return_inverse=True)
    where = torch.full((len(block), BLOCK), -1, dtype=torch.int64, device="cuda")
    where[unit, slot % BLOCK] = torch.arange(len(slot), device="cuda")
    return block, where, where[:, 0] < 0  # a block's tokens come in order: without its first token it was begun before


# ---------------------------------------------------------------- the plain forms


def _frequencies(case):
    """Pair frequencies and the factor on cos and sin (1e6 base, one over the scale where it is linear, ramped where it is YaRN)."""
    rd, base, factor = case["rope"], 1e6, case["factor"]
    plain = [math.pow(base, -2.0 * i / rd) for i in range(rd // 2)]
    if not case["yarn"]:
        return [f / factor for f in plain], 1.0

    def corr(rotations):
        return rd * math.log(4096 / (rotations * 2 * math.pi)) / (2 * math.log(base))

    low, high = max(0.0, math.floor(corr(32.0))), min(rd / 2 - 1.0, math.ceil(corr(1.0)))
    out = []
    for i, f in enumerate(plain):
        mix = 1.0 - min(1.0, max(0.0, (i - low) / max(0.001, high - low)))
        out.append(f / factor * (1.0 - mix) + f * mix)
    return out, 0.1 * math.log(factor) + 1.0


def _rotate(case, x, position):
    rd, half = case["rope"], case["half"]
    freq, mag = _frequencies(case)
    angle = position[:, None].double() * torch.tensor(freq, dtype=torch.float64, device="cuda")
    c, sn = (torch.cos(angle) * mag)[:, None], (torch.sin(angle) * mag)[:, None]
    out = x.clone()
    a, b = (x[..., :rd // 2], x[..., rd // 2:rd]) if half else (x[..., 0:rd:2], x[..., 1:rd:2])
    a, b = a.double(), b.double()
    ra, rb = (a * c - b * sn).float(), (a * sn + b * c).float()
    if half:
        out[..., :rd // 2], out[..., rd // 2:rd] = ra, rb
    else:
        out[..., 0:rd:2], out[..., 1:rd:2] = ra, rb
    return out


def _store(pool, x, units):
    codes, scales = pool
    block, where, begun = units
    new = (where >= 0)[:, None, :, None]
    x = torch.where(new, x[where.clamp(min=0)].transpose(1, 2), 0.0)  # [block, head, place, dim]
    finite = torch.isfinite(x).all(dim=3).all(dim=2)
    most = torch.full((), 127.0, device="cuda")  # on the device: by a host scalar torch multiplies with its reciprocal
    s_new = torch.where(finite, x.abs().amax(dim=(2, 3)) / most, math.nan)
    s_old = torch.where(begun[:, None], scales[block], 0.0)
    s = torch.maximum(s_old, s_new)
    by = s.double()[:, :, None, None]  # 64-bit quotients: an exact half is seen as one
    kept = torch.where(begun[:, None, None, None], codes[block].double() * s_old.double()[:, :, None, None], 0.0)
    q = torch.round(torch.where(new, x.double(), kept) / by).clamp(-127, 127)
    codes[block] = torch.where(by > 0, q, 0.0).to(torch.int8)
    scales[block] = s


def _read(pool, slot):
    codes, scales = pool
    return codes[slot // BLOCK, :, slot % BLOCK].float() * scales[slot // BLOCK][:, :, None]


def _plan(s):
    page, table, past, fresh = s["case"]["page"], s["table"], s["n_past"].long(), s["n_fresh"].long()
    b, width = len(past), table.shape[1]
    col = torch.arange(width, device="cuda")
    keep, need = (past + page - 1) // page, (past + fresh + page - 1) // page
    live = table >= 0
    live[:b] &= col < keep[:, None]
    used = torch.zeros(s["n_pages"] + 1, dtype=torch.bool, device="cuda")
    used[torch.where(live, table, s["n_pages"]).long().flatten()] = True
    free = ~used[:-1]
    by_rank = torch.zeros(s["n_pages"] + 1, dtype=torch.int64, device="cuda")
    by_rank[torch.where(free, torch.cumsum(free, 0) - 1, s["n_pages"])] = torch.arange(s["n_pages"], device="cuda")
    want = (col >= keep[:, None]) & (col < need[:, None])
    rank = (torch.cumsum(want.flatten(), 0) - 1).clamp(min=0).reshape(b, width)
    out = torch.where(want, by_rank[rank], torch.where(live[:b], table[:b].long(), -1))
    start = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), torch.cumsum(fresh, 0)])
    t = torch.arange(s["tokens"], device="cuda")
    row = torch.searchsorted(start, t, right=True) - 1
    inside = row < b
    row = row.clamp(max=b - 1)
    position = past[row] + t - start[row]
    slot = out[row, (position // page).clamp(max=width - 1)] * page + position % page
    res = {"table": out, "slot": torch.where(inside, slot, -1), "position": torch.where(inside, position, -1),
           "row": torch.where(inside, row, -1), "start": start}
    return {k: v.to(torch.int32) for k, v in res.items()}


def _attend(s):
    case = s["case"]
    h, d, g, page = case["kv_heads"], case["dim"], case["heads"] // case["kv_heads"], case["page"]
    table, row, position = s["table"], s["row"], s["position"]
    n, width = table.shape
    sub = page // BLOCK
    blocks = (table.clamp(min=0)[:, :, None] * sub + torch.arange(sub, device="cuda")).reshape(n, width * sub)
    keys, values = (pool[0][blocks].float() * pool[1][blocks][..., None, None] for pool in (s["pool"]["k"], s["pool"]["v"]))
    length = width * page
    keys = keys.permute(0, 2, 4, 1, 3).reshape(n, h, d, length)  # [request, head, dim, key]
    values = values.permute(0, 2, 1, 3, 4).reshape(n, h, length, d)
    first = torch.searchsorted(row, torch.arange(n, device="cuda"))
    place = torch.arange(len(row), device="cuda") - first[row]
    most = int(s["fresh"].max())
    q = torch.zeros((n, most, h * g, d), device="cuda")
    q[row, place] = s["q"]
    last = torch.full((n, most), length - 1, device="cuda")
    last[row, place] = position
    q = q.reshape(n, most, h, g, d).permute(0, 2, 1, 3, 4).reshape(n, h, most * g, d)
    p = torch.matmul(q, keys).mul_(s["scale"]).reshape(n, h, most, g, length)
    p.masked_fill_((torch.arange(length, device="cuda") > last[:, :, None])[:, None, :, None], -math.inf)
    p = p.sub_(p.amax(dim=-1, keepdim=True)).exp_()
    p = p.div_(p.sum(dim=-1, keepdim=True))
    o = torch.matmul(p.reshape(n, h, most * g, length), values)
    o = o.reshape(n, h, most, g, d).permute(0, 2, 1, 3, 4).reshape(n, most, h * g, d)
    return o[row, place]


def run(s):
    case = s["case"]
    kind = case["kind"]
    if own:
        return _run_own(s, kind)
    if kind == "plan":
        return _plan(s)
    if kind == "rotate":
        return _rotate(case, s["q"], s["position"])
    if kind == "attend":
        return _attend(s)
    q = _rotate(case, s["q"], s["position"])
    _store(s["pool"]["k"], _rotate(case, s["k"], s["position"]), s["units"])
    _store(s["pool"]["v"], s["v"], s["units"])
    return {"q": q, "k": _read(s["pool"]["k"], s["read"]), "v": _read(s["pool"]["v"], s["read"])}


def _run_own(s, kind):
    case, cache = s["case"], s["cache"]
    out = s["out"]
    if kind == "plan":
        cache.plan_device(s["request"].data_ptr(), s["n_past"].data_ptr(), s["n_fresh"].data_ptr(), case["requests"], s["tokens"],
                          table=out["table"].data_ptr(), slot=out["slot"].data_ptr(), position=out["position"].data_ptr(),
                          row=out["row"].data_ptr(), start=out["start"].data_ptr())
        return out
    if kind == "attend":
        cache.attend_device(0, s["q"].data_ptr(), out.data_ptr())
        return out
    width = case["heads"] * case["dim"]
    if kind == "rotate":
        cache.store_device(0, s["q"].data_ptr(), width, 0, 0, 0, out.data_ptr())
        return out
    cache.store_device(0, s["q"].data_ptr(), width, s["k"].data_ptr(), s["v"].data_ptr(), case["kv_heads"] * case["dim"], out.data_ptr())
    cache.read_device(0, s["read"].data_ptr(), len(s["read"]), s["read_k"].data_ptr(), s["read_v"].data_ptr())
    return {"q": out, "k": s["read_k"], "v": s["read_v"]}


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
    past, fresh = lengths(case)
    tokens = int(fresh.sum())
    if case["kind"] == "plan":
        width = _pages(int(case["past_hi"] + case["over"] + case["fresh_hi"]) + 900, case["page"])
        b, kept = case["requests"], int(_pages(past, case["page"]).sum())
        return {"bytes": 12.0 * b + 4.0 * kept + 4.0 * b * width + 12.0 * (tokens + case["pad"]) + 4.0 * (b + 1),
                "flops": float(tokens + b)}
    q, kv = case["heads"] * case["dim"], case["kv_heads"] * case["dim"]
    if case["kind"] == "rotate":
        return {"bytes": 8.0 * tokens * q, "flops": 3.0 * tokens * case["heads"] * case["rope"]}
    if case["kind"] == "store":
        touched = int((past % BLOCK).sum()) + tokens
        # queries in and out; keys and values in, their bytes out; the touched blocks back as floats
        return {"bytes": 8.0 * tokens * q + 2 * kv * (4.0 * tokens + tokens + touched + 4.0 * touched),
                "flops": 3.0 * tokens * (case["heads"] + case["kv_heads"]) * case["rope"] + 6.0 * touched * kv}
    total = past + fresh
    blocks = -(-total // BLOCK)
    pairs = float((fresh * past + fresh * (fresh + 1) // 2).sum())
    return {"bytes": 2.0 * kv * float(total.sum()) + 8.0 * case["kv_heads"] * float(blocks.sum()) + 8.0 * tokens * q, "flops": 4.0 * q * pairs}


# ---------------------------------------------------------------- the same in 64 bits


def _exact_rotated(case, x, pos):
    rd, base = case["rope"], 1e6
    n = rd // 2
    freq = [math.pow(base, -2.0 * i / rd) for i in range(n)]
    mag = 1.0
    if case["yarn"]:
        dims = [rd * math.log(4096 / (r * 2 * math.pi)) / (2 * math.log(base)) for r in (32.0, 1.0)]
        lo, hi = max(0.0, math.floor(dims[0])), min(n - 1.0, math.ceil(dims[1]))
        ramp = [min(1.0, max(0.0, (i - lo) / max(0.001, hi - lo))) for i in range(n)]
        freq = [f / case["factor"] * r + f * (1.0 - r) for f, r in zip(freq, ramp)]
        mag = 1.0 + 0.1 * math.log(case["factor"])
    else:
        freq = [f / case["factor"] for f in freq]
    turn = torch.polar(torch.full((len(pos), 1, n), mag, dtype=torch.float64, device="cuda"),
                       torch.as_tensor(pos, dtype=torch.float64, device="cuda")[:, None, None] * torch.tensor(freq, dtype=torch.float64, device="cuda"))
    x = x.double()
    head, tail = x[..., :rd], x[..., rd:]
    if case["half"]:
        z = torch.complex(head[..., :n], head[..., n:]) * turn
        head = torch.cat([z.real, z.imag], dim=-1)
    else:
        z = torch.complex(head[..., 0::2].contiguous(), head[..., 1::2].contiguous()) * turn
        head = torch.stack([z.real, z.imag], dim=-1).flatten(-2)
    return torch.cat([head, tail], dim=-1)


def _exact_values(old, new, begun):
    """The values that a request's touched blocks stand for after `begun` tokens and then the new ones were stored."""
    x = torch.cat([old, new]).float().double()  # what is stored is rounded to 32 bits once
    pad = -len(x) % BLOCK
    t = torch.arange(len(x) + pad, device="cuda")
    x = torch.cat([x, x.new_zeros((pad, *x.shape[1:]))]).reshape(-1, BLOCK, *x.shape[1:])

    def scale(mask):
        return ((x.abs() * mask).amax(dim=(1, 3)) / x.new_full((), 127.0)).float().double()[:, None, :, None]  # a scale is held in 32 bits

    def divided(a, by):
        return torch.where(by > 0, a / by, torch.zeros_like(a))

    was = (t < begun).reshape(-1, BLOCK, 1, 1)
    s0, s1 = scale(was), scale(~was)
    s = torch.maximum(s0, s1)
    q = torch.where(was, divided(torch.round(divided(x, s0)) * s0, s), divided(x, s))
    y = torch.round(q) * s
    return y.reshape(-1, *y.shape[2:])[:len(y) * BLOCK - pad]


def exact(case, seed):
    if case["kind"] == "plan":
        return None
    gen = torch.Generator(device="cuda").manual_seed(seed)
    past, fresh = lengths(case)
    tokens, kv = int(fresh.sum()), (case["kv_heads"], case["dim"])
    q = _values((tokens, case["heads"], case["dim"]), gen)
    total = past + fresh
    position = np.concatenate([np.arange(a, b) for a, b in zip(past, total)])
    if case["kind"] == "rotate":
        return _exact_rotated(case, q, position)
    k, v = _values((tokens, *kv), gen, True), _values((tokens, *kv), gen)
    begun = past % BLOCK if case["kind"] == "store" else past
    old = int(begun.sum())
    old_k, old_v = _values((max(old, 1), *kv), gen, True)[:old], _values((max(old, 1), *kv), gen)[:old]
    if case["kind"] == "store":
        old_pos = np.concatenate([np.arange(a - b, a) for a, b in zip(past, begun)])
        k, old_k = _exact_rotated(case, k, position), _exact_rotated(case, old_k, old_pos)
        q = _exact_rotated(case, q, position)
    a, f = np.concatenate([[0], begun.cumsum()]), np.concatenate([[0], fresh.cumsum()])
    keys = [_exact_values(old_k[a[r]:a[r + 1]], k[f[r]:f[r + 1]], int(begun[r])) for r in range(len(past))]
    values = [_exact_values(old_v[a[r]:a[r + 1]], v[f[r]:f[r + 1]], int(begun[r])) for r in range(len(past))]
    if case["kind"] == "store":
        return {"q": q, "k": torch.cat(keys), "v": torch.cat(values)}
    if work(case)["flops"] > 6e12:
        return None
    out = []
    g = case["heads"] // case["kv_heads"]
    for r in range(len(past)):
        kr, vr = keys[r].permute(1, 2, 0).contiguous(), values[r].transpose(0, 1).contiguous()
        for lo in range(0, int(fresh[r]), 256):
            hi = min(int(fresh[r]), lo + 256)
            x = q[f[r] + lo:f[r] + hi].double().reshape(hi - lo, case["kv_heads"], g, -1).permute(1, 0, 2, 3)
            w = torch.matmul(x.reshape(case["kv_heads"], (hi - lo) * g, -1), kr) / math.sqrt(case["dim"])
            hidden = torch.arange(int(total[r]), device="cuda") > torch.arange(int(past[r]) + lo, int(past[r]) + hi, device="cuda").repeat_interleave(g)[:, None]
            w = torch.softmax(w.masked_fill(hidden, -math.inf), dim=-1)
            o = torch.matmul(w, vr).reshape(case["kv_heads"], hi - lo, g, -1).permute(1, 0, 2, 3)
            out.append(o.reshape(hi - lo, case["heads"], -1))
    return torch.cat(out)
