"""Measured cases of the search over codings that branch off one decoded state.

An encoder (or a decoder of hypotheses) that searches keeps several branches of
one stream, its beams.  A step of it needs, beside what the cache has already:

* ``select``  -- from every beam's logits and score so far, the best
  continuations of each stream: their scores, parents and tokens;
* ``reorder`` -- the cache's streams follow that choice in place: stream i goes
  on from what stream parents[i] of its group held, full pages shared, partly
  filled last pages copied where two go on from one;
* ``attend``  -- attention of the beams' new tokens, which reads the pages that
  a group's tables begin with alike once for all of the group.

``run`` computes them in elementary torch operations, or with the framework's
own calls when ``own`` is set.  ``exact`` is written apart from it, in 64 bits,
from the definitions.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}


def _package():
    import __graft_entry__
    return __graft_entry__.load_package()


# ------------------------------------------------------------------ cases ----

def listed():
    return [
        # one stream's symbol, four branches, an alphabet of byte symbols (latency)
        {"name": "select_symbols_1_stream", "op": "select", "streams": 1, "beams": 4, "vocab": 256, "count": 4,
         "dtype": "f32", "padded": 0, "finished": False, "masked": False},
        # the first step of 16 streams: one live beam spreads into eight; an odd alphabet
        {"name": "select_first_step", "op": "select", "streams": 16, "beams": 1, "vocab": 4099, "count": 8,
         "dtype": "f16", "padded": 0, "finished": False, "masked": False},
        # a step of 64 streams with eight branches each; rows of logits in a padded buffer
        {"name": "select_64_streams", "op": "select", "streams": 64, "beams": 8, "vocab": 32768, "count": 8,
         "dtype": "bf16", "padded": 64, "finished": False, "masked": False},
        # odd rows in 32 bits, some tokens forbidden, some beams ended
        {"name": "select_masked_f32", "op": "select", "streams": 24, "beams": 5, "vocab": 65537, "count": 10,
         "dtype": "f32", "padded": 0, "finished": True, "masked": True},
        # wide search over a large vocabulary
        {"name": "select_wide", "op": "select", "streams": 32, "beams": 16, "vocab": 131072, "count": 32,
         "dtype": "bf16", "padded": 0, "finished": True, "masked": False},
        # one stream's four branches over less than a 626x352 frame of latent tokens (latency)
        {"name": "reorder_1_stream", "op": "reorder", "groups": 1, "beams": 4, "past": 439, "own": 21, "ragged": False,
         "layers": 2, "hk": 2, "dim": 64, "page": 16},
        # 16 streams x 8 branches, eight layers
        {"name": "reorder_16_streams", "op": "reorder", "groups": 16, "beams": 8, "past": 2 * 880, "own": 300,
         "ragged": True, "layers": 8, "hk": 4, "dim": 128, "page": 64},
        # the smallest attention: four branches of one stream over two 626x352 frames
        {"name": "attend_4_branches", "op": "attend", "groups": 1, "beams": 4, "past": 2 * 880, "own": 9, "new": 1,
         "ragged": False, "layers": 1, "hq": 8, "hk": 2, "dim": 64, "page": 16, "window": 0, "sinks": 0,
         "dtype": "f16"},
        # eight streams of eight branches, four layers, two 1920x1088 frames at most
        {"name": "attend_8_streams_8_branches", "op": "attend", "groups": 8, "beams": 8, "past": 2 * 8160, "own": 61,
         "new": 1, "ragged": True, "layers": 4, "hq": 16, "hk": 4, "dim": 128, "page": 64, "window": 0, "sinks": 0,
         "dtype": "bf16"},
        # a window of one 1920x1088 frame and 16 sinks, pairs of tokens, three queries to a key head
        {"name": "attend_window_sinks", "op": "attend", "groups": 3, "beams": 5, "past": 4 * 8160 + 5, "own": 203,
         "new": 2, "ragged": True, "layers": 1, "hq": 6, "hk": 2, "dim": 128, "page": 32, "window": 8160, "sinks": 16,
         "dtype": "f16"},
        # 16 branches of one stream, eight key heads
        {"name": "attend_16_branches", "op": "attend", "groups": 1, "beams": 16, "past": 2 * 8160, "own": 130, "new": 1,
         "ragged": False, "layers": 2, "hq": 32, "hk": 8, "dim": 128, "page": 64, "window": 0, "sinks": 0,
         "dtype": "bf16"},
        # the widest: 64 branches over eight 1920x1088 frames, eight queries to a key head
        {"name": "attend_64_branches", "op": "attend", "groups": 1, "beams": 64, "past": 8 * 8160, "own": 40, "new": 1,
         "ragged": False, "layers": 1, "hq": 64, "hk": 8, "dim": 128, "page": 128, "window": 0, "sinks": 0,
         "dtype": "bf16"},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["select", "select", "reorder", "attend", "attend"])
    if op == "select":
        dtype = rng.choice(["f32", "f16", "bf16"])
        streams, beams = _log(rng, 1, 64), _log(rng, 1, 32)
        vocab = _log(rng, 64, 131072)
        # no more logits than the largest listed call has bytes of
        vocab = max(33, min(vocab, 134217728 // (streams * beams * SIZES[dtype])))
        return {"op": op, "streams": streams, "beams": beams, "vocab": vocab, "count": rng.randint(1, 32),
                "dtype": dtype, "padded": rng.choice([0, 0, 8, 37]), "finished": rng.random() < 0.4,
                "masked": rng.random() < 0.4}
    dim, page, hk = rng.choice([64, 128]), rng.choice([16, 32, 64, 128]), rng.choice([1, 2, 4, 8])
    groups, beams = _log(rng, 1, 16), _log(rng, 2, 64)
    if op == "reorder":
        own_tokens = rng.randint(1, 400)
        layers = rng.randint(1, 8)
        # the pool stays in reach of the largest listed one
        while groups * beams * (own_tokens + 2 * page) * hk * dim * 2 * layers > 900000000:
            groups, beams = max(1, groups // 2), max(2, beams // 2)
        return {"op": op, "groups": groups, "beams": beams, "past": rng.randint(0, 2040), "own": own_tokens,
                "ragged": rng.random() < 0.5, "layers": layers, "hk": hk, "dim": dim, "page": page}
    group, new = rng.choice([1, 2, 3, 4, 5, 6, 8]), rng.choice([1, 1, 1, 2, 3, 5])
    past, own_tokens, layers = _log(rng, 16, 65280), rng.randint(new, 400), rng.randint(1, 2)
    # bounded by the cache and the products of the largest listed step
    while (groups * beams * new * past * hk * group * dim * layers > 3.2e10 or
           (groups * past + groups * beams * own_tokens) * hk * dim * 2 * layers > 150000000):
        if groups > 1 and rng.random() < 0.5:
            groups //= 2
        else:
            past = max(16, past // 2)
            beams = max(2, beams * 3 // 4)
    window = _log(rng, 1, 8160) if rng.random() < 0.4 else 0
    return {"op": op, "groups": groups, "beams": beams, "past": past, "own": own_tokens, "new": new,
            "ragged": rng.random() < 0.5, "layers": layers, "hq": hk * group, "hk": hk, "dim": dim, "page": page,
            "window": window, "sinks": rng.randint(0, 64) if window else 0, "dtype": rng.choice(["f16", "bf16"])}


# ----------------------------------------------------------------- lengths ----

def _share(b):
    """Fixed spread over (0, 1]."""
    return ((b * 37 + 11) % 64 + 1) / 64


def _past(case):
    """Tokens that a group's beams have in common."""
    if not case["ragged"]:
        return [case["past"]] * case["groups"]
    return [int(case["past"] * _share(g)) for g in range(case["groups"])]


def _own(case):
    """Each beam's own tokens; beams of one group that ended earlier are shorter."""
    new, n = case.get("new", 1), case["groups"] * case["beams"]
    if not case["ragged"]:
        return [case["own"]] * n
    return [max(new, int(case["own"] * (0.5 + 0.5 * _share(b)))) for b in range(n)]


def _lengths(case):
    past = _past(case)
    return [past[i // case["beams"]] + n for i, n in enumerate(_own(case))]


def _parents(case, seed):
    """A choice as a search makes it: most children come from the best beams."""
    rng = np.random.default_rng(seed + 29)
    k = case["beams"]
    weight = np.exp(-np.arange(k) / max(1.0, k / 3))
    return rng.choice(k, (case["groups"], k), p=weight / weight.sum()).astype(np.int32)


def _copies(case):
    """About how many last pages are copied: children past the first of each parent, over many choices."""
    k = case["beams"]
    weight = np.exp(-np.arange(k) / max(1.0, k / 3))
    weight /= weight.sum()
    return k - float((1 - (1 - weight) ** k).sum())


def work(case):
    op = case["op"]
    if op == "select":
        rows = case["streams"] * case["beams"]
        if case["finished"]:
            rows -= sum(_ended(case, i) for i in range(rows))
        out = case["streams"] * case["count"] * 12
        return {"bytes": rows * case["vocab"] * SIZES[case["dtype"]] + case["streams"] * case["beams"] * 5 + out,
                "flops": rows * case["vocab"] * 4}
    lengths, page = _lengths(case), case["page"]
    token = 2 * case["hk"] * case["dim"] * case["layers"]
    if op == "reorder":
        rest = sum(n % page for n in lengths) / len(lengths)
        entries = sum(-(-n // page) for n in lengths)
        return {"bytes": int(2 * _copies(case) * case["groups"] * rest * token + 8 * entries) + 1,
                "flops": int(case["groups"] * rest * token) + 1}
    window, sinks, new, group = case["window"], case["sinks"], case["new"], case["hq"] // case["hk"]
    keys = pairs = 0
    past = _past(case)
    for g in range(case["groups"]):
        mine = lengths[g * case["beams"]:(g + 1) * case["beams"]]
        low = max(0, min(mine) - new - window + 1) if window else 0
        common = max(0, past[g] - low) + min(sinks, low, past[g])
        keys += common + sum(n - max(past[g], low) for n in mine)
        for n in mine:
            for i in range(new):
                a = n - new + i
                first = max(0, a - window + 1) if window else 0
                pairs += a - first + 1 + min(sinks, first)
    rows = sum(1 for _ in lengths) * new * case["hq"]
    return {"bytes": keys * token + 2 * rows * case["dim"] * 2 * case["layers"],
            "flops": pairs * group * case["hk"] * case["dim"] * 4 * case["layers"]}


# ------------------------------------------------------------------ inputs ----

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ended(case, i):
    return i % case["beams"] > 0 and (i * 7 + 3) % 5 == 0


def _select_inputs(case, seed):
    gen = _gen(seed)
    b, k, v = case["streams"], case["beams"], case["vocab"]
    dtype = DTYPES[case["dtype"]]
    logits = torch.empty((b, k, v + case["padded"]), dtype=dtype, device="cuda")
    for i in range(b):
        # a few likely tokens over a broad floor, as a trained model's last product gives
        x = torch.randn((k, v + case["padded"]), device="cuda", generator=gen)
        logits[i] = (x * 2.0 + (x > 3.0) * (x - 3.0) * 6.0 - 1.5).to(dtype)
    logits = logits[..., :v]
    if case["masked"]:
        # forbidden tokens: a stretch of the alphabet, another one for each beam
        for j in range(k):
            logits[:, j, (j * 977) % v::13] = float("-inf")
    steps = torch.randn((b, k), device="cuda", generator=gen).mul_(2.0).sub_(20.0)
    finished = torch.tensor([bool(case["finished"] and _ended(case, i)) for i in range(b * k)], device="cuda")
    return {"logits": logits, "scores": steps, "finished": finished.view(b, k) if case["finished"] else None}


def _ints(shape, gen):
    """Stored integers as quantised normal activations have them."""
    out = torch.empty(shape, dtype=torch.int8, device="cuda")
    flat = out.view(-1)
    step = 1 << 27
    for i in range(0, flat.numel(), step):
        part = flat[i:i + step]
        part.copy_(torch.randn(part.numel(), device="cuda", generator=gen).mul_(36.0).round_().clamp_(-127, 127))
    return out


def _cache_inputs(case, seed):
    """A pool where the beams of a group share the pages of their common tokens."""
    gen = _gen(seed)
    page, k = case["page"], case["beams"]
    past, lengths = _past(case), _lengths(case)
    counts = [-(-n // page) for n in lengths]
    common = [p // page for p in past]
    pages = sum(common) + sum(c - common[i // k] for i, c in enumerate(counts))
    # free ones as well: no reorder needs more than one for each stream
    pages += len(lengths) if case["op"] == "reorder" else 5
    order = np.random.default_rng(seed).permutation(pages).astype(np.int32)
    table = np.full((len(lengths), max(counts) + 1), -1, np.int32)
    refs = np.zeros(pages, np.int32)
    at = 0
    for g, c in enumerate(common):
        table[g * k:(g + 1) * k, :c] = order[at:at + c]
        refs[order[at:at + c]] = k
        at += c
    for i, n in enumerate(counts):
        c = common[i // k]
        table[i, c:n] = order[at:at + n - c]
        refs[order[at:at + n - c]] = 1
        at += n - c
    scale = torch.exp(torch.randn((case["layers"], pages, 2, case["hk"]), device="cuda", generator=gen) * 0.3)
    return {"kv": _ints((case["layers"], pages, 2, case["hk"], page, case["dim"]), gen), "scale": scale * (3.5 / 127.0),
            "table": torch.from_numpy(table).cuda(), "refs": torch.from_numpy(refs).cuda(),
            "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda"), "gen": gen}


def _inputs(case, seed):
    if case["op"] == "select":
        return _select_inputs(case, seed)
    x = _cache_inputs(case, seed)
    if case["op"] == "reorder":
        x["parents"] = torch.from_numpy(_parents(case, seed)).cuda()
        return x
    tokens = case["groups"] * case["beams"] * case["new"]
    # queries are a slice of the projection that makes keys and values too
    qkv = torch.randn((case["layers"], tokens, case["hq"] + 2 * case["hk"], case["dim"]), device="cuda",
                      generator=x["gen"])
    x["q"] = (qkv * 1.5).to(DTYPES[case["dtype"]])[:, :, :case["hq"]]
    return x


def prepare(case, seed):
    x = _inputs(case, seed)
    x.pop("gen", None)
    state = {"case": case, **x}
    if case["op"] == "select":
        return state
    k, n = case["beams"], case["groups"] * case["beams"]
    if own:
        ufb = _package()
        layers, pages = x["kv"].shape[:2]
        cache = ufb.KVCache(layers=layers, pages=pages, heads=case["hk"], head_dim=case["dim"],
                            page_tokens=case["page"], slots=n, table_width=x["table"].shape[1], device="cuda")
        for name in ("kv", "scale", "table", "refs", "lengths"):
            getattr(cache, name).copy_(x[name])
            del state[name]
        state["cache"] = cache
        if case["op"] == "reorder":
            state["plan"] = cache.beam_plan(list(range(n)), k)
        else:
            state["plan"] = cache.plan(list(range(n)), [case["new"]] * n)
            state["groups"] = cache.group_plan(state["plan"], [k] * case["groups"])
    elif case["op"] == "attend":
        common = [p // case["page"] for p in _past(case)]
        state["common"] = torch.tensor(common, device="cuda")
        state["widest"] = max(common)
        state["longest"] = max(-(-n // case["page"]) - common[i // k] for i, n in enumerate(_lengths(case)))
    return state


# ------------------------------------------------------------- plain forms ----

def _ordered(x):
    """Integers in the order of the 32-bit floats x, equal zeros among them."""
    bits = (x + 0.0).view(torch.int32)
    return torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()


def _plain_select(state):
    case, scores, finished = state["case"], state["scores"], state["finished"]
    v = case["vocab"]
    b, k = scores.shape
    x = state["logits"]
    each, count = min(case["count"], v), min(case["count"], k * v)
    # the best of each beam: larger logits first, then lower tokens
    key = (_ordered(x.float()) << 32) + (0xFFFFFFFF - torch.arange(v, device=x.device))
    token = 0xFFFFFFFF - (key.topk(each, -1).values & 0xFFFFFFFF)
    del key
    # 64 bits: totals of different beams are next to each other, and their order is the result
    x = x.double()
    logit = x.gather(-1, token)
    top = x.amax(-1, keepdim=True)
    lse = top + (x - top).exp_().sum(-1, keepdim=True).log()
    total = (scores.double()[..., None] + (logit - lse)).float()
    live = torch.isfinite(top[..., 0]) & (scores > -math.inf)
    if finished is not None:
        live &= ~finished
    total.masked_fill_(~live[..., None], -math.inf)
    if finished is not None:
        total[..., 0] = torch.where(finished, scores, total[..., 0])
        token[..., 0].masked_fill_(finished, 0)
    # of all beams: higher totals first, then lower beams and a beam's own order
    total, token = total.view(b, -1), token.view(b, -1)
    key = (_ordered(total) << 32) + (0xFFFFFFFF - torch.arange(k * each, device=x.device))
    at = 0xFFFFFFFF - (key.topk(min(count, k * each), -1).values & 0xFFFFFFFF)
    total = total.gather(1, at)
    none = total == -math.inf
    rank = torch.arange(total.shape[1], device=total.device).clamp(max=k - 1)
    parents = torch.where(none, rank, at // each).int()
    tokens = torch.where(none, 0, token.gather(1, at)).int()
    return total, parents, tokens


def _plain_reorder(state):
    case = state["case"]
    kv, scale, table, refs, lengths = (state[n] for n in ("kv", "scale", "table", "refs", "lengths"))
    n, page = lengths.numel(), case["page"]
    slot = torch.arange(n, device=table.device)
    src = (slot // case["beams"] * case["beams"] + state["parents"].flatten()).long()
    rows, length = table[src], lengths[src]
    full, rest = (length // page).long(), length % page
    # the last page stays with the parent itself, else with its first child
    order = torch.where(src == slot, -1, slot)
    first = torch.full_like(slot, n).scatter_reduce_(0, src, order, "amin")
    split = torch.nonzero((rest > 0) & (order != first[src]))[:, 0]
    last = table.gather(1, (lengths // page).long()[:, None])[:, 0]
    left = last[(first == n) & (lengths % page > 0)].long()
    free = torch.nonzero(refs == 0)[:, 0]
    fresh = torch.cat([left, free])[:split.numel()]
    origin = rows[split, full[split]].long()
    rows[split, full[split]] = fresh.int()
    held = table[table >= 0].long()
    refs.index_add_(0, held, torch.full_like(held, -1, dtype=torch.int32))
    held = rows[rows >= 0].long()
    refs.index_add_(0, held, torch.ones_like(held, dtype=torch.int32))
    keep = (torch.arange(page, device=table.device) < rest[split][:, None])[None, :, None, None, :, None]
    kv[:, fresh] = torch.where(keep, kv[:, origin], kv[:, fresh])
    scale[:, fresh] = scale[:, origin]
    table.copy_(rows)
    lengths.copy_(length)
    return table, refs, lengths, kv, scale


def _seen(case, key, at, length):
    seen = (key <= at) & (key < length)
    if case["window"]:
        seen &= (key > at - case["window"]) | (key < case["sinks"])
    return seen


def _plain_attend(state):
    """Both parts of the keys, the common ones once for all rows of a group."""
    case = state["case"]
    g, k, new, hk, dim = case["groups"], case["beams"], case["new"], case["hk"], case["dim"]
    group, page = case["hq"] // hk, case["page"]
    table, common, wide, long = state["table"], state["common"], state["widest"], state["longest"]
    dev = table.device
    length = state["lengths"].view(g, 1, k, 1, 1).long()
    at = length - new + torch.arange(new, device=dev).repeat_interleave(group)[:, None]
    first = table.view(g, k, -1)[:, 0, :wide].clamp(min=0).long()
    column = common.repeat_interleave(k)[:, None] + torch.arange(long, device=dev)
    rest = table.gather(1, column.clamp(max=table.shape[1] - 1)).clamp(min=0).long()
    key1 = torch.arange(wide * page, device=dev)
    seen1 = _seen(case, key1, at, common.view(g, 1, 1, 1, 1) * page)
    key2 = common.view(g, 1, 1, 1, 1) * page + torch.arange(long * page, device=dev)
    seen2 = _seen(case, key2, at, length)
    result = []
    for layer in range(case["layers"]):
        kv, scale, q = state["kv"][layer], state["scale"][layer], state["q"][layer]
        pre = kv[first].float() * scale[first][..., None, None]
        pre = pre.permute(2, 0, 3, 1, 4, 5).reshape(2, g, hk, 1, wide * page, dim)
        mine = kv[rest].float() * scale[rest][..., None, None]
        mine = mine.view(g, k, long, 2, hk, page, dim).permute(3, 0, 4, 1, 2, 5, 6).reshape(2, g, hk, k, long * page, dim)
        rows = q.float().view(g, k, new, hk, group, dim).permute(0, 3, 1, 2, 4, 5).reshape(g, hk, k, new * group, dim)
        flat = rows.reshape(g, hk, 1, k * new * group, dim)
        s1 = torch.matmul(flat, pre[0].mT).view(g, hk, k, new * group, wide * page)
        s = torch.cat([s1, torch.matmul(rows, mine[0].mT)], -1)
        s *= dim ** -0.5
        s.masked_fill_(~torch.cat([seen1, seen2], -1), -math.inf)
        s -= s.amax(-1, keepdim=True)
        s.exp_()
        total = s.sum(-1, keepdim=True)
        p1 = s[..., :wide * page].reshape(g, hk, 1, k * new * group, wide * page)
        o = torch.matmul(p1, pre[1]).view(g, hk, k, new * group, dim)
        o = (o + torch.matmul(s[..., wide * page:], mine[1])) / total
        o = o.view(g, hk, k, new, group, dim).permute(0, 2, 3, 1, 4, 5).reshape(q.shape)
        result.append(o.to(q.dtype))
    return result


def run(state):
    case = state["case"]
    op = case["op"]
    if op == "select":
        if own:
            return _package().beam_select(state["logits"], state["scores"], case["count"], finished=state["finished"])
        return _plain_select(state)
    if op == "reorder":
        if own:
            c = state["cache"]
            c.reorder(state["plan"], state["parents"])
            return c.table, c.refs, c.lengths, c.kv, c.scale
        return _plain_reorder(state)
    if own:
        c = state["cache"]
        # once a step, for all layers
        c.share(state["groups"])
        return [c.attend(layer, state["plan"], state["q"][layer], window=case["window"], sinks=case["sinks"],
                         groups=state["groups"]) for layer in range(case["layers"])]
    return _plain_attend(state)


# ------------------------------------------------------------------- exact ----

def _exact_select(case, x):
    scores, parents, tokens = [], [], []
    for b in range(case["streams"]):
        names, totals = [], []
        for k in range(case["beams"]):
            base = x["scores"][b, k].double()
            if x["finished"] is not None and bool(x["finished"][b, k]):
                names.append(torch.tensor([k * case["vocab"]], device="cuda"))
                totals.append(base[None])
                continue
            t = base + torch.log_softmax(x["logits"][b, k].double(), -1)
            # no more of one beam than are asked for, in the order of their logits and tokens
            order = torch.sort(x["logits"][b, k].double(), descending=True, stable=True).indices[:case["count"]]
            order = order[t[order] > -math.inf]
            names.append(order + k * case["vocab"])
            totals.append(t[order])
        name, total = torch.cat(names), torch.cat(totals)
        order = torch.sort(total.float(), descending=True, stable=True).indices[:case["count"]]
        n, most = order.numel(), min(case["count"], case["beams"] * case["vocab"])
        fill = torch.arange(n, most, device="cuda").clamp(max=case["beams"] - 1)
        scores.append(torch.cat([total[order], torch.full((most - n,), -math.inf, device="cuda", dtype=torch.float64)]))
        parents.append(torch.cat([torch.div(name[order], case["vocab"], rounding_mode="floor"), fill]))
        tokens.append(torch.cat([name[order] % case["vocab"], fill * 0]))
    return torch.stack(scores), torch.stack(parents), torch.stack(tokens)


def _exact_reorder(case, x):
    before, refs = x["table"].cpu().numpy(), x["refs"].cpu().numpy()
    lengths, parents = x["lengths"].cpu().numpy(), x["parents"].cpu().numpy()
    kv, scale, k, page = x["kv"], x["scale"], case["beams"], case["page"]
    table, after = before.copy(), lengths.copy()
    children = [[] for _ in lengths]
    for i in range(len(lengths)):
        children[i // k * k + parents[i // k, i % k]].append(i)
    spare = [before[p, lengths[p] // page] for p in range(len(lengths)) if not children[p] and lengths[p] % page]
    spare += list(np.flatnonzero(refs == 0))
    for i in range(len(lengths)):
        p = i // k * k + parents[i // k, i % k]
        full, rest = divmod(int(lengths[p]), page)
        table[i], after[i] = before[p], lengths[p]
        if rest and i != (p if p in children[p] else children[p][0]):
            to, origin = int(spare.pop(0)), int(before[p, full])
            table[i, full] = to
            kv[:, to, :, :, :rest] = kv[:, origin, :, :, :rest]
            scale[:, to] = scale[:, origin]
    np.subtract.at(refs, before[before >= 0], 1)
    np.add.at(refs, table[table >= 0], 1)
    return tuple(torch.from_numpy(a).cuda() for a in (table, refs, after)) + (kv, scale.double())


def _exact_attend(case, x):
    group, page, new = case["hq"] // case["hk"], case["page"], case["new"]
    table = x["table"].cpu().numpy().astype(np.int64)
    result = []
    for layer in range(case["layers"]):
        out = torch.empty(x["q"].shape[1:], dtype=torch.float64, device="cuda")
        for b, length in enumerate(_lengths(case)):
            ids = torch.from_numpy(table[b, :-(-length // page)]).cuda()
            at = torch.arange(length - new, length, device="cuda")[:, None, None]
            key = torch.arange(length, device="cuda")[None, None, :]
            hidden = key > at
            if case["window"]:
                hidden = hidden | ((at - key >= case["window"]) & (key >= case["sinks"]))
            for h in range(case["hk"]):
                both = []
                for side in range(2):
                    t = x["kv"][layer, ids, side, h].double() * x["scale"][layer, ids, side, h].double()[:, None, None]
                    both.append(t.reshape(-1, case["dim"])[:length])
                q = x["q"][layer, b * new:(b + 1) * new, h * group:(h + 1) * group].double()
                score = torch.einsum("ngd,kd->ngk", q, both[0]) / math.sqrt(case["dim"])
                p = torch.softmax(score.masked_fill(hidden, -math.inf), -1)
                out[b * new:(b + 1) * new, h * group:(h + 1) * group] = torch.einsum("ngk,kd->ngd", p, both[1])
        result.append(out)
    return result


def exact(case, seed):
    x = _inputs(case, seed)
    return {"select": _exact_select, "reorder": _exact_reorder, "attend": _exact_attend}[case["op"]](case, x)
