"""Measured cases of the attention-side operators of a learned video codec.

A context model of a codec attends from the latent tokens of the packet that is
being coded (one token per latent position, 16 x 16 pixels) to the tokens of
earlier packets.  Its operators here:

* ``rotary``  -- rotary positions over the axes (time, height, width), for
  queries and keys, in both directions (the inverse is the gradient);
* ``append``  -- new keys and values into a paged cache of 8-bit integers with
  one scale for each page, head and side (key or value), and the values the
  touched pages then stand for;
* ``attend``  -- attention of new tokens over that cache, with an optional
  sliding window and first tokens that stay visible;
* ``fork`` / ``compact`` -- cache pages shared by branching streams (an encoder
  that tries several codings from one decoded state) and moved together.

``run`` computes them in elementary 32-bit torch operations, or with the
framework's own calls when ``own`` is set.  ``exact`` is written apart from it,
in 64 bits, from the definitions.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}

# latent positions per frame: 626x352 (padded to 640x352) and 1920x1088
GRID_352 = (22, 40)
GRID_1088 = (68, 120)


def _package():
    import __graft_entry__
    return __graft_entry__.load_package()


# ------------------------------------------------------------------ cases ----

def listed():
    return [
        # one decoding step of eight streams: eight new latent tokens (latency)
        {"name": "rotary_step_8_streams", "op": "rotary", "tokens": 8, "hq": 8, "hk": 2, "dim": 64, "pt": 8, "ph": 12,
         "pw": 12, "grid_h": 22, "grid_w": 40, "layout": "half", "dtype": "bf16", "inverse": False},
        # an 8-frame packet at 626x352 in float32, pairs next to each other, a rotated part of the head only
        {"name": "rotary_packet_626x352", "op": "rotary", "tokens": 8 * 880, "hq": 6, "hk": 3, "dim": 64, "pt": 4,
         "ph": 8, "pw": 7, "grid_h": 22, "grid_w": 40, "layout": "interleaved", "dtype": "f32", "inverse": False},
        # gradient direction, one 1920x1088 frame of sixteen streams
        {"name": "rotary_gradient_1080p", "op": "rotary", "tokens": 16 * 8160, "hq": 16, "hk": 4, "dim": 128,
         "pt": 16, "ph": 24, "pw": 24, "grid_h": 68, "grid_w": 120, "layout": "half", "dtype": "bf16",
         "inverse": True},
        # one token for each of 64 streams, into pages that already hold some
        {"name": "append_step_64_streams", "op": "append", "streams": 64, "new": 1, "past": 880, "ragged": True,
         "hk": 8, "dim": 128, "page": 64, "dtype": "bf16"},
        # one 1920x1088 frame of four streams
        {"name": "append_frame_1080p", "op": "append", "streams": 4, "new": 8160, "past": 0, "ragged": False, "hk": 8,
         "dim": 128, "page": 64, "dtype": "f16"},
        # the smallest step: one token of one stream over two 626x352 frames
        {"name": "attend_token_1_stream", "op": "attend", "streams": 1, "new": 1, "past": 2 * 880, "ragged": False,
         "hq": 8, "hk": 2, "dim": 64, "page": 16, "window": 0, "sinks": 0, "causal": True, "dtype": "f16"},
        # one token for each of 64 streams of very different lengths, up to two 1920x1088 frames
        {"name": "attend_tokens_64_streams", "op": "attend", "streams": 64, "new": 1, "past": 2 * 8160,
         "ragged": True, "hq": 16, "hk": 4, "dim": 128, "page": 64, "window": 0, "sinks": 0, "causal": True,
         "dtype": "bf16"},
        # a window of one 1920x1088 frame and 16 sinks over eight frames, five queries to a key head
        {"name": "attend_tokens_window_sinks", "op": "attend", "streams": 32, "new": 1, "past": 8 * 8160,
         "ragged": False, "hq": 10, "hk": 2, "dim": 128, "page": 32, "window": 8160, "sinks": 16, "causal": True,
         "dtype": "bf16"},
        # a whole 1920x1088 frame sees itself and two earlier frames, in both directions
        {"name": "attend_frame_1080p", "op": "attend", "streams": 1, "new": 8160, "past": 2 * 8160, "ragged": False,
         "hq": 16, "hk": 4, "dim": 128, "page": 64, "window": 0, "sinks": 0, "causal": False, "dtype": "bf16"},
        # causal pieces of odd lengths from eight streams, window and sinks
        {"name": "attend_pieces_8_streams", "op": "attend", "streams": 8, "new": 2039, "past": 3 * 880 + 5,
         "ragged": True, "hq": 6, "hk": 2, "dim": 64, "page": 32, "window": 1761, "sinks": 7, "causal": True,
         "dtype": "f16"},
        # 64 trial codings branch off 16 decoded states, eight attention layers
        {"name": "fork_64_trials", "op": "fork", "streams": 16, "forks": 64, "past": 439, "layers": 8, "hk": 4,
         "dim": 128, "page": 64},
        # a pool of 1024 pages, half of them live and scattered, four attention layers
        {"name": "compact_1024_pages", "op": "compact", "streams": 48, "past": 1471, "pages": 1024, "layers": 4,
         "hk": 4, "dim": 128, "page": 64},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["rotary", "append", "attend", "attend", "attend", "fork", "compact"])
    dim = rng.choice([64, 128])
    grid = rng.choice([GRID_352, GRID_1088])
    if op == "rotary":
        hk = rng.choice([1, 2, 3, 4])
        hq = hk * rng.choice([1, 2, 3, 4])
        half = rng.randint(dim // 4, dim // 2)
        pt = rng.randint(1, half // 3)
        ph = (half - pt) // 2
        return {"op": op, "tokens": _log(rng, 1, 130560), "hq": hq, "hk": hk, "dim": dim, "pt": pt, "ph": ph,
                "pw": half - pt - ph, "grid_h": grid[0], "grid_w": grid[1],
                "layout": rng.choice(["half", "interleaved"]), "dtype": rng.choice(["f32", "f16", "bf16"]),
                "inverse": rng.random() < 0.5}
    if op == "append":
        streams = _log(rng, 1, 64)
        return {"op": op, "streams": streams, "new": _log(rng, 1, 32640 // streams), "past": rng.randint(0, 880),
                "ragged": rng.random() < 0.5, "hk": rng.choice([1, 2, 3, 8]), "dim": dim,
                "page": rng.choice([16, 32, 64, 128]), "dtype": rng.choice(["f32", "f16", "bf16"])}
    if op == "attend":
        hk = rng.choice([1, 2, 4, 8])
        group = rng.choice([1, 2, 3, 4, 5, 6, 8])
        streams = _log(rng, 1, 64)
        kind = rng.choice(["token", "few", "piece"])
        new = {"token": 1, "few": rng.randint(2, 16), "piece": _log(rng, 17, 2040)}[kind]
        # bounded by the cache of the largest listed step and the products of the largest listed frame
        past = _log(rng, 1, max(2, min(65280, 1000000000 // (streams * hk * dim * 2))))
        while streams * new * (past + new) * hk * group * dim > 3.2e11:
            new = max(1, new // 2)
            past = max(1, past // 2)
        window = _log(rng, 1, 8160) if rng.random() < 0.5 else 0
        return {"op": op, "streams": streams, "new": new, "past": past, "ragged": rng.random() < 0.6, "hq": hk * group,
                "hk": hk, "dim": dim, "page": rng.choice([16, 32, 64, 128]), "window": window,
                "sinks": rng.randint(0, 64) if window else 0, "causal": rng.random() < 0.7,
                "dtype": rng.choice(["f16", "bf16"])}
    if op == "fork":
        return {"op": op, "streams": rng.randint(1, 16), "forks": _log(rng, 1, 64), "past": _log(rng, 1, 500),
                "layers": rng.randint(1, 8), "hk": rng.choice([1, 2, 4]), "dim": dim,
                "page": rng.choice([16, 32, 64, 128])}
    pages = _log(rng, 16, 1024)
    page = rng.choice([16, 32, 64, 128])
    streams = rng.randint(2, 48)
    return {"op": op, "streams": streams, "past": max(1, pages * page // (2 * streams)), "pages": pages,
            "layers": rng.randint(1, 4), "hk": rng.choice([1, 2, 4]), "dim": dim, "page": page}


# ----------------------------------------------------------------- lengths ----

def _share(b):
    """Fixed spread of stream lengths over (0, 1]."""
    return ((b * 37 + 11) % 64 + 1) / 64


def _past(case):
    if not case.get("ragged", True):
        return [case["past"]] * case["streams"]
    return [int(case["past"] * _share(b)) for b in range(case["streams"])]


def _new(case):
    if not case["ragged"] or case["new"] == 1:
        return [case["new"]] * case["streams"]
    return [max(1, int(case["new"] * _share(b + 5))) for b in range(case["streams"])]


def _visible(case, past, new):
    """Keys that the tokens of one stream see together, and (row, key) pairs."""
    length = past + new
    window, sinks = case["window"], case["sinks"]
    pairs = 0
    for i in range(new):
        a = past + i
        top = a if case["causal"] else length - 1
        low = max(0, a - window + 1) if window else 0
        pairs += top - low + 1 + min(sinks, low)
    low = max(0, past - window + 1) if window else 0
    return length - low + min(sinks, low), pairs


def _compact_lengths(case):
    past = [max(1, int(case["past"] * _share(b))) for b in range(case["streams"])]
    need = sum(-(-n // case["page"]) for n in past)
    while need > case["pages"]:
        past = [max(1, n // 2) for n in past]
        new_need = sum(-(-n // case["page"]) for n in past)
        if new_need == need:
            past = past[: case["pages"]]
            break
        need = new_need
    return past


def _compact_layout(case, seed):
    """Page ids of each stream: a scattered choice of the pool."""
    order = np.random.default_rng(seed + 17).permutation(case["pages"])
    rows, at = [], 0
    for n in _compact_lengths(case):
        k = -(-n // case["page"])
        rows.append(order[at:at + k])
        at += k
    return rows


def work(case):
    op = case["op"]
    if op == "rotary":
        heads = case["hq"] + case["hk"]
        n = case["tokens"] * heads * case["dim"]
        pairs = case["pt"] + case["ph"] + case["pw"]
        return {"bytes": 2 * n * SIZES[case["dtype"]] + case["tokens"] * 12, "flops": case["tokens"] * heads * pairs * 6}
    if op == "append":
        row = 2 * case["hk"] * case["dim"]
        tokens = sum(_new(case))
        touched = sum(len(r) for r in _touched(case))
        values = touched * case["page"] * row
        return {"bytes": tokens * row * (SIZES[case["dtype"]] + 1) + values * 4, "flops": tokens * row * 3 + values}
    if op == "attend":
        keys = pairs = 0
        for past, new in zip(_past(case), _new(case)):
            k, p = _visible(case, past, new)
            keys, pairs = keys + k, pairs + p
        tokens = sum(_new(case))
        return {"bytes": keys * 2 * case["hk"] * case["dim"] + 2 * tokens * case["hq"] * case["dim"] * 2,
                "flops": pairs * case["hq"] * case["dim"] * 4}
    token = 2 * case["hk"] * case["dim"] * case["layers"]
    if op == "fork":
        past = [max(1, int(case["past"] * _share(b))) for b in range(case["streams"])]
        tokens = sum(past[f % case["streams"]] % case["page"] for f in range(case["forks"]))
        entries = sum(-(-past[f % case["streams"]] // case["page"]) for f in range(case["forks"]))
        return {"bytes": 2 * tokens * token + 16 * entries, "flops": tokens * token}
    rows = [-(-n // case["page"]) for n in _compact_lengths(case)]
    live = sum(rows)
    # a random choice of the pool leaves this many live pages above the live count
    moved = live * (case["pages"] - live) / case["pages"]
    return {"bytes": int(2 * moved * case["page"] * token + 12 * case["pages"]) + 1, "flops": int(moved * case["page"] * token)}


# ------------------------------------------------------------------ inputs ----

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ints(shape, gen):
    """Stored integers as quantised normal activations have them."""
    out = torch.empty(shape, dtype=torch.int8, device="cuda")
    flat = out.view(-1)
    step = 1 << 27
    for i in range(0, flat.numel(), step):
        part = flat[i:i + step]
        part.copy_(torch.randn(part.numel(), device="cuda", generator=gen).mul_(36.0).round_().clamp_(-127, 127))
    return out


def _scales(shape, gen):
    return torch.exp(torch.randn(shape, device="cuda", generator=gen) * 0.3) * (3.5 / 127.0)


def _touched(case):
    """(page entry, first slot, end slot, first token) of every page each stream's new tokens reach."""
    rows, token = [], 0
    for past, new in zip(_past(case), _new(case)):
        items = []
        for entry in range(past // case["page"], -(-(past + new) // case["page"])):
            lo = max(past, entry * case["page"])
            hi = min(past + new, (entry + 1) * case["page"])
            items.append((entry, lo - entry * case["page"], hi - entry * case["page"], token + lo - past))
        rows.append(items)
        token += new
    return rows


def _rotary_inputs(case, seed):
    gen = _gen(seed)
    dtype = DTYPES[case["dtype"]]
    heads = case["hq"] + 2 * case["hk"]
    qkv = torch.randn((case["tokens"], heads, case["dim"]), device="cuda", generator=gen).to(dtype)
    i = torch.arange(case["tokens"], device="cuda") + int(torch.randint(0, 1000, (1,), generator=gen, device="cuda"))
    per = case["grid_h"] * case["grid_w"]
    pos = torch.stack([i // per, i % per // case["grid_w"], i % case["grid_w"]], 1).to(torch.int32)
    return {"q": qkv[:, :case["hq"]], "k": qkv[:, case["hq"]:case["hq"] + case["hk"]], "positions": pos,
            "extents": (512, case["grid_h"], case["grid_w"]), "pairs": (case["pt"], case["ph"], case["pw"]),
            "bases": (10000.0, 100.0, 100.0)}


def _cache_inputs(case, seed, lengths):
    """A pool whose streams own scattered pages."""
    gen = _gen(seed)
    page = case["page"]
    counts = [-(-n // page) for n in lengths]
    pages = sum(counts) + 3
    order = np.random.default_rng(seed).permutation(pages)
    table = np.full((len(lengths), max(counts) + 1), -1, np.int32)
    refs = np.zeros(pages, np.int32)
    at = 0
    for b, k in enumerate(counts):
        table[b, :k] = order[at:at + k]
        refs[order[at:at + k]] = 1
        at += k
    layers = case.get("layers", 1)
    return {"kv": _ints((layers, pages, 2, case["hk"], page, case["dim"]), gen),
            "scale": _scales((layers, pages, 2, case["hk"]), gen), "table": torch.from_numpy(table).cuda(),
            "refs": torch.from_numpy(refs).cuda(), "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda"),
            "gen": gen, "host_table": table}


def _inputs(case, seed):
    op = case["op"]
    if op == "rotary":
        return _rotary_inputs(case, seed)
    if op in ("append", "attend"):
        past, new = _past(case), _new(case)
        x = _cache_inputs(case, seed, [p + n for p, n in zip(past, new)])
        gen, tokens = x["gen"], sum(new)
        if op == "append":
            dtype = DTYPES[case["dtype"]]
            # heads of different ranges, as projections have them
            kv = torch.randn((tokens, 2 * case["hk"], case["dim"]), device="cuda", generator=gen)
            kv *= torch.exp(torch.randn((1, 2 * case["hk"], 1), device="cuda", generator=gen) * 0.5)
            x["k"], x["v"] = kv.to(dtype).split(case["hk"], 1)
            rows = _touched(case)
            items = [(x["host_table"][b, e], lo, hi, t) for b, r in enumerate(rows) for e, lo, hi, t in r]
            x["items"] = torch.tensor(np.array(items, np.int32).reshape(-1, 4), device="cuda")
        else:
            q = torch.randn((tokens, case["hq"] + 2 * case["hk"], case["dim"]), device="cuda", generator=gen)
            x["q"] = (q * 1.5).to(DTYPES[case["dtype"]])[:, :case["hq"]]
        return x
    if op == "fork":
        past = [max(1, int(case["past"] * _share(b))) for b in range(case["streams"])]
        x = _cache_inputs(case, seed, past)
        # empty slots for the trials, free pages for their last ones
        table = torch.full((case["streams"] + case["forks"], x["table"].shape[1]), -1, dtype=torch.int32, device="cuda")
        table[:case["streams"]] = x["table"]
        pages = x["refs"].numel() + case["forks"]
        keep = np.random.default_rng(seed + 1).permutation(pages)[:x["refs"].numel()]
        keep = torch.from_numpy(keep).cuda()
        refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
        refs[keep] = x["refs"]
        table = torch.where(table >= 0, keep[table.clamp(min=0).long()].to(torch.int32), table)
        x.update(table=table, refs=refs,
                 lengths=torch.tensor(past + [0] * case["forks"], dtype=torch.int32, device="cuda"),
                 kv=_ints((case["layers"], pages, 2, case["hk"], case["page"], case["dim"]), x["gen"]),
                 scale=_scales((case["layers"], pages, 2, case["hk"]), x["gen"]),
                 src=[f % case["streams"] for f in range(case["forks"])],
                 dst=[case["streams"] + f for f in range(case["forks"])])
        return x
    gen = _gen(seed)
    rows = _compact_layout(case, seed)
    width = max(len(r) for r in rows)
    table = np.full((len(rows) + 1, width), -1, np.int32)
    refs = np.zeros(case["pages"], np.int32)
    for b, r in enumerate(rows):
        table[b, :len(r)] = r
        refs[r] += 1
    # the last slot branched off the first: their pages are shared
    table[-1] = table[0]
    refs[rows[0]] += 1
    lengths = _compact_lengths(case)
    return {"kv": _ints((case["layers"], case["pages"], 2, case["hk"], case["page"], case["dim"]), gen),
            "scale": _scales((case["layers"], case["pages"], 2, case["hk"]), gen),
            "table": torch.from_numpy(table).cuda(), "refs": torch.from_numpy(refs).cuda(),
            "lengths": torch.tensor(lengths + lengths[:1], dtype=torch.int32, device="cuda")}


def prepare(case, seed):
    x = _inputs(case, seed)
    state = {"case": case, **x}
    state.pop("gen", None)
    op = case["op"]
    if op == "rotary":
        if own:
            state["rotary"] = _package().Rotary(x["pairs"], x["extents"], bases=x["bases"], layout=case["layout"],
                                                device="cuda")
        else:
            tables = []
            for pairs, extent, base in zip(x["pairs"], x["extents"], x["bases"]):
                i = torch.arange(pairs, dtype=torch.float64, device="cuda")
                angle = torch.arange(extent, dtype=torch.float64, device="cuda")[:, None] * base ** (-i / pairs)
                tables.append((angle.cos().float(), angle.sin().float()))
            state["tables"] = tables
        return state
    if op in ("append", "attend"):
        past, new = _past(case), _new(case)
        state["starts"] = past
        state["counts"] = new
    if op == "compact":
        state["saved"] = (x["table"].clone(), x["refs"].clone())
    if own:
        ufb = _package()
        layers, pages = x["kv"].shape[:2]
        cache = ufb.KVCache(layers=layers, pages=pages, heads=case["hk"], head_dim=case["dim"],
                            page_tokens=case["page"], slots=x["table"].shape[0], table_width=x["table"].shape[1],
                            device="cuda")
        for name in ("kv", "scale", "table", "refs", "lengths"):
            getattr(cache, name).copy_(x[name])
            del state[name]
        state["cache"] = cache
        if op in ("append", "attend"):
            state["plan"] = cache.plan(list(range(case["streams"])), new)
        if op == "append":
            state["pages"] = x["items"][:, 0].contiguous()
        if op == "fork":
            state["plan"] = cache.fork_plan(x["src"], x["dst"])
    elif op == "fork":
        state["src_ids"] = torch.tensor(x["src"], device="cuda")
        state["dst_ids"] = torch.tensor(x["dst"], device="cuda")
    return state


# ------------------------------------------------------------- plain forms ----

def _plain_rotary(state):
    case, pos = state["case"], state["positions"].long()
    cos = torch.cat([c[pos[:, a]] for a, (c, s) in enumerate(state["tables"])], 1)[:, None]
    sin = torch.cat([s[pos[:, a]] for a, (c, s) in enumerate(state["tables"])], 1)[:, None]
    if case["inverse"]:
        sin = -sin
    n = cos.shape[-1]
    out = []
    for x in (state["q"], state["k"]):
        y = x.float()
        if case["layout"] == "half":
            a, b = y[..., :n], y[..., n:2 * n]
            r = torch.cat([a * cos - b * sin, a * sin + b * cos, y[..., 2 * n:]], -1)
        else:
            a, b = y[..., 0:2 * n:2], y[..., 1:2 * n:2]
            r = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
            r = torch.cat([r, y[..., 2 * n:]], -1)
        out.append(r.to(x.dtype))
    return out


def _plain_append(state):
    items = state["items"].long()
    page, lo, hi, token = items.unbind(1)
    kv, scale = state["kv"][0], state["scale"][0]
    slot = torch.arange(kv.shape[3], device=kv.device)
    fresh = (slot >= lo[:, None]) & (slot < hi[:, None])
    old = slot < lo[:, None]
    index = (token[:, None] + slot - lo[:, None]).clamp(0, state["k"].shape[0] - 1)
    for side, x in enumerate((state["k"], state["v"])):
        new = x.float()[index].permute(0, 2, 1, 3)
        top = new.abs().amax(-1).masked_fill(~fresh[:, None], 0).amax(-1)
        before = torch.where(lo[:, None] > 0, scale[page, side], torch.zeros_like(top))
        after = torch.maximum(before, top / 127.0)
        safe = torch.where(after > 0, after, torch.ones_like(after))
        kept = torch.round(kv[page, side].float() * (before / safe)[..., None, None])
        put = torch.round(new / safe[..., None, None]).clamp(-127, 127)
        stale = kv[page, side].float()
        value = torch.where(fresh[:, None, :, None], put, torch.where(old[:, None, :, None], kept, stale))
        kv[page, side] = value.to(torch.int8)
        scale[page, side] = after
    return kv[page].float() * scale[page][..., None, None]


def _plain_attend(state):
    case = state["case"]
    group = case["hq"] // case["hk"]
    out = torch.empty_like(state["q"], memory_format=torch.contiguous_format)
    token = 0
    for b, (past, new) in enumerate(zip(state["starts"], state["counts"])):
        length = past + new
        pages = state["table"][b, :-(-length // case["page"])].long()
        kv = state["kv"][0][pages].float() * state["scale"][0][pages][..., None, None]
        kv = kv.permute(1, 2, 0, 3, 4).flatten(2, 3)[:, :, :length]
        key = torch.arange(length, device=kv.device)
        at = past + torch.arange(new, device=kv.device)[:, None]
        seen = key <= at if case["causal"] else torch.ones((new, length), dtype=torch.bool, device=kv.device)
        if case["window"]:
            seen = seen & ((key > at - case["window"]) | (key < case["sinks"]))
        q = state["q"][token:token + new].float()
        for h in range(case["hk"]):
            rows = q[:, h * group:(h + 1) * group].permute(1, 0, 2)
            s = torch.matmul(rows, kv[0, h].T) * case["dim"] ** -0.5
            s.masked_fill_(~seen, float("-inf"))
            s -= s.amax(-1, keepdim=True)
            s.exp_()
            o = torch.matmul(s, kv[1, h]) / s.sum(-1, keepdim=True)
            out[token:token + new, h * group:(h + 1) * group] = o.permute(1, 0, 2).to(out.dtype)
        token += new
    return out


def _plain_fork(state):
    kv, scale, table, refs, lengths = (state[n] for n in ("kv", "scale", "table", "refs", "lengths"))
    src, dst, page = state["src_ids"], state["dst_ids"], state["case"]["page"]
    held = table[dst]
    held = held[held >= 0].long()
    refs.index_add_(0, held, torch.full_like(held, -1, dtype=torch.int32))
    rows, n = table[src], lengths[src]
    full, rest = n // page, n % page
    entry = torch.arange(rows.shape[1], device=rows.device)
    shared = rows[(entry < full[:, None]) & (rows >= 0)].long()
    refs.index_add_(0, shared, torch.ones_like(shared, dtype=torch.int32))
    split = torch.nonzero(rest > 0)[:, 0]
    fresh = torch.nonzero(refs == 0)[:split.numel(), 0]
    last = full[split].long()
    origin = rows[split, last].long()
    rows[split, last] = fresh.to(torch.int32)
    refs[fresh] = 1
    keep = (torch.arange(page, device=rows.device) < rest[split][:, None])[None, :, None, None, :, None]
    kv[:, fresh] = torch.where(keep, kv[:, origin], kv[:, fresh])
    scale[:, fresh] = scale[:, origin]
    table[dst] = rows
    lengths[dst] = n
    return table, refs, lengths, kv, scale


def _plain_compact(state):
    kv, scale, table, refs = (state[n] for n in ("kv", "scale", "table", "refs"))
    live = refs > 0
    count = int(live.sum())
    ids = torch.arange(refs.numel(), device=refs.device)
    movers = ids[live & (ids >= count)]
    holes = ids[~live & (ids < count)]
    place = ids.clone()
    place[movers] = holes
    kv[:, holes] = kv[:, movers]
    scale[:, holes] = scale[:, movers]
    refs[holes] = refs[movers]
    refs[movers] = 0
    table.copy_(torch.where(table >= 0, place[table.clamp(min=0).long()].to(torch.int32), table))
    return table, refs, kv, scale


def run(state):
    case = state["case"]
    op = case["op"]
    if op == "rotary":
        if own:
            return state["rotary"].apply(state["positions"], state["q"], state["k"], inverse=case["inverse"])
        return _plain_rotary(state)
    if op == "append":
        if own:
            cache = state["cache"]
            cache.append(0, state["plan"], state["k"], state["v"])
            return cache.read(0, state["pages"])
        return _plain_append(state)
    if op == "attend":
        if own:
            return state["cache"].attend(0, state["plan"], state["q"], window=case["window"], sinks=case["sinks"],
                                         causal=case["causal"])
        return _plain_attend(state)
    if op == "fork":
        if own:
            c = state["cache"]
            c.fork(state["plan"])
            return c.table, c.refs, c.lengths, c.kv, c.scale
        return _plain_fork(state)
    # the program goes back to the tables it saved before this trial
    table, refs = state["saved"]
    if own:
        c = state["cache"]
        c.table.copy_(table)
        c.refs.copy_(refs)
        c.compact()
        return c.table, c.refs, c.kv, c.scale
    state["table"].copy_(table)
    state["refs"].copy_(refs)
    return _plain_compact(state)


# ------------------------------------------------------------------- exact ----

def _exact_rotary(case, x):
    pos = x["positions"].double()
    angles = []
    for a in range(3):
        for i in range(x["pairs"][a]):
            angles.append(pos[:, a] * x["bases"][a] ** (-i / x["pairs"][a]))
    turn = torch.stack(angles, 1)
    if case["inverse"]:
        turn = -turn
    turn = torch.polar(torch.ones_like(turn), turn)[:, None]
    n = turn.shape[-1]
    result = []
    for t in (x["q"], x["k"]):
        y = t.double().clone()
        if case["layout"] == "half":
            z = torch.complex(y[..., :n], y[..., n:2 * n]) * turn
            y[..., :n], y[..., n:2 * n] = z.real, z.imag
        else:
            z = torch.view_as_complex(y[..., :2 * n].reshape(*y.shape[:2], n, 2).contiguous()) * turn
            y[..., :2 * n] = torch.view_as_real(z).flatten(-2)
        result.append(y)
    return result


def _exact_append(case, x):
    kv, scale = x["kv"][0].double(), x["scale"][0].double()
    done = []
    for page, lo, hi, token in x["items"].tolist():
        sides = []
        for side, t in enumerate((x["k"], x["v"])):
            new = t[token:token + hi - lo].double().transpose(0, 1)
            old = kv[page, side]
            s = new.abs().flatten(1).max(1).values / 127
            if lo:
                s = torch.maximum(s, scale[page, side])
            unit = torch.where(s > 0, s, 1.0)[:, None, None]
            q = old.clone()
            if lo:
                q[:, :lo] = torch.round(old[:, :lo] * (scale[page, side][:, None, None] / unit))
            q[:, lo:hi] = torch.round(new / unit)
            sides.append(q * s[:, None, None])
        done.append(torch.stack(sides))
    return torch.stack(done)


def _exact_attend(case, x):
    group, page = case["hq"] // case["hk"], case["page"]
    out = torch.empty(x["q"].shape, dtype=torch.float64, device="cuda")
    token = 0
    for b, (past, new) in enumerate(zip(_past(case), _new(case))):
        length = past + new
        ids = torch.from_numpy(x["host_table"][b, :-(-length // page)].astype(np.int64)).cuda()
        for h in range(case["hk"]):
            both = []
            for side in range(2):
                t = x["kv"][0, ids, side, h].double() * x["scale"][0, ids, side, h].double()[:, None, None]
                both.append(t.reshape(-1, case["dim"])[:length])
            for first in range(0, new, 1024):
                end = min(new, first + 1024)
                q = x["q"][token + first:token + end, h * group:(h + 1) * group].double()
                score = torch.einsum("ngd,kd->ngk", q, both[0]) / math.sqrt(case["dim"])
                at = torch.arange(past + first, past + end, device="cuda")[:, None, None]
                key = torch.arange(length, device="cuda")[None, None, :]
                hidden = key > at if case["causal"] else torch.zeros_like(key > at)
                if case["window"]:
                    hidden = hidden | ((at - key >= case["window"]) & (key >= case["sinks"]))
                p = torch.softmax(score.masked_fill(hidden, -math.inf), -1)
                out[token + first:token + end, h * group:(h + 1) * group] = torch.einsum("ngk,kd->ngd", p, both[1])
        token += new
    return out


def _exact_fork(case, x):
    table, refs, lengths = x["table"].cpu().numpy(), x["refs"].cpu().numpy(), x["lengths"].cpu().numpy()
    kv, scale = x["kv"], x["scale"]
    rows = []
    for s, d in zip(x["src"], x["dst"]):
        full, rest = divmod(int(lengths[s]), case["page"])
        for e in range(full):
            table[d, e] = table[s, e]
            refs[table[s, e]] += 1
        lengths[d] = lengths[s]
        rows.append((s, d, full, rest))
    for s, d, full, rest in rows:
        if rest:
            page = int(np.flatnonzero(refs == 0)[0])
            refs[page] = 1
            table[d, full] = page
            kv[:, page, :, :, :rest] = kv[:, int(table[s, full]), :, :, :rest]
            scale[:, page] = scale[:, int(table[s, full])]
    return tuple(torch.from_numpy(a).cuda() for a in (table, refs, lengths)) + (kv, scale.double())


def _exact_compact(case, x):
    table, refs = x["table"].cpu().numpy(), x["refs"].cpu().numpy()
    kv, scale = x["kv"], x["scale"]
    count, hole = int((refs > 0).sum()), 0
    for page in range(count, refs.size):
        if refs[page] > 0:
            while refs[hole] > 0:
                hole += 1
            kv[:, hole], scale[:, hole] = kv[:, page].clone(), scale[:, page].clone()
            table[table == page] = hole
            refs[hole], refs[page] = refs[page], 0
    return torch.from_numpy(table).cuda(), torch.from_numpy(refs).cuda(), kv, scale.double()


def exact(case, seed):
    x = _inputs(case, seed)
    return {"rotary": _exact_rotary, "append": _exact_append, "attend": _exact_attend, "fork": _exact_fork,
            "compact": _exact_compact}[case["op"]](case, x)
