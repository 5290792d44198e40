"""GPU: streams that branch off one another -- reorder, share, attention over groups --
against plain implementations, and a search that runs them all.

Attention is held to the tolerances of the plain attention (test_gpu_attention.py).
The join of a row's parts adds to a weight what its logarithms (base 2, at most a few
units beyond the scores, whose own rounding is counted there) and two exponentials lose:
below 2^-19 of it.
"""
import math

import numpy as np
import pytest
import torch
from test_gpu_attention import F16_TINY, ULP, Pages, _clean, _same, attend_ref, contents, gen, make_cache, randn
from test_gpu_beams import select_ref

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- reorder ----

class Branches(Pages):
    """The page operators in plain Python, with reorder."""

    def reorder(self, slots, width, parents):
        src = [slots[i // width * width + p] for i, p in enumerate(parents)]
        rest = {s: self.lengths[s] % self.P for s in slots}
        last = {s: self.table[s][self.lengths[s] // self.P] if rest[s] else -1 for s in slots}
        keeper = {}
        for s, d in zip(src, slots):
            if s == d or s not in keeper:
                keeper[s] = d
        spare = [last[s] for s in slots if s not in src and last[s] >= 0]
        copies = [(s, d) for s, d in zip(src, slots) if last[s] >= 0 and keeper[s] != d]
        spare += self.free()
        if len(copies) > len(spare):
            return None
        rows = {d: list(self.table[s]) for s, d in zip(src, slots)}
        lengths = {d: self.lengths[s] for s, d in zip(src, slots)}
        moves = []
        for (s, d), page in zip(copies, spare):
            rows[d][self.lengths[s] // self.P] = page
            moves.append((last[s], page, rest[s]))
        for s in slots:
            for p in self.table[s]:
                if p >= 0:
                    self.refs[p] -= 1
        for s in slots:
            self.table[s], self.lengths[s] = rows[s], lengths[s]
            for p in rows[s]:
                if p >= 0:
                    self.refs[p] += 1
        return moves


@pytest.mark.parametrize("page,pages,slots,width,seed",
                         [(16, 44, 6, 3, 0), (32, 300, 12, 4, 1), (64, 3000, 130, 64, 2), (128, 14, 4, 2, 3), (16, 900, 40, 1, 4),
                          (16, 6000, 1290, 43, 5)])
def test_reorder_random_operations(ufb, dev, page, pages, slots, width, seed):
    """Tables, counts, lengths and the bytes of every page follow a plain model, whatever the order of calls."""
    rng = np.random.default_rng(seed)
    columns = max(3, 2 * pages // slots) if slots < 1000 else 140
    cache = ufb.KVCache(2, pages, 3, 64, page, slots, columns, device=dev)
    cache.kv.copy_(torch.randint(-128, 128, cache.kv.shape, generator=gen(dev, seed), device=dev, dtype=torch.int8))
    cache.scale.copy_(torch.rand(cache.scale.shape, generator=gen(dev, seed), device=dev))
    kv, scale = cache.kv.clone(), cache.scale.clone()
    model = Branches(pages, slots, columns, page)
    failed = done = 0
    for step in range(70 if slots < 1000 else 12):
        op = rng.choice(["extend", "extend", "reorder", "reorder", "reorder", "release", "fork", "trim", "compact"])
        some = rng.permutation(slots)[:rng.integers(1, slots + 1)].tolist()
        if op == "extend":
            if slots > 1000:
                some = some[:max(1, len(some) // 3)]
            counts = rng.integers(0, (2 * page + 2) if slots < 1000 else page, len(some)).tolist()
            cache.extend(cache.plan(some, counts))
            assert ufb.device_status(0) == (0 if model.extend(some, counts) else 31)
        elif op == "release":
            some = some[:max(1, len(some) // 3)]
            cache.release(cache.plan(some, [0] * len(some)))
            model.release(some)
        elif op == "trim":
            window, sinks = int(rng.integers(1, 4 * page)), int(rng.integers(0, 2 * page))
            cache.trim(cache.plan(some, [0] * len(some)), window, sinks)
            model.trim(some, window, sinks)
        elif op == "fork":
            cut = max(1, len(some) // 3)
            dst, src = some[:cut], some[cut:]
            if not src:
                continue
            src = [src[int(rng.integers(len(src)))] for _ in dst]
            cache.fork(cache.fork_plan(src, dst))
            moves = model.fork(src, dst)
            assert ufb.device_status(0) == (0 if moves is not None else 31)
        elif op == "reorder":
            n = int(rng.integers(1, slots // width + 1))
            some = rng.permutation(slots)[:n * width].tolist()
            parents = rng.integers(0, width, (n, width)) if step % 3 else np.minimum(rng.integers(0, 2, (n, width)), width - 1)
            if step % 5 == 0:
                parents[:] = np.argsort(rng.random((n, width)), 1)   # every stream goes on somewhere
            before = cache.table.clone(), cache.lengths.clone(), cache.refs.clone()
            cache.reorder(cache.beam_plan(some, width), torch.from_numpy(parents.astype(np.int32)).to(dev))
            moves = model.reorder(some, width, parents.reshape(-1).tolist())
            assert ufb.device_status(0) == (0 if moves is not None else 31)
            if moves is None:
                failed += 1
                for a, b in zip(before, (cache.table, cache.lengths, cache.refs)):
                    assert torch.equal(a, b)
            done += moves is not None
        else:
            cache.compact()
            moves = [(a, b, page) for a, b in model.compact()]
        if op in ("fork", "reorder", "compact"):
            for a, b, n in moves or []:
                kv[:, b, :, :, :n] = kv[:, a, :, :, :n]
                scale[:, b] = scale[:, a]
        _same(cache, model)
        assert torch.equal(cache.kv, kv) and torch.equal(cache.scale, scale)
    assert done > 0
    _clean(ufb)


def test_reorder_without_pages(ufb, dev):
    """Streams of one length need no free page; of several, one that is missing changes nothing."""
    cache = make_cache(ufb, dev, [21] * 4, 1, 64, 16, spare=0)
    assert bool((cache.refs > 0).all())
    plan = cache.beam_plan([0, 1, 2, 3], 4)
    parents = lambda *p: torch.tensor([p], dtype=torch.int32, device=dev)
    old = [contents(cache, 0, s)[0] for s in range(4)]
    cache.reorder(plan, parents(2, 2, 2, 1))
    for s, p in enumerate((2, 2, 2, 1)):
        assert torch.equal(contents(cache, 0, s)[0], old[p])
    _clean(ufb)
    cache = make_cache(ufb, dev, [21, 32, 32, 5], 1, 64, 16, spare=0)
    state = [t.clone() for t in (cache.table, cache.lengths, cache.refs, cache.kv, cache.scale)]
    cache.reorder(cache.beam_plan([0, 1, 2, 3], 4), parents(0, 0, 3, 3))   # two copies, no page left behind
    assert ufb.device_status(0) == 31
    for bad in ((0, 4, 1, 1), (-1, 0, 0, 0)):
        cache.reorder(cache.beam_plan([0, 1, 2, 3], 4), parents(*bad))
        assert ufb.device_status(0) == 32
    for a, b in zip(state, (cache.table, cache.lengths, cache.refs, cache.kv, cache.scale)):
        assert torch.equal(a, b)


def test_reorder_takes_marks_along(ufb, dev):
    """A stream whose extend was refused gives its mark to those that go on from it."""
    cache = make_cache(ufb, dev, [20, 20, 20], 1, 64, 16, spare=0)
    cache.extend(cache.plan([1], [400]))
    assert ufb.device_status(0) == 31
    cache.reorder(cache.beam_plan([0, 1, 2], 3), torch.tensor([[1, 0, 1]], dtype=torch.int32, device=dev))
    _clean(ufb)
    q = randn(dev, (3, 1, 64), 1, torch.float16)
    out = cache.attend(0, cache.plan([0, 1, 2], [1, 1, 1]), q)
    assert ufb.device_status(0) == 31
    assert not bool(out[[0, 2]].any()) and bool(out[1].any())


def test_reorder_refusals(ufb, dev):
    cache = make_cache(ufb, dev, [20] * 6, 1, 64, 16)
    other = make_cache(ufb, dev, [20] * 6, 1, 64, 16)
    for slots, width in (([0, 1, 2], 2), ([0, 0], 2), ([0, 6], 2), ([-1, 0], 1), ([0, 1], 0), ([0, 1], 65)):
        with pytest.raises(ufb.UfbError):
            cache.beam_plan(slots, width)
    plan = cache.beam_plan([0, 1, 2, 3], 2)
    good = torch.zeros((2, 2), dtype=torch.int32, device=dev)
    for bad in (good.long(), good[:1], good.cpu(), good.flatten(), None):
        with pytest.raises(ufb.UfbError):
            cache.reorder(plan, bad)
    with pytest.raises(ufb.UfbError):
        other.reorder(plan, good)
    with pytest.raises(ufb.UfbError):
        cache.reorder(cache.plan([0, 1], [0, 0]), good[:1])
    cache.reorder(cache.beam_plan([], 3), good.new_zeros((0, 3)))
    cache.reorder(plan, good.t())
    _clean(ufb)


# ------------------------------------------------------- groups: share, attend ----

def make_groups(ufb, dev, groups, heads, dim, page, layers=1, seed=0, spare=2):
    """groups: for each the common tokens and its streams' own ones.  Pages of whole common
    pages are shared, all others a stream's own."""
    lengths = [c + o for c, own in groups for o in own]
    cache = make_cache(ufb, dev, lengths, heads, dim, page, seed=seed, layers=layers, spare=spare)
    s = 0
    for c, own in groups:
        full = c // page
        for i in range(1, len(own)):
            cache.refs[cache.table[s + i, :full].long()] = 0
            cache.table[s + i, :full] = cache.table[s, :full]
        cache.refs[cache.table[s, :full].long()] = len(own)
        s += len(own)
    return cache, lengths, [len(own) for _, own in groups]


def check_groups(ufb, cache, slots, counts, sizes, hq, dtype, window=0, sinks=0, causal=True, scale=None, mul=1.0, seed=5,
                 layer=0, shared=None):
    plan = cache.plan(slots, counts)
    groups = cache.group_plan(plan, sizes)
    cache.share(groups)
    if shared is not None:
        assert groups.shared.tolist() == shared
    qkv = randn(cache.device, (sum(counts), hq + 2 * cache.heads, cache.head_dim), seed, dtype, mul)
    q = qkv[:, :hq]
    kw = dict(window=window, sinks=sinks, causal=causal, scale=scale, groups=groups)
    got, lse = cache.attend(layer, plan, q, lse=True, **kw)
    want, wl, tol, tl = attend_ref(cache, layer, slots, counts, q, window, sinks, causal,
                                   cache.head_dim ** -0.5 if scale is None else scale)
    # p |v| is within tol / 2^-11
    full = tol * (1 + 2.0 ** -8) + ULP[dtype] * want.abs() + (F16_TINY if dtype == torch.float16 else 0)
    lost = torch.isnan(want).any(-1)
    assert bool(torch.isnan(got[lost]).all()) and bool(torch.isnan(lse[lost]).all())
    wl = torch.where(lost, 0, wl)
    error = torch.where(lost[..., None], 0, (got.double() - want).abs())
    full = torch.where(lost[..., None], 0, full)
    assert bool((error <= full).all()), float((error - full).max())
    empty = torch.isinf(wl)
    assert bool((lse[empty] == -math.inf).all()) and bool((got[empty] == 0).all())
    known = ~empty & ~lost
    assert bool(((lse.double() - wl).abs()[known] <= tl[known] + 2.0 ** -19).all())
    again = cache.attend(layer, plan, q, **kw)
    assert torch.equal(again[~lost], got[~lost])  # no order of work shows
    _clean(ufb)
    return got


# heads, group, dim, page; the rows of a group of few and of many streams lie on both sides of each kernel's range
SHAPES = [(1, 1, 64, 16), (2, 4, 64, 32), (2, 5, 128, 64), (3, 3, 128, 128), (1, 8, 128, 16), (1, 70, 64, 64)]
GROUPS = [
    [(100, [1])],
    [(33, [1, 5])],
    [(640, [3, 1, 1, 9])],
    [(1000, [70, 65, 129, 1, 2, 3, 40]), (64, [1, 1]), (0, [200, 3]), (15, [1, 1, 1])],
    [(2049, list(range(1, 34)))],
    [(777, [7] * 5), (1500, [300] * 3), (128, [1]), (5000, [20] * 12)],
]


@pytest.mark.parametrize("case", range(len(GROUPS)))
@pytest.mark.parametrize("heads,group,dim,page", SHAPES)
def test_groups_single_tokens(ufb, dev, heads, group, dim, page, case):
    cache, lengths, sizes = make_groups(ufb, dev, GROUPS[case], heads, dim, page, seed=case)
    shared = [0 if len(own) == 1 else min(c // page * page, min(c + o - 1 for o in own) // page * page)
              for c, own in GROUPS[case]]
    for dtype in (torch.float16, torch.bfloat16):
        check_groups(ufb, cache, list(range(len(lengths))), [1] * len(lengths), sizes, heads * group, dtype, shared=shared)


@pytest.mark.parametrize("new", [2, 5, 33, 150])
@pytest.mark.parametrize("heads,group,dim,page", SHAPES[1:4])
def test_groups_pieces(ufb, dev, heads, group, dim, page, new):
    """Several tokens a stream, ragged, also none; streams of a group in any order of slots; causal and not."""
    cache, lengths, _ = make_groups(ufb, dev, [(300, [new, new + 9, 200, new]), (1100, [new, new + 1])], heads, dim, page)
    for causal in (True, False):
        check_groups(ufb, cache, [2, 0, 3, 1, 5, 4], [1, new, 0, new, max(1, new // 2), new], [4, 2], heads * group,
                     torch.bfloat16, causal=causal)
        check_groups(ufb, cache, [4, 1, 2], [0, 0, new], [1, 2], heads * group, torch.float16, causal=causal)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 5), (16, 16), (64, 0), (300, 64), (5000, 3), (100, 2000), (700, 1300)])
def test_groups_window_sinks(ufb, dev, window, sinks):
    """Windows that begin in the common keys, at their end and behind it; sinks that reach past them."""
    for page, dim, group in ((16, 64, 3), (64, 128, 12)):
        cache, lengths, sizes = make_groups(ufb, dev, [(1200, [1, 90, 400, 3]), (320, [5, 5, 5])], 2, dim, page)
        for counts in ([1] * 7, [1, 9, 30, 2, 5, 1, 4]):
            for causal in (True, False):
                check_groups(ufb, cache, list(range(7)), counts, sizes, 2 * group, torch.float16, window=window, sinks=sinks,
                             causal=causal)


def test_groups_that_see_nothing(ufb, dev):
    """Dropped pages, common and own, empty streams, queries before the first key."""
    cache, lengths, sizes = make_groups(ufb, dev, [(512, [3, 9, 40]), (96, [1, 1])], 2, 128, 32)
    cache.table[:3, 2:9] = -1
    cache.table[3:, :] = -1
    cache.table[1, 16:] = -1
    slots = list(range(5))
    check_groups(ufb, cache, slots, [1] * 5, sizes, 4, torch.bfloat16, shared=[512, 96])
    check_groups(ufb, cache, slots, [1] * 5, sizes, 36, torch.bfloat16, window=7)
    check_groups(ufb, cache, slots, [3, 9, 2, 1, 1], sizes, 4, torch.bfloat16)
    cache = make_cache(ufb, dev, [0, 2, 1, 300], 1, 64, 16)
    check_groups(ufb, cache, [0, 1, 2, 3], [4, 4, 4, 4], [4], 2, torch.float16)


@pytest.mark.parametrize("mul,scale", [(30.0, None), (1e-6, None), (1.0, 0.0), (1.0, -0.1), (3e4, 1e-5)])
@pytest.mark.parametrize("beams", [2, 40])
def test_groups_score_ranges(ufb, dev, mul, scale, beams):
    cache, lengths, sizes = make_groups(ufb, dev, [(700, [30] * beams)], 2, 64, 16)
    for dtype in (torch.float16, torch.bfloat16):
        check_groups(ufb, cache, list(range(beams)), [1] * beams, sizes, 4, dtype, mul=mul, scale=scale)


def test_groups_values_that_are_not_finite(ufb, dev):
    """Stale and hidden values change nothing; a query that is not finite spoils its own head only."""
    cache, lengths, sizes = make_groups(ufb, dev, [(640, [9, 70])], 2, 128, 64, spare=4)
    plan = cache.plan([0, 1], [1, 1])
    groups = cache.group_plan(plan, sizes)
    cache.share(groups)
    q = randn(dev, (2, 4, 128), 3, torch.bfloat16)
    want = cache.attend(0, plan, q, window=100, sinks=3, groups=groups)
    cache.scale[0, cache.refs == 0] = math.nan
    for e in range(1, 6):
        cache.scale[0, int(cache.table[0, e])] = math.nan if e % 2 else math.inf
    last = int(cache.table[1, 11])
    cache.kv[0, last, :, :, (640 + 70) % 64:] = -128
    assert torch.equal(cache.attend(0, plan, q, window=100, sinks=3, groups=groups), want)
    q[1, 2, 5] = math.inf
    got = cache.attend(0, plan, q, window=100, sinks=3, groups=groups)
    assert bool(torch.isnan(got[1, 2]).all())
    got[1, 2] = want[1, 2]
    assert torch.equal(got, want)
    _clean(ufb)


def test_groups_with_a_refused_extend(ufb, dev):
    """A stream left out gives zeros, and the others keep what they have in common."""
    for beams, hq in ((3, 2), (40, 4)):
        cache, lengths, sizes = make_groups(ufb, dev, [(320, [5] * beams)], 2, 64, 16, spare=0)
        cache.extend(cache.plan([1], [4000]))
        assert ufb.device_status(0) == 31
        plan = cache.plan(list(range(beams)), [1] * beams)
        groups = cache.group_plan(plan, sizes)
        cache.share(groups)
        assert groups.shared.tolist() == [320]
        q = randn(dev, (beams, hq, 64), 2, torch.float16)
        got, lse = cache.attend(0, plan, q, groups=groups, lse=True)
        assert ufb.device_status(0) == 31
        assert not bool(got[1].any()) and bool((lse[1] == -math.inf).all())
        rest = [i for i in range(beams) if i != 1]
        want, _, tol, _ = attend_ref(cache, 0, rest, [1] * len(rest), q[rest], 0, 0, True, 64 ** -0.5)
        full = tol * (1 + 2.0 ** -8) + ULP[torch.float16] * want.abs() + F16_TINY
        assert bool(((got[rest].double() - want).abs() <= full).all())
    _clean(ufb)


def test_groups_long_streams_and_layers(ufb, dev):
    cache, lengths, sizes = make_groups(ufb, dev, [(70000, [1, 40, 5, 700]), (9, [3])], 1, 64, 64, layers=2)
    for counts in ([1] * 5, [1, 6, 5, 129, 2]):
        check_groups(ufb, cache, list(range(5)), counts, sizes, 8, torch.bfloat16, layer=1)


def test_groups_refusals(ufb, dev):
    cache, lengths, sizes = make_groups(ufb, dev, [(100, [5, 5]), (20, [5])], 2, 64, 16)
    plan = cache.plan([0, 1, 2], [1, 1, 1])
    for bad in ([], [2], [2, 2], [0, 3], [3, 0], [-1, 4]):
        with pytest.raises(ufb.UfbError):
            cache.group_plan(plan, bad)
    groups = cache.group_plan(plan, sizes)
    q = randn(dev, (3, 4, 64), 1, torch.float16)
    with pytest.raises(ufb.UfbError, match="share"):
        cache.attend(0, plan, q, groups=groups)   # not looked at yet
    cache.share(groups)
    cache.attend(0, plan, q, groups=groups)
    with pytest.raises(ufb.UfbError):
        cache.attend(0, cache.plan([0, 1, 2], [1, 1, 1]), q, groups=groups)
    other = make_cache(ufb, dev, [20] * 3, 2, 64, 16)
    with pytest.raises(ufb.UfbError):
        other.share(groups)
    beams = cache.beam_plan([0, 1], 2)
    for change in (lambda: cache.extend(plan), lambda: cache.trim(plan, 50),
                   lambda: cache.reorder(beams, torch.zeros((1, 2), dtype=torch.int32, device=dev)),
                   lambda: cache.release(cache.plan([2], [0])), lambda: cache.fork(cache.fork_plan([0], [2]))):
        change()
        with pytest.raises(ufb.UfbError, match="share"):
            cache.attend(0, plan, q, groups=groups)   # not since then
        cache.share(groups)
        cache.attend(0, plan, q, groups=groups)
    empty = cache.plan([], [])
    none = cache.group_plan(empty, [])
    cache.share(none)
    assert cache.attend(0, empty, q[:0], groups=none).shape == (0, 4, 64)
    _clean(ufb)


@pytest.mark.parametrize("which", ["first", "offsets"])
def test_groups_that_are_not_the_streams(ufb, dev, which):
    """Group bounds that do not belong to the batch: reported, the group's results left alone."""
    cache, lengths, sizes = make_groups(ufb, dev, [(100, [5] * 3), (200, [5] * 2)], 2, 64, 16)
    plan = cache.plan(list(range(5)), [2] * 5)
    groups = cache.group_plan(plan, sizes)
    q = randn(dev, (10, 4, 64), 1, torch.float16)
    cache.share(groups)
    want = cache.attend(0, plan, q, groups=groups)
    _clean(ufb)
    getattr(groups, which)[1] -= 1   # the border between the groups
    cache.share(groups)
    assert ufb.device_status(0) == 32
    getattr(groups, which)[1] += 1
    cache.share(groups)
    assert torch.equal(cache.attend(0, plan, q, groups=groups), want)
    _clean(ufb)


def test_groups_on_streams_and_in_graphs(ufb, dev):
    """Calls side by side do not share scratch; a captured step follows tables and lengths."""
    cache, lengths, sizes = make_groups(ufb, dev, [(3000, [9] * 4), (2000, [9] * 20)], 2, 64, 32, spare=80)
    plans = [cache.plan(list(range(4)), [1] * 4), cache.plan(list(range(4, 24)), [1] * 20)]
    groups = [cache.group_plan(p, [p.n]) for p in plans]
    for g in groups:
        cache.share(g)
    qs = [randn(dev, (p.n, 8, 64), i, torch.float16) for i, p in enumerate(plans)]
    want = [cache.attend(0, p, q, groups=g) for p, q, g in zip(plans, qs, groups)]
    side = [torch.cuda.Stream(dev) for _ in plans]
    torch.cuda.synchronize(dev)
    got = []
    for _ in range(20):
        for s, p, q, g in zip(side, plans, qs, groups):
            with torch.cuda.stream(s):
                got.append(cache.attend(0, p, q, groups=g))
    torch.cuda.synchronize(dev)
    for i, g in enumerate(got):
        assert torch.equal(g, want[i % 2])
    plan, group, q = plans[1], groups[1], qs[1]
    beams = cache.beam_plan(list(range(4, 24)), 20)
    parents = torch.arange(20, dtype=torch.int32, device=dev)[None].clone()
    k = randn(dev, (20, 2, 64), 7, torch.float16)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side[1]):
        cache.reorder(beams, parents)
        cache.extend(plan)
        cache.share(group)
        cache.append(0, plan, k, -k)
        out = cache.attend(0, plan, q, groups=group)
    for step in range(4):
        parents.copy_(torch.randint(0, 20, (1, 20), generator=gen(dev, step), device=dev))
        graph.replay()
        torch.cuda.synchronize(dev)
        assert cache.lengths[4:].tolist() == [2010 + step] * 20
        want, _, tol, _ = attend_ref(cache, 0, list(range(4, 24)), [1] * 20, q, 0, 0, True, 64 ** -0.5)
        full = tol * (1 + 2.0 ** -8) + ULP[torch.float16] * want.abs() + F16_TINY
        assert bool(((out.double() - want).abs() <= full).all())
    _clean(ufb)


@pytest.mark.parametrize("groups", [33, 70, 150])
def test_groups_of_any_number(ufb, dev, groups):
    """The work is divided by one warp, 32 (group, row tile) pairs at a time, or by a block where there are many."""
    made = [((i * 37) % 300, [1 + i % 3] * (1 + i % 4)) for i in range(groups)]
    cache, lengths, sizes = make_groups(ufb, dev, made, 2, 64, 16, seed=groups)
    for dtype in (torch.float16, torch.bfloat16):
        check_groups(ufb, cache, list(range(len(lengths))), [1] * len(lengths), sizes, 10, dtype)


@pytest.mark.parametrize("rows", [31, 32, 33, 64, 65, 96, 97, 128, 129, 161])
@pytest.mark.parametrize("dim", [64, 128])
def test_groups_row_counts(ufb, dev, rows, dim):
    """Rows around the numbers that lie in a tile four times, two times and once; short items that no
    other block shares, and long ones."""
    cache, lengths, sizes = make_groups(ufb, dev, [(70, [3] * rows), (2500, [3] * rows)], 1, dim, 32, seed=rows)
    check_groups(ufb, cache, list(range(rows)), [1] * rows, [rows], 1, torch.float16)
    check_groups(ufb, cache, list(range(2 * rows)), [1] * (2 * rows), sizes, 1, torch.bfloat16)


def test_groups_captured_behind_other_work(ufb, dev):
    """In a graph the attention follows a copy, a fill, or what another stream did."""
    cache, lengths, sizes = make_groups(ufb, dev, [(500, [9] * 6)], 2, 128, 32)
    plan = cache.plan(list(range(6)), [1] * 6)
    group = cache.group_plan(plan, [6])
    cache.share(group)
    source = [randn(dev, (6, 4, 128), i, torch.float16) for i in range(3)]
    want = [cache.attend(0, plan, q, groups=group) for q in source]
    given, q = torch.empty_like(source[0]), torch.empty_like(source[0])
    main, side = torch.cuda.Stream(dev), torch.cuda.Stream(dev)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize(dev)
    with torch.cuda.graph(graph, stream=main):
        q.copy_(given)
        after_copy = cache.attend(0, plan, q, groups=group)
        q.zero_()
        after_fill = cache.attend(0, plan, q, groups=group)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            q.copy_(given)
        main.wait_stream(side)
        after_side = cache.attend(0, plan, q, groups=group)
    zero = cache.attend(0, plan, torch.zeros_like(q), groups=group)
    for x, w in zip(source, want):
        given.copy_(x)
        graph.replay()
        torch.cuda.synchronize(dev)
        assert torch.equal(after_copy, w) and torch.equal(after_side, w) and torch.equal(after_fill, zero)
    _clean(ufb)


# --------------------------------------------------------- a search over them ----

def test_search(ufb, dev):
    """Steps of a search: the choice, the cache's streams behind it, and attention, against
    whole sequences kept on the host."""
    streams, width, vocab, heads, dim, page = 3, 6, 50, 2, 64, 16
    n = streams * width
    cache = ufb.KVCache(1, 260, heads, dim, page, n, 12, device=dev)
    table = randn(dev, (vocab, 2 * heads, dim), 1, torch.float16)     # keys and values of the tokens
    queries = randn(dev, (vocab, 4, dim), 2, torch.float16)
    project = randn(dev, (4 * dim, vocab), 3, torch.float32) * 0.5
    prompt = torch.randint(0, vocab, (streams, 40), generator=gen(dev, 4), device=dev)
    first = cache.plan([b * width for b in range(streams)], [40] * streams)
    cache.extend(first)
    kv = table[prompt.flatten()]
    cache.append(0, first, kv[:, :heads], kv[:, heads:])
    # the first streams' state goes to all their beams
    beams = cache.beam_plan(range(n), width)
    cache.reorder(beams, torch.zeros((streams, width), dtype=torch.int32, device=dev))
    plan = cache.plan(range(n), [1] * n)
    groups = cache.group_plan(plan, [width] * streams)
    words = [[prompt[b].tolist() for _ in range(width)] for b in range(streams)]
    scores = torch.full((streams, width), -math.inf, device=dev)
    scores[:, 0] = 0.0
    last = prompt[:, -1:].expand(streams, width)
    finished = torch.zeros((streams, width), dtype=torch.bool, device=dev)
    x = randn(dev, (n, 4 * dim), 5)
    for step in range(30):
        logits = (x.view(streams, width, -1) @ project)
        want = select_ref(logits, scores, width, finished, 0)
        scores, parents, tokens = ufb.beam_select(logits, scores, width, finished, 0)
        assert np.array_equal(parents.cpu().numpy(), want[1]) and np.array_equal(tokens.cpu().numpy(), want[2])
        finished = finished.gather(1, parents.long()) | (tokens == 1)
        cache.reorder(beams, parents)
        cache.extend(plan)
        cache.share(groups)
        kv = table[tokens.flatten().long()]
        cache.append(0, plan, kv[:, :heads], kv[:, heads:])
        q = queries[tokens.flatten().long()]
        out = cache.attend(0, plan, q, groups=groups)
        words = [[words[b][int(parents[b, j])] + [int(tokens[b, j])] for j in range(width)] for b in range(streams)]
        assert cache.lengths.tolist() == [41 + step] * n
        # what the cache holds of every beam is its sequence: a value is rounded once when it is stored and
        # again when a later one of the page's 16 tokens makes the scale grow, by half a final step at most
        for b in range(streams):
            for j in range(width):
                got, ok = contents(cache, 0, b * width + j)
                assert bool(ok.all())
                rows = table[torch.tensor(words[b][j], device=dev)].double()
                pages = cache.table[b * width + j, :-(-(41 + step) // page)].long()
                unit = cache.scale[0, pages].double().permute(1, 2, 0).repeat_interleave(page, 2)[..., :41 + step, None]
                both = torch.stack([rows[:, :heads], rows[:, heads:]]).permute(0, 2, 1, 3)
                assert bool(((got - both).abs() <= 8.5 * unit).all())
        want, _, tol, _ = attend_ref(cache, 0, list(range(n)), [1] * n, q, 0, 0, True, dim ** -0.5)
        full = tol * (1 + 2.0 ** -8) + ULP[torch.float16] * want.abs() + F16_TINY
        assert bool(((out.double() - want).abs() <= full).all())
        x = out.float().flatten(1)
    assert int(cache.refs.sum()) == int((cache.table >= 0).sum())
    cache.release(plan)
    assert int(cache.refs.sum()) == 0
    _clean(ufb)
