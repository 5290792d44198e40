"""GPU: the latent-attention operators (rotary positions, 8-bit paged cache,
attention over it, pages) against plain 64-bit implementations.

Tolerances follow from the number formats.  u is half a unit in the last place
of the output type (2^-24, 2^-11, 2^-8 relative for float32, float16, bfloat16,
one more bit than the rounding needs).  Rotary: two 32-bit products and a sum of
table values rounded to 32 bits, below 2^-21 (|a| + |b|).  Attention: the weights
enter the tensor cores with 11 significant bits, so the sum over p v errs by up
to 2^-11 sum p |v|; a score errs by up to 2^-16 sum |q k| scale (128 products
summed in 32 bits, in any order, and the conversion to base 2), which moves each
weight by twice that.  Integers of the cache and of the page tables are equal.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

ULP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
F16_TINY = 2.0 ** -25  # half the spacing of float16 near zero


def gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def randn(dev, shape, seed, dtype=torch.float32, mul=1.0):
    return (torch.randn(shape, device=dev, generator=gen(dev, seed)) * mul).to(dtype)


def _clean(ufb):
    assert ufb.device_status(0) == 0


# ----------------------------------------------------------------- rotary ----

def rotary_ref(x, positions, pairs, bases, layout, inverse):
    y = x.double().clone()
    n, at = sum(pairs), 0
    bound = torch.zeros_like(y)
    for a, p in enumerate(pairs):
        for i in range(p):
            angle = positions[:, a].double() * bases[a] ** (-i / p) * (-1 if inverse else 1)
            c, s = angle.cos()[:, None], angle.sin()[:, None]
            j = at + i
            e, f = (j, j + n) if layout == "half" else (2 * j, 2 * j + 1)
            u, v = x[..., e].double(), x[..., f].double()
            y[..., e], y[..., f] = u * c - v * s, u * s + v * c
            bound[..., e] = bound[..., f] = u.abs() + v.abs()
        at += p
    return y, bound


ROTARY = [
    # tokens, hq, hk, dim, pairs, extents, layout, dtype
    (1, 1, 1, 64, (32,), (4096,), "half", torch.float16),
    (5, 3, 1, 64, (8, 12, 12), (16, 22, 40), "half", torch.bfloat16),
    (33, 4, 2, 128, (11, 19, 20), (64, 68, 120), "half", torch.bfloat16),       # partner at an odd offset
    (17, 5, 5, 80, (3, 7, 9), (9, 31, 33), "half", torch.float16),              # 19 of 40 pairs, copied tail
    (29, 2, 1, 128, (1, 20, 22, 21), (5, 6, 7, 8), "half", torch.float32),
    (64, 6, 3, 64, (4, 8, 7), (16, 22, 40), "interleaved", torch.float32),
    (31, 3, 2, 96, (5, 17, 13), (3, 68, 120), "interleaved", torch.bfloat16),
    (7, 8, 1, 256, (40, 44, 44), (3, 68, 120), "interleaved", torch.float16),
    (20011, 8, 2, 64, (10, 11, 11), (32, 68, 120), "half", torch.float16),      # several heads to a thread
]


@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("case", ROTARY, ids=lambda c: f"{c[0]}x{c[1]}x{c[3]}-{c[6]}-{str(c[7])[6:]}")
def test_rotary(ufb, dev, case, inverse):
    tokens, hq, hk, dim, pairs, extents, layout, dtype = case
    bases = [10000.0, 100.0, 50.0, 30.0][:len(pairs)]
    rot = ufb.Rotary(pairs, extents, bases, layout, device=dev)
    pos = torch.stack([torch.randint(0, e, (tokens,), generator=gen(dev, i), device=dev)
                       for i, e in enumerate(extents)], 1).to(torch.int32)
    pos[0] = torch.tensor([e - 1 for e in extents])  # the last position of every axis
    qkv = randn(dev, (tokens, hq + 2 * hk, dim), 7, dtype)
    q, k = qkv[:, :hq], qkv[:, hq:hq + hk]
    got = rot.apply(pos, q, k, inverse=inverse)
    for x, y in zip((q, k), got):
        want, bound = rotary_ref(x, pos, pairs, bases, layout, inverse)
        assert y.shape == x.shape and y.dtype == dtype
        tol = ULP[dtype] * want.abs() + 2.0 ** -21 * bound + (F16_TINY if dtype == torch.float16 else 0)
        assert bool(((y.double() - want).abs() <= tol).all())
    n = sum(pairs)
    assert torch.equal(got[0][..., 2 * n:], q[..., 2 * n:])  # past the pairs: copied bit for bit
    one = rot.apply(pos, q, inverse=inverse)
    assert torch.equal(one, got[0])
    _clean(ufb)


def test_rotary_gradient(ufb, dev):
    """The inverse is the transpose, and agrees with differences of the forward."""
    pairs, extents = (5, 6, 9), (30, 40, 50)
    for layout in ("half", "interleaved"):
        rot = ufb.Rotary(pairs, extents, (10000.0, 100.0, 100.0), layout, device=dev)
        pos = torch.randint(0, 30, (6, 3), generator=gen(dev, 1), device=dev, dtype=torch.int32)
        x, g = randn(dev, (6, 2, 48), 2), randn(dev, (6, 2, 48), 3)
        grad = rot.apply(pos, g, inverse=True)
        left, right = (rot.apply(pos, x).double() * g).sum(), (grad.double() * x).sum()
        size = (x.double().abs() * g.abs()).sum()
        assert abs(float(left - right)) <= 2.0 ** -20 * float(size) * 2
        # d loss / d x[t, h, e], loss = <apply(x), g>; the map is linear, so a step of 1 has no curvature error
        for t, h, e in [(0, 0, 0), (1, 1, 7), (2, 0, 19), (3, 1, 20), (4, 0, 39), (5, 1, 40), (5, 0, 47)]:
            up, down = x.clone(), x.clone()
            up[t, h, e] += 1.0
            down[t, h, e] -= 1.0
            diff = ((rot.apply(pos, up).double() - rot.apply(pos, down).double()) * g).sum() / 2
            # each of the 48 outputs of the head errs by 2^-21 of its pair's size at most
            tol = 2.0 ** -20 * float((g[t, h].double().abs() * (x[t, h].double().abs().max() + 1) * 2).sum())
            assert abs(float(diff - grad[t, h, e].double())) <= tol
        back = rot.apply(pos, rot.apply(pos, x), inverse=True)
        assert float((back - x).abs().max()) <= 2.0 ** -20 * 2 * float(x.abs().max())


def test_rotary_position_out_of_range(ufb, dev):
    rot = ufb.Rotary((4, 4), (10, 20), device=dev)
    _clean(ufb)
    x = randn(dev, (4, 2, 16), 1, torch.float16)
    pos = torch.tensor([[9, 19], [10, 0], [0, -1], [0, 0]], dtype=torch.int32, device=dev)
    y = rot.apply(pos, x)
    assert ufb.device_status(0) == 21
    assert bool(torch.isnan(y[1:3]).all()) and not bool(torch.isnan(y[[0, 3]]).any())
    _clean(ufb)


def test_rotary_empty_and_refusals(ufb, dev):
    rot = ufb.Rotary((4, 4), (10, 20), device=dev)
    none = torch.empty((0, 2), dtype=torch.int32, device=dev)
    assert rot.apply(none, torch.empty((0, 3, 32), dtype=torch.float16, device=dev)).shape == (0, 3, 32)
    pos = torch.zeros((2, 2), dtype=torch.int32, device=dev)
    x = torch.zeros((2, 1, 32), dtype=torch.float16, device=dev)
    for args in [(pos.long(), x), (pos[:1], x), (pos[:, :1], x), (pos, x.cpu()), (pos, x.double()), (pos, x[:, 0]),
                 (pos, x[..., :8]), (pos, x, x.float())]:
        with pytest.raises(ufb.UfbError):
            rot.apply(*args)
    with pytest.raises(ufb.UfbError):
        ufb.Rotary((20, 20), (4, 4), device=dev).apply(pos, x)  # 40 pairs in a head of 32
    _clean(ufb)


# ------------------------------------------------------------- the cache ----

def make_cache(ufb, dev, lengths, heads, dim, page, seed=0, layers=1, spare=2, slots=None):
    """A cache whose streams own scattered pages of random integers."""
    rng = np.random.default_rng(seed)
    counts = [-(-n // page) for n in lengths]
    pages = sum(counts) + spare
    slots = slots or len(lengths)
    cache = ufb.KVCache(layers, pages, heads, dim, page, slots, max(max(counts), 1) + 2, device=dev)
    order, at = rng.permutation(pages), 0
    table, refs = np.full((slots, cache.table_width), -1, np.int32), np.zeros(pages, np.int32)
    for b, k in enumerate(counts):
        table[b, :k] = order[at:at + k]
        refs[order[at:at + k]] = 1
        at += k
    cache.table.copy_(torch.from_numpy(table))
    cache.refs.copy_(torch.from_numpy(refs))
    cache.lengths[:len(lengths)] = torch.tensor(lengths, dtype=torch.int32)
    cache.kv.copy_(torch.randint(-127, 128, cache.kv.shape, generator=gen(dev, seed + 1), device=dev, dtype=torch.int8))
    cache.scale.copy_(torch.rand(cache.scale.shape, generator=gen(dev, seed + 2), device=dev) * 0.02 + 0.005)
    return cache


def contents(cache, layer, slot):
    """[2, heads, length, dim] in 64 bits, and which tokens have a page."""
    n = int(cache.lengths[slot])
    ids = cache.table[slot, :-(-n // cache.page_tokens)].long()
    ok = ids >= 0
    ids = ids.clamp(min=0)
    x = cache.kv[layer, ids].double() * cache.scale[layer, ids].double()[..., None, None]
    x = x.permute(1, 2, 0, 3, 4).flatten(2, 3)[:, :, :n]
    return x, ok.repeat_interleave(cache.page_tokens)[:n]


def attend_ref(cache, layer, slots, counts, q, window, sinks, causal, scale):
    """out, lse and the tolerance of out's sum and of lse, in 64 bits."""
    group = q.shape[1] // cache.heads
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    tol, tol_lse = torch.zeros_like(out), torch.zeros_like(lse)
    ids = {s: cache.table[s, :-(-int(cache.lengths[s]) // cache.page_tokens)].long().clamp(min=0) for s in slots}
    t = 0
    for slot, n in zip(slots, counts):
        kv, ok = contents(cache, layer, slot)
        length = kv.shape[2]
        key = torch.arange(length, device=q.device)
        at = length - n + torch.arange(n, device=q.device)[:, None]
        seen = (key <= at) if causal else (key < length).expand(n, length)
        if window:
            seen = seen & ((key > at - window) | (key < sinks))
        seen = seen & ok
        for h in range(q.shape[1]):
            k, v = kv[0, h // group], kv[1, h // group]
            x = q[t:t + n, h].double()
            s = (x @ k.T) * scale
            size = (x.abs() @ k.T.abs()) * abs(scale)
            s = torch.where(seen, s, -math.inf)
            some = seen.any(1)
            if length == 0 or not bool(some.any()):
                continue
            l = torch.logsumexp(s[some], 1)
            p = torch.exp(s[some] - l[:, None])
            err = 2.0 ** -16 * torch.where(seen, size, 0).amax(1)[some] + 2.0 ** -20
            rows = torch.nonzero(some)[:, 0] + t
            out[rows, h] = p @ v
            lse[rows, h] = l
            unit = cache.scale[layer, ids[slot], 1, h // group].double().repeat_interleave(cache.page_tokens)[:length]
            steps = torch.where(unit[:, None] > 0, v.abs() / unit[:, None], 0)
            small = 2.0 ** -38 * (p * unit).amax(1)[:, None] * (seen[some].double() @ steps)
            tol[rows, h] = (p @ v.abs()) * (2.0 ** -11 + 2 * err[:, None]) + small
            tol_lse[rows, h] = err + 2.0 ** -20 * l.abs()
        t += n
    return out, lse, tol, tol_lse


def check_attend(ufb, cache, slots, counts, hq, dtype, window=0, sinks=0, causal=True, scale=None, mul=1.0, seed=5,
                 layer=0, fused=True):
    plan = cache.plan(slots, counts)
    qkv = randn(cache.device, (sum(counts), hq + 2 * cache.heads, cache.head_dim), seed, dtype, mul)
    q = qkv[:, :hq] if fused else qkv[:, :hq].contiguous()
    got, lse = cache.attend(layer, plan, q, window=window, sinks=sinks, causal=causal, scale=scale, lse=True)
    want, wl, tol, tl = attend_ref(cache, layer, slots, counts, q, window, sinks, causal,
                                   cache.head_dim ** -0.5 if scale is None else scale)
    full = tol + ULP[dtype] * want.abs() + (F16_TINY if dtype == torch.float16 else 0)
    # queries that are not finite (float16 overflow in the inputs) give NaN, for the whole head
    lost = torch.isnan(want).any(-1)
    assert bool(torch.isnan(got[lost]).all()) and bool(torch.isnan(lse[lost]).all())
    wl = torch.where(lost, 0, wl)
    error = torch.where(lost[..., None], 0, (got.double() - want).abs())
    full = torch.where(lost[..., None], 0, full)
    assert bool((error <= full).all()), float((error - full).max())
    empty = torch.isinf(wl)
    assert bool((lse[empty] == -math.inf).all()) and bool((got[empty] == 0).all())
    known = ~empty & ~lost
    assert bool(((lse.double() - wl).abs()[known] <= tl[known]).all())
    again = cache.attend(layer, plan, q, window=window, sinks=sinks, causal=causal, scale=scale)
    assert torch.equal(again[~lost], got[~lost])  # no order of work shows
    _clean(ufb)
    return got


SHAPES = [(1, 1, 64, 16), (2, 4, 64, 32), (2, 5, 128, 64), (3, 3, 128, 128), (1, 8, 128, 16), (1, 128, 64, 64)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("heads,group,dim,page", SHAPES)
def test_attend_single_tokens(ufb, dev, heads, group, dim, page, dtype):
    """One token a stream: lengths from one token to many pages, odd ones."""
    lengths = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 777, 2500]
    cache = make_cache(ufb, dev, lengths, heads, dim, page)
    check_attend(ufb, cache, list(range(len(lengths))), [1] * len(lengths), heads * group, dtype)


@pytest.mark.parametrize("new", [1, 2, 3, 7, 16, 33, 130, 300])
@pytest.mark.parametrize("heads,group,dim,page", SHAPES)
def test_attend_pieces(ufb, dev, heads, group, dim, page, new):
    """Several tokens a stream, ragged, causal and not."""
    counts = [new, max(1, new // 2), 1, 0, new]
    lengths = [new, 300 + new // 2, 40, 9, 1000 + new]
    cache = make_cache(ufb, dev, lengths, heads, dim, page, seed=new)
    for causal in (True, False):
        check_attend(ufb, cache, [0, 1, 2, 3, 4], counts, heads * group, torch.bfloat16, causal=causal)


@pytest.mark.parametrize("new", [1, 9, 200])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 5), (16, 16), (63, 7), (64, 0), (300, 64), (5000, 3), (100, 2000)])
def test_attend_window_sinks(ufb, dev, window, sinks, new):
    lengths, counts = [new, 300, 1500], [new, min(new, 300), new]
    for page, dim in ((16, 64), (64, 128)):
        cache = make_cache(ufb, dev, lengths, 2, dim, page, seed=window)
        for causal in (True, False):
            check_attend(ufb, cache, [0, 1, 2], counts, 6, torch.float16, window=window, sinks=sinks, causal=causal)


@pytest.mark.parametrize("new", [1, 40])
def test_attend_rows_that_see_nothing(ufb, dev, new):
    """Dropped pages, empty streams and queries before the first key give zeros."""
    cache = make_cache(ufb, dev, [500, 0, 10, 200], 2, 128, 32)
    cache.table[0, 3:9] = -1
    cache.table[3, :] = -1
    check_attend(ufb, cache, [0, 1, 2, 3], [new] * 4, 4, torch.bfloat16)
    check_attend(ufb, cache, [3, 0, 2, 1], [new] * 4, 4, torch.bfloat16, window=7, sinks=0)


@pytest.mark.parametrize("mul,scale", [(30.0, None), (1e-6, None), (1.0, 4.0), (1.0, 0.0), (1.0, -0.1), (3e4, 1e-5)])
@pytest.mark.parametrize("new", [1, 50])
def test_attend_score_ranges(ufb, dev, mul, scale, new):
    """Large, tiny, equal and negative scores; queries near the float16 limit."""
    cache = make_cache(ufb, dev, [700, 90], 2, 64, 16)
    check_attend(ufb, cache, [0, 1], [new, new], 6, torch.float16, mul=mul, scale=scale)
    check_attend(ufb, cache, [0, 1], [new, new], 6, torch.bfloat16, mul=mul, scale=scale)


@pytest.mark.parametrize("new", [1, 70])
def test_attend_queries_beyond_float16(ufb, dev, new):
    """bfloat16 queries whose values float16 cannot hold."""
    cache = make_cache(ufb, dev, [400], 1, 128, 64)
    check_attend(ufb, cache, [0], [new], 3, torch.bfloat16, mul=1e20, scale=1e-21)
    check_attend(ufb, cache, [0], [new], 3, torch.bfloat16, mul=1e-20, scale=1e19)


@pytest.mark.parametrize("new", [1, 70])
def test_attend_scales_of_very_different_size(ufb, dev, new):
    """Pages of zeros, and value scales over eight decades; the heaviest page sets the error."""
    cache = make_cache(ufb, dev, [640], 2, 64, 16)
    pages = cache.table[0, :40].long()
    cache.scale[0, pages[5]] = 0.0
    cache.kv[0, pages[5]] = 0
    spread = torch.logspace(-4, 4, 40, device=dev)[torch.randperm(40, generator=gen(dev, 3), device=dev)]
    cache.scale[0, pages, 1] *= spread[:, None]
    check_attend(ufb, cache, [0], [new], 4, torch.bfloat16)
    # only pages of zero values: weights still count, the result is zero
    cache.scale[0, :, 1] = 0.0
    check_attend(ufb, cache, [0], [new], 4, torch.float16)


@pytest.mark.parametrize("new", [1, 65])
def test_attend_ignores_what_is_not_visible(ufb, dev, new):
    """Not-finite scales and stale integers of hidden pages and slots change nothing."""
    cache = make_cache(ufb, dev, [900], 2, 128, 64, spare=3)
    plan = cache.plan([0], [new])
    q = randn(dev, (new, 4, 128), 3, torch.bfloat16)
    want = cache.attend(0, plan, q, window=100, sinks=3)
    last = int(cache.table[0, 14])
    cache.kv[0, last, :, :, 900 % 64:] = -128
    for e in range(1, 10):  # beyond the sinks' page, before the window
        if (e + 1) * 64 <= 900 - new - 100:
            cache.scale[0, int(cache.table[0, e])] = float("nan") if e % 2 else float("inf")
    free = (cache.refs == 0)
    cache.scale[0, free] = float("nan")
    assert torch.equal(cache.attend(0, plan, q, window=100, sinks=3), want)
    _clean(ufb)


def test_attend_long_stream_and_layers(ufb, dev):
    """A long stream split over the GPU; another layer; queries of a plain tensor."""
    cache = make_cache(ufb, dev, [70001, 3], 1, 64, 64, layers=2)
    for new in (1, 6, 129):
        check_attend(ufb, cache, [0, 1], [new, 1], 8, torch.bfloat16, layer=1, fused=False)


def test_attend_offsets_beyond_32_bits(ufb, dev):
    """Pages past byte 2^32 of the cache."""
    page_bytes = 2 * 8 * 128 * 128
    pages = 2 ** 32 // page_bytes + 24
    cache = ufb.KVCache(1, pages, 8, 128, 128, 1, 16, device=dev)
    ids = torch.arange(pages - 9, pages, dtype=torch.int32, device=dev)
    cache.table[0, :9] = ids
    cache.refs[ids.long()] = 1
    cache.lengths[0] = 9 * 128 - 5
    cache.kv[0, pages - 9:] = torch.randint(-127, 128, cache.kv[0, pages - 9:].shape, generator=gen(dev, 1), device=dev,
                                            dtype=torch.int8)
    cache.scale[0, pages - 9:] = 0.01
    for new in (1, 100):
        check_attend(ufb, cache, [0], [new], 16, torch.float16)
    plan = cache.plan([0], [200])
    k, v = randn(dev, (200, 8, 128), 1, torch.float16), randn(dev, (200, 8, 128), 2, torch.float16)
    cache.append(0, plan, k, v)
    x, _ = contents(cache, 0, 0)
    assert float((x[0, :, -200:].permute(1, 0, 2) - k.double()).abs().max()) <= 0.51 * float(cache.scale.max())
    _clean(ufb)


def test_attend_other_streams(ufb, dev):
    """Calls on two streams do not share scratch."""
    cache = make_cache(ufb, dev, [5000, 4000], 2, 128, 64)
    plans = [cache.plan([0], [3]), cache.plan([1], [3])]
    q = randn(dev, (3, 8, 128), 1, torch.float16)
    want = [cache.attend(0, p, q) for p in plans]
    side = [torch.cuda.Stream(dev) for _ in plans]
    torch.cuda.synchronize(dev)
    got = []
    for _ in range(20):
        for s, p in zip(side, plans):
            with torch.cuda.stream(s):
                got.append(cache.attend(0, p, q))
    torch.cuda.synchronize(dev)
    for i, g in enumerate(got):
        assert torch.equal(g, want[i % 2])
    _clean(ufb)


def test_attend_in_a_graph(ufb, dev):
    """The step is capturable; replays follow the lengths on the device."""
    cache = make_cache(ufb, dev, [300, 200], 2, 64, 32, spare=8)
    plan = cache.plan([0, 1], [1, 1])
    k, v, q = (randn(dev, (2, h, 64), i, torch.float16) for i, h in enumerate((2, 2, 4)))
    side = torch.cuda.Stream(dev)
    with torch.cuda.stream(side):
        cache.attend(0, plan, q)  # this stream's workspace
    torch.cuda.synchronize(dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        cache.extend(plan)
        cache.append(0, plan, k, v)
        out = cache.attend(0, plan, q)
    for step in range(3):
        graph.replay()
        torch.cuda.synchronize(dev)
        assert cache.lengths.tolist() == [301 + step, 201 + step]
        want, _, tol, _ = attend_ref(cache, 0, [0, 1], [1, 1], q, 0, 0, True, 64 ** -0.5)
        assert bool(((out.double() - want).abs() <= tol + ULP[torch.float16] * want.abs() + F16_TINY).all())
    _clean(ufb)


def test_attend_captured_without_an_earlier_call(ufb, dev):
    """The scratch of a capturing stream is zero before any graph runs, whichever
    graph runs first; a second capturing stream has to have called before."""
    cache = make_cache(ufb, dev, [3000, 200], 2, 64, 32, spare=8)
    side, other = torch.cuda.Stream(dev), torch.cuda.Stream(dev)
    graphs, outs, qs, plans = [], [], [], []   # a graph reads them at every replay
    for i, new in enumerate((40, 3)):   # tiles of many rows, of few rows
        plan = cache.plan([0, 1], [new, new])
        plans.append(plan)
        q = randn(dev, (2 * new, 4, 64), i, torch.float16)
        torch.cuda.synchronize(dev)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append(cache.attend(0, plan, q))
        graphs.append(graph)
        qs.append((q, new))
    (scratch,) = [w[2] for w in cache._workspaces.values()]
    assert not bool(scratch.any())
    for i in (1, 0, 1):
        outs[i].fill_(float("nan"))
        graphs[i].replay()
        torch.cuda.synchronize(dev)
        q, new = qs[i]
        want, _, tol, _ = attend_ref(cache, 0, [0, 1], [new, new], q, 0, 0, True, 64 ** -0.5)
        assert bool(((outs[i].double() - want).abs() <= tol + ULP[torch.float16] * want.abs() + F16_TINY).all())
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(ufb.UfbError, match="before capturing"):
        with torch.cuda.graph(graph, stream=other):
            cache.attend(0, plan, q)
    _clean(ufb)


@pytest.mark.parametrize("new", [3, 50])
def test_attend_windows_at_the_ends_of_the_range(ufb, dev, new):
    """The largest window is none; queries before the first key keep their place."""
    cache = make_cache(ufb, dev, [100, 2], 2, 64, 16)
    plan = cache.plan([0, 1], [new, new])
    q = randn(dev, (2 * new, 4, 64), 1, torch.bfloat16)
    for causal in (True, False):
        want = cache.attend(0, plan, q, causal=causal)
        for window, sinks in ((2 ** 31 - 1, 0), (2 ** 31 - 1, 2 ** 31 - 1), (1, 2 ** 31 - 1), (2 ** 30, 1)):
            assert torch.equal(cache.attend(0, plan, q, window=window, sinks=sinks, causal=causal), want)
        check_attend(ufb, cache, [0, 1], [new, new], 4, torch.bfloat16, window=2, sinks=1, causal=causal)
    for kw in ({"window": 2 ** 31}, {"sinks": 2 ** 32}, {"window": -2 ** 33}):
        with pytest.raises(ufb.UfbError):
            cache.attend(0, plan, q, **kw)
    with pytest.raises(ufb.UfbError):
        cache.attend(2 ** 32, plan, q)
    _clean(ufb)


def test_attend_refusals(ufb, dev):
    cache = make_cache(ufb, dev, [100, 50], 2, 64, 16)
    plan = cache.plan([0, 1], [2, 1])
    q = torch.zeros((3, 4, 64), dtype=torch.float16, device=dev)
    for bad in (q.float(), q[:2], q[:, :3], q[..., :32], q.cpu(), q[0]):
        with pytest.raises(ufb.UfbError):
            cache.attend(0, plan, bad)
    for kw in ({"window": -1}, {"sinks": -1}, {"scale": float("inf")}, {"scale": float("nan")}):
        with pytest.raises(ufb.UfbError):
            cache.attend(0, plan, q, **kw)
    for layer in (-1, 1):
        with pytest.raises(ufb.UfbError):
            cache.attend(layer, plan, q)
    other = make_cache(ufb, dev, [100, 50], 2, 64, 16)
    with pytest.raises(ufb.UfbError):
        other.attend(0, plan, q)
    for slots, counts in (([0, 0], [1, 1]), ([2], [1]), ([-1], [1]), ([0], [-1]), ([0], [1, 1])):
        with pytest.raises(ufb.UfbError):
            cache.plan(slots, counts)
    for kw in ({"page_tokens": 48}, {"head_dim": 96}, {"pages": 0}, {"heads": 0}):
        with pytest.raises(ufb.UfbError):
            ufb.KVCache(**{**dict(layers=1, pages=4, heads=1, head_dim=64, page_tokens=16, device=dev), **kw})
    empty = cache.plan([], [])
    assert cache.attend(0, empty, q[:0]).shape == (0, 4, 64)
    _clean(ufb)


# ------------------------------------------------------------ append, read ----

def quantise_page(x, old, before, lo):
    """The stated formula in numpy's 32-bit arithmetic: x [n, heads, dim] float32 from token lo on."""
    finite = np.where(np.isfinite(x), np.abs(x), np.float32(0))
    top = finite.max(axis=(0, 2)) if x.size else np.zeros(old.shape[0], np.float32)
    after = np.maximum(before if lo else np.zeros_like(before), top * (np.float32(1) / np.float32(127)))
    unit = np.where(after > 0, after, np.float32(1))
    new = np.clip(np.rint(np.where(np.isnan(x), np.float32(0), x) / unit[None, :, None]), -127, 127)
    new = np.where(after[None, :, None] > 0, new, 0).astype(np.int8)
    kept = np.rint(old[:, :lo].astype(np.float32) * (before / unit)[:, None, None]).astype(np.int8) if lo else None
    return new, kept, after


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,dim,page", [(1, 64, 16), (3, 128, 32), (2, 64, 64), (2, 128, 128)])
def test_append(ufb, dev, heads, dim, page, dtype):
    """Integers and scales equal the formula; values stand within half a step; the rest is untouched."""
    start = [0, 1, page - 1, page, 3 * page + 5, 0]
    counts = [1, 1, 1, page + 3, 2 * page, 3 * page]
    for mul, bad in ((1.0, False), (0.01, False), (50.0, True)):
        cache = make_cache(ufb, dev, [s + c for s, c in zip(start, counts)], heads, dim, page, seed=3)
        plan = cache.plan(range(6), counts)
        kv = randn(dev, (sum(counts), 2 * heads, dim), 9, dtype, mul)
        if bad:
            kv[::7, 0, 3] = float("inf")
            kv[::5, -1, 4] = float("nan")
            kv[::3, 1, 5] = -float("inf")
        k, v = kv[:, :heads], kv[:, heads:]
        kv0, scale0 = cache.kv.cpu().numpy(), cache.scale.cpu().numpy()
        want_kv, want_scale = kv0.copy(), scale0.copy()
        table, t = cache.table.cpu().numpy(), 0
        for b, (s, c) in enumerate(zip(start, counts)):
            for e in range(s // page, -(-(s + c) // page)):
                lo, hi = max(s - e * page, 0), min(s + c - e * page, page)
                for side, x in enumerate((k, v)):
                    at = t + e * page + lo - s
                    vals = x[at:at + hi - lo].float().cpu().numpy()
                    p = table[b, e]
                    new, kept, after = quantise_page(vals, kv0[0, p, side], scale0[0, p, side], lo)
                    want_kv[0, p, side, :, lo:hi] = new.transpose(1, 0, 2)
                    if lo:
                        want_kv[0, p, side, :, :lo] = kept
                    want_scale[0, p, side] = after
            t += c
        cache.append(0, plan, k, v)
        assert np.array_equal(cache.kv.cpu().numpy(), want_kv)
        assert np.array_equal(cache.scale.cpu().numpy(), want_scale)
        first = cache.kv.clone()
        cache.append(0, plan, k, v)  # the same tokens again change nothing
        assert torch.equal(cache.kv, first)
        ids = torch.tensor([int(table[4, 3]), int(table[0, 0]), int(table[5, 2])], dtype=torch.int32, device=dev)
        for out in (torch.float32, dtype):
            want = (cache.kv[0, ids.long()].double() * cache.scale[0, ids.long()].double()[..., None, None])
            got = cache.read(0, ids, out)
            tiny = F16_TINY if out == torch.float16 else 0
            assert bool(((got.double() - want).abs() <= ULP[out] * want.abs() + tiny).all())
    _clean(ufb)


def test_append_zeros_and_one_by_one(ufb, dev):
    """Zeros keep a scale of zero; tokens that arrive one by one stand within their steps."""
    cache = ufb.KVCache(1, 8, 2, 64, 32, 1, 4, device=dev)
    one = cache.plan([0], [1])
    zero = torch.zeros((1, 2, 64), dtype=torch.bfloat16, device=dev)
    cache.scale.fill_(float("nan"))  # stale scales of unused pages do not count
    cache.extend(one)
    cache.append(0, one, zero, zero)
    page = int(cache.table[0, 0])
    assert bool((cache.scale[0, page] == 0).all()) and bool((cache.kv[0, page, :, :, 0] == 0).all())
    xs = [randn(dev, (1, 2, 64), i, torch.bfloat16, 1.0 + i) for i in range(70)]
    for x in xs:
        cache.extend(one)
        cache.append(0, one, x, -x)
    values, _ = contents(cache, 0, 0)
    x = torch.cat(xs).double().permute(1, 0, 2)
    steps = cache.scale[0, cache.table[0, :3].long()].double().amax(dim=(0, 1, 2))
    # every growth of the scale may add half a step of the final scale, shrinking geometrically at worst to 32 of them
    assert float((values[0, :, 1:] - x).abs().max()) <= 16.5 * float(steps)
    assert torch.equal(values[0], -values[1])
    _clean(ufb)


def test_append_without_room(ufb, dev):
    """Tokens without a page are skipped and reported."""
    cache = make_cache(ufb, dev, [40], 1, 64, 16)
    cache.table[0, 1] = -1
    before = cache.kv.clone()
    plan = cache.plan([0], [40])
    x = randn(dev, (40, 1, 64), 1)
    cache.append(0, plan, x, x)
    assert ufb.device_status(0) == 32
    gone = cache.refs == 0
    assert torch.equal(cache.kv[:, gone], before[:, gone])
    cache.append(0, cache.plan([0], [41]), randn(dev, (41, 1, 64), 1), randn(dev, (41, 1, 64), 1))
    assert ufb.device_status(0) == 32  # more new tokens than the stream holds
    with pytest.raises(ufb.UfbError):
        cache.append(0, plan, x, x[:39])
    with pytest.raises(ufb.UfbError):
        cache.append(0, plan, x, x.half())
    with pytest.raises(ufb.UfbError):
        cache.read(0, torch.tensor([0], device=dev))
    got = cache.read(0, torch.tensor([0, cache.pages, -1], dtype=torch.int32, device=dev))
    assert ufb.device_status(0) == 32
    assert bool(torch.isnan(got[1:]).all()) and not bool(torch.isnan(got[0]).any())
    _clean(ufb)


# -------------------------------------------------------------------- pages ----

class Pages:
    """The page operators in plain Python."""

    def __init__(self, pages, slots, width, page):
        self.P, self.width = page, width
        self.table = [[-1] * width for _ in range(slots)]
        self.lengths, self.refs = [0] * slots, [0] * pages
        self.data = {}  # (page, token) -> label

    def drop(self, s, first, end):
        for e in range(first, end):
            p = self.table[s][e]
            if p >= 0:
                self.refs[p] -= 1
                self.table[s][e] = -1

    def free(self):
        return [p for p, r in enumerate(self.refs) if r == 0]

    def extend(self, slots, counts):
        ceil = lambda n: -(-n // self.P)
        need = [ceil(self.lengths[s] + c) - ceil(self.lengths[s]) for s, c in zip(slots, counts)]
        if sum(need) > len(self.free()) or any(ceil(self.lengths[s] + c) > self.width for s, c in zip(slots, counts)):
            return False
        for s, c, n in zip(slots, counts, need):
            for _ in range(n):
                p = self.free()[0]
                self.table[s][ceil(self.lengths[s])] = p
                self.refs[p] = 1
                self.lengths[s] += self.P  # for the next entry; set right below
            self.lengths[s] += c - n * self.P
        return True

    def release(self, slots):
        for s in slots:
            self.drop(s, 0, self.width)
            self.lengths[s] = 0

    def trim(self, slots, window, sinks):
        for s in slots:
            for e in range(self.width):
                if e * self.P >= sinks and (e + 1) * self.P <= self.lengths[s] - window + 1:
                    self.drop(s, e, e + 1)

    def fork(self, src, dst):
        for d in dst:
            self.drop(d, 0, self.width)
            self.lengths[d] = 0
        moves = []
        for s, d in zip(src, dst):
            for e in range(self.lengths[s] // self.P):
                p = self.table[d][e] = self.table[s][e]
                if p >= 0:
                    self.refs[p] += 1
        part = [(s, d) for s, d in zip(src, dst) if self.lengths[s] % self.P and
                self.table[s][self.lengths[s] // self.P] >= 0]
        if len(part) > len(self.free()):
            for d in dst:
                self.drop(d, 0, self.width)
            return None
        for s, d in part:
            p, e = self.free()[0], self.lengths[s] // self.P
            self.table[d][e] = p
            self.refs[p] = 1
            moves.append((self.table[s][e], p, self.lengths[s] % self.P))
        for s, d in zip(src, dst):
            self.lengths[d] = self.lengths[s]
        return moves

    def compact(self):
        live = [p for p, r in enumerate(self.refs) if r]
        holes = [p for p in range(len(live)) if not self.refs[p]]
        moves = list(zip([p for p in live if p >= len(live)], holes))
        for a, b in moves:
            self.refs[b], self.refs[a] = self.refs[a], 0
        place = dict(moves)
        self.table = [[place.get(p, p) for p in row] for row in self.table]
        return moves


def _same(cache, model):
    assert cache.table.tolist() == model.table
    assert cache.lengths.tolist() == model.lengths
    assert cache.refs.tolist() == model.refs


@pytest.mark.parametrize("page,pages,slots,seed", [(16, 40, 5, 0), (32, 300, 12, 1), (64, 5000, 40, 2), (128, 9, 3, 3)])
def test_pages_random_operations(ufb, dev, page, pages, slots, seed):
    """Tables, counts, lengths and the bytes of every page follow a plain model, whatever the order of calls."""
    rng = np.random.default_rng(seed)
    width = max(2, 2 * pages // slots)
    cache = ufb.KVCache(3, pages, 2, 64, page, slots, width, device=dev)
    cache.kv.copy_(torch.randint(-128, 128, cache.kv.shape, generator=gen(dev, seed), device=dev, dtype=torch.int8))
    cache.scale.copy_(torch.rand(cache.scale.shape, generator=gen(dev, seed), device=dev))
    kv, scale = cache.kv.clone(), cache.scale.clone()
    model = Pages(pages, slots, width, page)
    failed = 0
    for step in range(60):
        op = rng.choice(["extend", "extend", "extend", "release", "fork", "fork", "trim", "compact"])
        some = rng.permutation(slots)[:rng.integers(1, slots + 1)].tolist()
        if op == "extend":
            counts = rng.integers(0, 3 * page + 2, len(some)).tolist()
            cache.extend(cache.plan(some, counts))
            ok = model.extend(some, counts)
            assert ufb.device_status(0) == (0 if ok else 31)
            failed += not ok
        elif op == "release":
            some = some[:max(1, len(some) // 2)]
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
            for a, b, n in moves or []:
                kv[:, b, :, :, :n] = kv[:, a, :, :, :n]
                scale[:, b] = scale[:, a]
        else:
            cache.compact()
            for a, b in model.compact():
                kv[:, b], scale[:, b] = kv[:, a], scale[:, a]
        _same(cache, model)
        assert torch.equal(cache.kv, kv) and torch.equal(cache.scale, scale)
    assert pages >= 300 or failed > 0  # the smallest pools ran out at least once
    _clean(ufb)


def test_pages_refusals(ufb, dev):
    cache = make_cache(ufb, dev, [40, 20], 1, 64, 16, slots=4)
    for src, dst in (([0], [0]), ([0, 1], [2, 2]), ([0, 2], [2, 3]), ([0], [4]), ([0, 1], [2])):
        with pytest.raises(ufb.UfbError):
            cache.fork_plan(src, dst)
    with pytest.raises(ufb.UfbError):
        cache.trim(cache.plan([0], [0]), 0)
    with pytest.raises(ufb.UfbError):
        cache.trim(cache.plan([0], [0]), 4, -1)
    before = cache.table.clone(), cache.lengths.clone(), cache.refs.clone()
    cache.extend(cache.plan([0, 1], [1, 4000]))  # the second stream does not fit: nobody grows
    assert ufb.device_status(0) == 31
    for a, b in zip(before, (cache.table, cache.lengths, cache.refs)):
        assert torch.equal(a, b)
    _clean(ufb)


def test_step_with_branches(ufb, dev):
    """Branches that go on by themselves see the shared past and their own tokens."""
    heads, dim = 2, 64
    cache = ufb.KVCache(2, 64, heads, dim, 16, 4, 16, device=dev)
    rot = ufb.Rotary((8, 12, 12), (64, 22, 40), (10000.0, 100.0, 100.0), device=dev)
    first = cache.plan([0], [50])
    pos = torch.randint(0, 22, (50, 3), generator=gen(dev, 0), device=dev, dtype=torch.int32)
    cache.extend(first)
    for layer in range(2):
        q, k = rot.apply(pos, randn(dev, (50, 4, dim), layer, torch.bfloat16), randn(dev, (50, heads, dim), 5 + layer, torch.bfloat16))
        cache.append(layer, first, k, randn(dev, (50, heads, dim), 9 + layer, torch.bfloat16))
    cache.fork(cache.fork_plan([0, 0], [2, 3]))
    step = cache.plan([0, 2, 3], [7, 7, 20])
    cache.extend(step)
    for layer in range(2):
        k, v = randn(dev, (34, heads, dim), 20 + layer, torch.bfloat16), randn(dev, (34, heads, dim), 30, torch.bfloat16)
        cache.append(layer, step, k, v)
        check_attend(ufb, cache, [0, 2, 3], [7, 7, 20], 4, torch.bfloat16, window=30, sinks=4, layer=layer)
    a, _ = contents(cache, 1, 0)
    b, _ = contents(cache, 1, 2)
    assert torch.equal(a[:, :, :48], b[:, :, :48]) and not torch.equal(a[:, :, 50:], b[:, :, 50:])
    assert cache.lengths.tolist() == [57, 0, 57, 70]
    cache.release(cache.plan([0, 2, 3], [0, 0, 0]))
    assert int(cache.refs.sum()) == 0 and int((cache.table >= 0).sum()) == 0
    _clean(ufb)
