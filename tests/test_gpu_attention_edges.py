"""GPU: the ends of what the latent-attention operators take -- steps that were
refused, queries and scores of any size, pages of zeros, graphs on one stream.

Tolerances are those of test_gpu_attention.py, which derives them: a score errs
by up to 2^-16 sum |q k| scale, so a weight exp(s - s') is known to a factor
exp(2 err)."""
import math

import pytest
import torch

from test_gpu_attention import F16_TINY, ULP, _clean, attend_ref, check_attend, contents, make_cache, randn

pytestmark = pytest.mark.gpu


def stored(cache):
    return cache.kv.clone(), cache.scale.clone(), cache.table.clone(), cache.lengths.clone(), cache.refs.clone()


def same(before, cache):
    return all(torch.equal(a, b) for a, b in zip(before, (cache.kv, cache.scale, cache.table, cache.lengths, cache.refs)))


@pytest.mark.parametrize("new", [3, 30])
def test_append_after_a_refused_extend(ufb, dev, new):
    """A step that got no pages leaves what is stored alone, and its queries see nothing."""
    cache = make_cache(ufb, dev, [47, 20], 2, 64, 16, spare=0, slots=3)
    plan = cache.plan([0], [new])
    x, q = randn(dev, (new, 2, 64), 1, torch.bfloat16), randn(dev, (new, 4, 64), 2, torch.bfloat16)
    before = stored(cache)
    cache.extend(plan)
    assert ufb.device_status(0) == 31
    cache.append(0, plan, x, -x)
    assert ufb.device_status(0) == 31 and same(before, cache)
    out, lse = cache.attend(0, plan, q, lse=True)
    assert ufb.device_status(0) == 31 and not bool(out.any()) and bool((lse == -math.inf).all())
    # another stream goes on as ever
    check_attend(ufb, cache, [1], [1], 4, torch.bfloat16)
    # a step that is granted takes it off, one of no tokens too
    cache.extend(cache.plan([0], [0]))
    check_attend(ufb, cache, [0], [new], 4, torch.bfloat16)
    cache.extend(plan)
    assert ufb.device_status(0) == 31
    cache.release(cache.plan([1], [0]))
    cache.extend(plan)
    cache.append(0, plan, x, -x)
    check_attend(ufb, cache, [0], [new], 4, torch.bfloat16)
    assert cache.lengths.tolist() == [47 + new, 0, 0]
    got, _ = contents(cache, 0, 0)
    steps = float(cache.scale[0, cache.table[0, 47 // 16:-(-(47 + new) // 16)].long()].max())
    assert float((got[0, :, 47:] - x.double().permute(1, 0, 2)).abs().max()) <= 0.501 * steps
    _clean(ufb)


def test_append_to_shared_pages_after_a_refused_extend(ufb, dev):
    """Branches that share a full last page keep it, and each other's tokens, when neither is granted its step;
    a branch made in between is left out as its source is."""
    cache = make_cache(ufb, dev, [48], 2, 128, 16, layers=2, spare=0, slots=5)
    cache.fork(cache.fork_plan([0, 0], [1, 2]))
    assert cache.refs.max() == 3
    step = cache.plan([1, 2, 4], [20, 7, 0])
    x = randn(dev, (27, 2, 128), 1, torch.float16)
    before = stored(cache)
    cache.extend(step)
    for layer in range(2):
        cache.append(layer, step, x, -x)
        out = cache.attend(layer, step, randn(dev, (27, 4, 128), 2, torch.float16), causal=False)
        assert not bool(out.any())
    assert ufb.device_status(0) == 31 and same(before, cache)
    cache.fork(cache.fork_plan([1, 0], [3, 4]))
    before = stored(cache)
    late = cache.plan([3], [5])
    cache.append(0, late, x[:5], x[:5])
    assert ufb.device_status(0) == 31 and same(before, cache)
    check_attend(ufb, cache, [0, 4], [3, 1], 4, torch.float16)   # these asked for nothing
    cache.release(late)
    assert cache.refs.max() == 4
    # its own pages again: the step is granted
    cache.release(cache.plan([0, 1, 2, 4], [0] * 4))
    cache.extend(late)
    cache.append(0, late, x[:5], x[:5])
    check_attend(ufb, cache, [3], [5], 4, torch.float16)
    _clean(ufb)


def test_refused_steps_of_a_graph(ufb, dev):
    """A captured step that runs out of pages stops changing what is stored."""
    cache = make_cache(ufb, dev, [29, 30], 1, 64, 16, spare=2)
    plan = cache.plan([0, 1], [9, 4])
    x, q = randn(dev, (13, 1, 64), 1, torch.float16), randn(dev, (13, 4, 64), 2, torch.float16)
    side = torch.cuda.Stream(dev)
    torch.cuda.synchronize(dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        cache.extend(plan)
        cache.append(0, plan, x, x)
        out = cache.attend(0, plan, q)
    granted = 0
    for step in range(4):
        before = stored(cache)
        graph.replay()
        torch.cuda.synchronize(dev)
        status = ufb.device_status(0)
        if status:
            assert status == 31 and same(before, cache) and not bool(out.any())
        else:
            granted += 1
            want, _, tol, _ = attend_ref(cache, 0, [0, 1], [9, 4], q, 0, 0, True, 64 ** -0.5)
            assert bool(((out.double() - want).abs() <= tol + ULP[torch.float16] * want.abs() + F16_TINY).all())
    assert granted == 2 and cache.lengths.tolist() == [47, 38]


def check_sharp(cache, slots, counts, q, scale):
    """Rows whose best key leads by more than the scores' error give that key's value."""
    plan = cache.plan(slots, counts)
    got, lse = cache.attend(0, plan, q, scale=scale, lse=True)
    assert bool(torch.isfinite(got).all()) and bool(torch.isfinite(lse).all())
    group, t, sharp = q.shape[1] // cache.heads, 0, 0
    for slot, n in zip(slots, counts):
        kv, _ = contents(cache, 0, slot)
        length = kv.shape[2]
        at = length - n + torch.arange(n, device=q.device)[:, None]
        seen = torch.arange(length, device=q.device) <= at
        for h in range(q.shape[1]):
            k, v, x = kv[0, h // group], kv[1, h // group], q[t:t + n, h].double()
            s = torch.where(seen, (x @ k.T) * scale, -math.inf)
            err = 2.0 ** -16 * torch.where(seen, (x.abs() @ k.T.abs()) * scale, 0).amax(1)
            best = s.topk(2, dim=1)
            # the others together: length exp(2 err - lead), below 2^-30 from here on
            lead = best.values[:, 0] - best.values[:, 1]
            clear = lead > 2 * err + math.log(length) + 21
            assert bool(((lse[t:t + n, h].double() - best.values[:, 0]).abs()[clear]
                         <= (err + 2.0 ** -20 * best.values[:, 0].abs())[clear]).all())
            want = v[best.indices[:, 0]]
            tol = (ULP[q.dtype] + 2.0 ** -11) * want.abs() + 2.0 ** -30 * v.abs().max()
            assert bool(((got[t:t + n, h].double() - want).abs() <= tol)[clear].all())
            sharp += int(clear.sum())
        t += n
    assert sharp * 2 > q.shape[0] * q.shape[1]  # the leads of so few keys are far above the error


@pytest.mark.parametrize("mul", [1e5, 1e25, 1e33, 1e36, 2e37])
@pytest.mark.parametrize("heads,dim,page", [(2, 64, 16), (1, 128, 64)])
def test_queries_of_any_size(ufb, dev, heads, dim, page, mul):
    """bfloat16 queries up to the end of their type, scores inside float32's range: few rows."""
    cache = make_cache(ufb, dev, [70, 41], heads, dim, page)
    check_sharp(cache, [0, 1], [3, 1], randn(dev, (4, 3 * heads, dim), 11, torch.bfloat16, mul), dim ** -0.5)
    _clean(ufb)


@pytest.mark.parametrize("new", [1, 40])
def test_scores_beside_an_outlier(ufb, dev, new):
    """Integers of size 1 and 2 beside the one that sets the page's scale keep their scores."""
    cache = make_cache(ufb, dev, [500], 2, 128, 64)
    cache.kv[:, :, 0] = torch.sign(cache.kv[:, :, 0]) * (1 + cache.kv[:, :, 0] % 2)
    cache.scale[:, :, 0] = 10.0 / 127
    q = randn(dev, (new, 6, 128), 4, torch.bfloat16).abs() * 30   # of one sign: sum q is as large as sum |q|
    plan = cache.plan([0], [new])
    got, lse = cache.attend(0, plan, q, lse=True)
    want, wl, tol, tl = attend_ref(cache, 0, [0], [new], q, 0, 0, True, 128 ** -0.5)
    assert bool(((lse.double() - wl).abs() <= tl).all()), float(((lse.double() - wl).abs() / tl).max())
    assert bool(((got.double() - want).abs() <= tol + ULP[torch.bfloat16] * want.abs()).all())
    _clean(ufb)


@pytest.mark.parametrize("mul", [1e5, 1e6, 3e6, 1e7, 3e7, 1e8, 3e8, 1e9, 1e15, 1e25, 1e33, 2e37])
@pytest.mark.parametrize("heads,dim,page", [(2, 64, 16), (1, 128, 64)])
def test_scores_of_any_size_of_many_rows(ufb, dev, heads, dim, page, mul):
    """Scores whose spacing in 32 bits passes 1, in tiles of many rows: masked and not."""
    cache = make_cache(ufb, dev, [70, 600], heads, dim, page)
    check_sharp(cache, [0, 1], [50, 33], randn(dev, (83, 3 * heads, dim), 12, torch.bfloat16, mul), dim ** -0.5)
    _clean(ufb)


@pytest.mark.parametrize("mul", [1e6, 3e6, 1e7, 3e7, 1e8, 3e8])
@pytest.mark.parametrize("heads,dim,page", [(2, 64, 16), (1, 128, 64)])
def test_scores_of_any_size_of_few_rows(ufb, dev, heads, dim, page, mul):
    """The same where the spacing of the scores is about that of the weights' range."""
    cache = make_cache(ufb, dev, [70, 600], heads, dim, page)
    check_sharp(cache, [0, 1], [5, 5], randn(dev, (10, 3 * heads, dim), 13, torch.bfloat16, mul), dim ** -0.5)
    _clean(ufb)


@pytest.mark.parametrize("new", [1, 70])
def test_lse_of_a_long_stream_of_zero_values(ufb, dev, new):
    """The weights of many thousand keys whose values are all zero add up."""
    cache = make_cache(ufb, dev, [40000 if new == 1 else 300000], 1, 64, 64)
    cache.kv[:, :, 1] = 0
    cache.scale[:, :, 1] = 0.0
    check_attend(ufb, cache, [0], [new], 4, torch.bfloat16, mul=0.1)


@pytest.mark.parametrize("new", [1, 40])
def test_queries_with_one_large_value(ufb, dev, new):
    """Where the keys are zero the query is as large as float16 goes: its other values keep theirs."""
    cache = make_cache(ufb, dev, [300], 2, 64, 32)
    cache.kv[:, :, 0, :, :, 5] = 0
    q = randn(dev, (new, 6, 64), 4, torch.float16, 1e-3)
    q[..., 5] = 60000.0
    plan = cache.plan([0], [new])
    got, lse = cache.attend(0, plan, q, scale=100.0, lse=True)
    want, wl, tol, tl = attend_ref(cache, 0, [0], [new], q, 0, 0, True, 100.0)
    assert bool(((lse.double() - wl).abs() <= tl).all()), float(((lse.double() - wl).abs() / tl).max())
    assert bool(((got.double() - want).abs() <= tol + ULP[torch.float16] * want.abs() + F16_TINY).all())
    _clean(ufb)


def test_graphs_of_one_stream(ufb, dev):
    """Graphs captured on one stream, and its own calls, share no scratch: they may run side by side."""
    cache = make_cache(ufb, dev, [5000, 4000, 3000], 2, 128, 64)
    plans = [cache.plan([0], [3]), cache.plan([1], [2]), cache.plan([2], [40])]
    qs = [randn(dev, (p.tokens, 8, 128), i, torch.float16) for i, p in enumerate(plans)]
    want = [cache.attend(0, p, q) for p, q in zip(plans, qs)]
    side, others = torch.cuda.Stream(dev), [torch.cuda.Stream(dev) for _ in range(3)]
    torch.cuda.synchronize(dev)
    graphs, outs, places = [], [], set()
    for p, q in zip(plans, qs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append([cache.attend(0, p, q) for _ in range(3)])
        graphs.append(graph)
        (held,) = cache._captures.values()
        places.add(held[1][0])
    with torch.cuda.stream(side):
        assert torch.equal(cache.attend(0, plans[0], qs[0]), want[0])
    places |= {w[0] for w in cache._workspaces.values()}
    assert len(places) == 5   # three graphs, the default stream, the side stream
    for _ in range(10):
        torch.cuda.synchronize(dev)
        for o in sum(outs, []):
            o.fill_(float("nan"))
        torch.cuda.synchronize(dev)
        for s, graph in zip(others, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        with torch.cuda.stream(side):
            eager = [cache.attend(0, p, q) for p, q in zip(plans, qs)]
        torch.cuda.synchronize(dev)
        for w, e, o in zip(want, eager, outs):
            assert torch.equal(e, w) and all(torch.equal(x, w) for x in o)
    _clean(ufb)


def test_caches_on_two_devices(ufb, dev):
    """One process, two GPUs, one of them not the current device: both kernels run on either."""
    if torch.cuda.device_count() < 2:
        pytest.skip("one GPU")
    for device in (dev, torch.device("cuda:1"), dev):
        cache = make_cache(ufb, device, [300, 70], 2, 64, 16, spare=12)
        for new in (3, 50):
            check_attend(ufb, cache, [0, 1], [new, new], 4, torch.float16)
            plan = cache.plan([0, 1], [new, 1])
            x = randn(device, (new + 1, 2, 64), 1, torch.float16)
            cache.extend(plan)
            cache.append(0, plan, x, x)
        assert ufb.device_status(device.index) == 0


def test_results_in_strided_places(ufb, dev):
    """The C entries write results as parts of one buffer, head after head, or between other rows."""
    import ctypes as C
    import sys
    att = sys.modules[ufb.__name__ + ".attention"]
    stream, t, d = torch.cuda.current_stream(dev).cuda_stream, 5, 64
    rot = ufb.Rotary((8, 12, 12), (64, 22, 40), (10000.0, 100.0, 100.0), device=dev)
    pos = torch.randint(0, 22, (t, 3), generator=torch.Generator(device=dev).manual_seed(1), device=dev, dtype=torch.int32)
    q, k = randn(dev, (t, 4, d), 1, torch.float16), randn(dev, (t, 2, d), 2, torch.float16)
    want = rot.apply(pos, q, k)
    x = att._heads2(q.data_ptr(), 4 * d, d, 4, k.data_ptr(), 2 * d, d, 2)
    # [tokens, 6 heads]; [6 heads, tokens]; heads of two results in turn
    for layout in ((6 * d, d, 4 * d, d), (d, t * d, 4 * t * d, t * d), (8 * d, 2 * d, d, 2 * d)):
        ts, hs, second, hs2 = layout
        out = torch.zeros(64 * t * d, dtype=torch.float16, device=dev)
        y = att._heads2(out.data_ptr(), ts, hs, 4, out.data_ptr() + 2 * second, ts, hs2, 2)
        assert rot._fn(rot._table, 3, rot._pairs_at, rot._extents_at, 0, 0, pos.data_ptr(), t, d, 1, 2, x, y, stream) == 0
        assert torch.equal(torch.as_strided(out, (t, 4, d), (ts, hs, 1)), want[0])
        assert torch.equal(torch.as_strided(out, (t, 2, d), (ts, hs2, 1), second), want[1])
    _clean(ufb)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_in_autograd(ufb, dev, layout):
    """A result of inputs that require a gradient carries it: the inverse turn of its own gradient."""
    rot = ufb.Rotary((5, 6, 9), (30, 40, 50), (10000.0, 100.0, 100.0), layout, device=dev)
    pos = torch.randint(0, 30, (6, 3), generator=torch.Generator(device=dev).manual_seed(1), device=dev, dtype=torch.int32)
    q, k = randn(dev, (6, 4, 48), 2), randn(dev, (6, 2, 48), 3)
    gq, gk = randn(dev, (6, 4, 48), 4), randn(dev, (6, 2, 48), 5)
    for inverse in (False, True):
        plain = rot.apply(pos, q, k, inverse=inverse)
        a, b = q.clone().requires_grad_(), k.clone().requires_grad_()
        y, z = rot.apply(pos, a, b, inverse=inverse)
        assert torch.equal(y, plain[0]) and torch.equal(z, plain[1])
        ((y * gq).sum() + (z * gk).sum()).backward()
        want = rot.apply(pos, gq, gk, inverse=not inverse)
        assert torch.equal(a.grad, want[0]) and torch.equal(b.grad, want[1])
        # one of the two inputs alone, one of the two results alone
        a.grad = None
        rot.apply(pos, a, k, inverse=inverse)[0].backward(gq)
        assert torch.equal(a.grad, want[0])
        b.grad = None
        (rot.apply(pos, q, b, inverse=inverse)[1] * gk).sum().backward()
        assert torch.equal(b.grad, want[1])
        # an input of two uses of a fused projection: the parts' gradients meet in it
        qkv = torch.cat([q, k], 1).requires_grad_()
        y, z = rot.apply(pos, qkv[:, :4], qkv[:, 4:], inverse=inverse)
        ((y * gq).sum() + (z * gk).sum()).backward()
        assert torch.equal(qkv.grad, torch.cat(want, 1))
        x = rot.apply(pos, q.clone().requires_grad_(), inverse=inverse)
        assert x.requires_grad
        with torch.no_grad():
            assert not rot.apply(pos, a, b, inverse=inverse)[0].requires_grad
    assert not rot.apply(pos, q).requires_grad
    _clean(ufb)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
def test_append_infinities_alone(ufb, dev, dtype):
    """Without a finite value other than zero the scale is 0 and every new integer with it;
    beside one, infinities are the ends of the range."""
    cache = ufb.KVCache(1, 4, 2, 64, 16, 1, 4, device=dev)
    cache.kv.fill_(55)
    plan = cache.plan([0], [5])
    cache.extend(plan)
    x = torch.zeros((5, 2, 64), dtype=dtype, device=dev)
    x[0, 0, :4] = torch.tensor([math.inf, -math.inf, math.nan, 0.0])
    x[1, 1, :4] = torch.tensor([math.inf, -math.inf, math.nan, 1.0])
    cache.append(0, plan, x, x)
    page = int(cache.table[0, 0])
    kv, scale = cache.kv[0, page], cache.scale[0, page]
    assert bool((scale[:, 0] == 0).all()) and bool((kv[:, 0, :5] == 0).all())
    assert bool((scale[:, 1] == torch.tensor(1.0 / 127, dtype=torch.float32)).all())
    assert kv[0, 1, 1, :5].tolist() == [127, -127, 0, 127, 0] and torch.equal(kv[0, 1], kv[1, 1])
    assert bool((kv[:, :, 5:] == 55).all())
    _clean(ufb)
