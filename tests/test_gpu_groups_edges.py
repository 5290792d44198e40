"""GPU: the ends of what attention over groups takes -- sinks and windows up to the type's
largest, groups that share has not seen as they are, groups that it turned away.

Attention is held to the tolerances of test_gpu_groups.py."""
import ctypes as C
import math
import struct

import pytest
import torch
from test_gpu_attention import _clean, randn
from test_gpu_groups import check_groups, make_groups

pytestmark = pytest.mark.gpu

LARGEST = 2 ** 31 - 1


@pytest.mark.parametrize("window,sinks", [(1, LARGEST), (1, LARGEST - 20), (9, 2 ** 30), (LARGEST, 0), (LARGEST, LARGEST), (2 ** 30, 1)])
def test_sinks_and_windows_of_any_size(ufb, dev, window, sinks):
    """Groups that share little or nothing, whose streams lie together in a tile: a stream's first own key is
    then behind the tile's, and its keys are counted from there."""
    for page, dim, group in ((16, 64, 3), (64, 128, 40)):
        cache, lengths, sizes = make_groups(ufb, dev, [(0, [20, 40, 9, 300]), (130, [5, 5, 90])], 2, dim, page)
        for counts in ([1] * 7, [4, 30, 9, 200, 2, 5, 1]):
            for causal in (True, False):
                check_groups(ufb, cache, list(range(7)), counts, sizes, 2 * group, torch.float16, window=window, sinks=sinks,
                             causal=causal)


# ------------------------------------- groups that share has not seen as they are ----

def refused(ufb, cache, plan, groups, q, status):
    """Their queries see no key, and the status says so."""
    out, lse = cache.attend(0, plan, q, groups=groups, lse=True)
    assert ufb.device_status(0) == status
    assert not bool(out.any()) and bool((lse == -math.inf).all())


def test_attend_between_capture_and_replay(ufb, dev):
    """A captured share has not run: attention before the first replay is refused by the device."""
    cache, lengths, sizes = make_groups(ufb, dev, [(300, [9] * 4), (64, [3] * 2)], 2, 64, 16, spare=40)
    plan = cache.plan(list(range(6)), [2] * 6)
    groups = cache.group_plan(plan, sizes)
    q, k = randn(dev, (12, 6, 64), 1, torch.float16), randn(dev, (12, 2, 64), 2, torch.float16)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.extend(plan)
        cache.share(groups)
        cache.append(0, plan, k, -k)
        out = cache.attend(0, plan, q, groups=groups)
    refused(ufb, cache, plan, groups, q, 33)
    for step in range(2):
        graph.replay()
        assert torch.equal(cache.attend(0, plan, q, groups=groups), out)
        assert cache.lengths.tolist() == [n + 2 * step + 2 for n in lengths]
    _clean(ufb)
    check_groups(ufb, cache, list(range(6)), [2] * 6, sizes, 6, torch.float16)


@pytest.mark.parametrize("change", ["extend", "refused extend", "trim", "release", "fork", "reorder"])
def test_attend_after_replayed_changes(ufb, dev, change):
    """A replay changes tables or lengths behind share: refused until share has seen them, moved pages are not."""
    cache, lengths, sizes = make_groups(ufb, dev, [(300, [9] * 4), (64, [3] * 2), (40, [5])], 2, 64, 16, spare=40)
    plan = cache.plan(list(range(6)), [1] * 6)
    groups = cache.group_plan(plan, sizes[:2])
    beams, fork, last = cache.beam_plan(range(4), 4), cache.fork_plan([0], [6]), cache.plan([6], [0])
    parents = torch.tensor([[1, 1, 0, 0]], dtype=torch.int32, device=dev)
    much = cache.plan([6], [16 * 60])
    calls = {"extend": lambda: cache.extend(plan), "refused extend": lambda: cache.extend(much),
             "trim": lambda: cache.trim(plan, 50), "release": lambda: cache.release(last),
             "fork": lambda: cache.fork(fork), "reorder": lambda: cache.reorder(beams, parents)}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls[change]()
    q = randn(dev, (6, 6, 64), 1, torch.float16)
    cache.share(groups)
    before = cache.attend(0, plan, q, groups=groups)
    cache.compact()   # new ids, the same pages
    assert torch.equal(cache.attend(0, plan, q, groups=groups), before)
    _clean(ufb)
    graph.replay()
    assert ufb.device_status(0) == (31 if change == "refused extend" else 0)
    refused(ufb, cache, plan, groups, q, 33)
    cache.share(groups)
    got = cache.attend(0, plan, q, groups=groups)
    _clean(ufb)
    check_groups(ufb, cache, list(range(6)), [1] * 6, sizes[:2], 6, torch.float16)
    if change in ("refused extend", "release", "fork"):   # streams of no group here
        assert torch.equal(got, before)


# ------------------------------------------------------ groups that are turned away ----

def call_groups(cache, plan, groups, q, out, lse):
    """ufb_kv_attend_groups into given results."""
    heads = lambda t: C.create_string_buffer(struct.pack("@Pqqi4x", t.data_ptr(), t.stride(0), t.stride(1), t.shape[1]))  # noqa: E731
    room = cache._L.ufb_kv_attend_workspace()
    work = torch.zeros(room, dtype=torch.uint8, device=q.device)
    rc = cache._L.ufb_kv_attend_groups(cache._ref, 0, plan._slots, plan._offsets, plan.n, plan.max_new, plan.tokens, 1,
                                       heads(q), heads(out), lse.data_ptr(), 0, 0, 1, 0.125, groups._ref,
                                       work.data_ptr(), room, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert rc == 0


@pytest.mark.parametrize("which", ["first", "offsets"])
def test_attend_over_groups_that_are_not_the_streams(ufb, dev, which):
    """Bounds that do not belong to the batch: attention reports them too, leaves these groups' results alone
    and answers the others."""
    cache, lengths, sizes = make_groups(ufb, dev, [(100, [5] * 3), (200, [5] * 2), (70, [9] * 4)], 2, 64, 16)
    plan = cache.plan(list(range(9)), [2] * 9)
    groups = cache.group_plan(plan, sizes)
    q = randn(dev, (18, 4, 64), 1, torch.float16)
    cache.share(groups)
    want, wl = cache.attend(0, plan, q, groups=groups, lse=True)
    getattr(groups, which)[1] -= 1   # the border between the first two
    cache.share(groups)
    assert ufb.device_status(0) == 32
    out, lse = torch.full_like(want, 7.0), torch.full_like(wl, 7.0)
    call_groups(cache, plan, groups, q, out, lse)
    assert ufb.device_status(0) == 32
    assert bool((out[:10] == 7).all()) and bool((lse[:10] == 7).all())
    assert torch.equal(out[10:], want[10:]) and torch.equal(lse[10:], wl[10:])
    getattr(groups, which)[1] += 1
    cache.share(groups)
    call_groups(cache, plan, groups, q, out, lse)
    assert torch.equal(out, want) and torch.equal(lse, wl)
    _clean(ufb)


def test_attend_over_groups_of_too_many_keys(ufb, dev):
    """2^31 own keys and more: status of share and of attention, queries that see no key; the others' are right."""
    cache, lengths, sizes = make_groups(ufb, dev, [(100, [5] * 3), (70, [9] * 4)], 2, 64, 16)
    plan = cache.plan(list(range(7)), [2] * 7)
    groups = cache.group_plan(plan, sizes)
    q = randn(dev, (14, 4, 64), 1, torch.float16)
    cache.share(groups)
    want, wl = cache.attend(0, plan, q, groups=groups, lse=True)
    cache.lengths[:3] = 2 ** 30   # no table has that many: share alone looks at them
    cache.share(groups)
    assert ufb.device_status(0) == 32
    out, lse = cache.attend(0, plan, q, groups=groups, lse=True)
    assert ufb.device_status(0) == 32
    assert not bool(out[:6].any()) and bool((lse[:6] == -math.inf).all())
    assert torch.equal(out[6:], want[6:]) and torch.equal(lse[6:], wl[6:])
    _clean(ufb)
