"""GPU: the selection over beams against a plain 64-bit implementation.

A score is s + (l - ln sum exp l), rounded once to 32 bits (half a step, 2^-24 of
it) from a value good to 2^-27, and to 2^-50 of the largest of its terms where these
are large (64-bit sums of them).  Parents and tokens are equal: two continuations of
different beams whose scores are that close and round apart do not occur in the
seeded inputs here; equal rows and equal logits, which have to go by their places, do.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def select_ref(logits, scores, count, finished=None, pad=0):
    logits, scores = logits.double().cpu().numpy(), scores.double().cpu().numpy()
    finished = np.zeros(scores.shape, bool) if finished is None else finished.cpu().numpy()
    streams, beams, vocab = logits.shape
    best = np.full((streams, count), -np.inf)
    parents = np.broadcast_to(np.minimum(np.arange(count), beams - 1), (streams, count)).copy()
    tokens, size = np.zeros((streams, count), int), np.zeros((streams, count))
    for b in range(streams):
        found = []
        for k in range(beams):
            s = scores[b, k]
            if not s > -np.inf:
                continue
            if finished[b, k]:
                found.append((-np.float32(s), k, 0.0, pad, s, 0.0))
                continue
            row = logits[b, k]
            top = row.max()
            if np.isnan(row).any() or not np.isfinite(top):
                continue
            lse = top + np.log(np.exp(row - top).sum())
            order = np.lexsort((np.arange(vocab), -row))[:count]
            for v in order:
                total = s + (row[v] - lse)
                with np.errstate(over="ignore"):
                    if np.float32(total) > -np.inf:
                        found.append((-np.float32(total), k, -row[v], v, total, max(abs(s), abs(row[v]), abs(lse))))
        for i, (_, k, _, v, total, large) in enumerate(sorted(found, key=lambda f: f[:4])[:count]):
            best[b, i], parents[b, i], tokens[b, i], size[b, i] = total, k, v, large
    return best, parents, tokens, size


def check(ufb, logits, scores, count, finished=None, pad=0, status=0):
    got = ufb.beam_select(logits, scores, count, finished, pad)
    assert ufb.device_status(0) == status
    compare(got, select_ref(logits, scores, count, finished, pad))
    return got


def compare(got, want):
    best, parents, tokens = (t.cpu().numpy() for t in got)
    assert best.dtype == np.float32 and parents.dtype == tokens.dtype == np.int32
    assert np.array_equal(parents, want[1])
    assert np.array_equal(tokens, want[2])
    none = np.isneginf(want[0])
    assert np.array_equal(np.isneginf(best), none)
    inf = np.isposinf(want[0])
    assert np.array_equal(np.isposinf(best), inf)
    far = np.abs(np.where(none | inf, 0, best.astype(float)) - np.where(none | inf, 0, want[0]))
    tol = 2.0 ** -24 * np.abs(np.where(none | inf, 0, want[0])) + 2.0 ** -27 + 2.0 ** -50 * want[3] + 2.0 ** -150
    assert (far <= tol).all(), float((far / tol).max())


def inputs(dev, streams, beams, vocab, dtype, seed=1, mul=3.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    logits = (torch.randn((streams, beams, vocab), device=dev, generator=g) * mul).to(dtype)
    return logits, torch.randn((streams, beams), device=dev, generator=g) * 2.0 - 15.0


SIZES = [
    # streams, beams, vocab, count
    (1, 1, 1, 1), (1, 1, 1, 5), (2, 3, 2, 4), (1, 4, 256, 4), (3, 2, 7, 14), (5, 7, 33, 9), (2, 64, 63, 64),
    (1, 64, 1000, 64), (16, 1, 4099, 8), (7, 5, 2048, 10), (3, 8, 8191, 33), (2, 3, 50021, 64), (1, 1, 131071, 17),
    (150, 4, 1025, 3), (700, 2, 129, 2), (1, 9, 16383, 1), (20, 30, 9001, 12), (5000, 1, 130, 3), (3, 64, 30000, 9),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_select(ufb, dev, size, dtype):
    streams, beams, vocab, count = size
    check(ufb, *inputs(dev, streams, beams, vocab, dtype), count)


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])
def test_select_few_rows_of_many(ufb, dev, dtype):
    """Most beams without a score or at their end: the others are shared out by all of the GPU."""
    logits, scores = inputs(dev, 64, 16, 20001, dtype)
    g = torch.Generator(device=dev).manual_seed(9)
    scores[torch.rand(scores.shape, device=dev, generator=g) < 0.9] = -math.inf
    finished = torch.rand(scores.shape, device=dev, generator=g) < 0.3
    check(ufb, logits, scores, 18, finished, pad=3)
    scores[:] = -math.inf
    scores[37, 11] = -2.0
    check(ufb, logits, scores, 64)
    scores[:] = -math.inf
    check(ufb, logits, scores, 2)


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])
def test_select_strides(ufb, dev, dtype):
    logits, scores = inputs(dev, 3, 4, 1200, dtype)
    for view in (logits[:, :, 1:1190], logits[..., 5:], logits[..., ::2], logits.transpose(0, 1)[:3, :3],
                 logits[:1].expand(3, 4, 1200), logits[:, :1].expand(3, 4, 1200), logits.permute(0, 2, 1)[:, :60]):
        s = scores.new_tensor(np.linspace(-9, -1, view.shape[0] * view.shape[1])).view(view.shape[:2])
        check(ufb, view, s, 7)
        check(ufb, view, s.t().contiguous().t(), 7)


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])
def test_select_beams_without_continuations(ufb, dev, dtype):
    logits, scores = inputs(dev, 6, 5, 999, dtype)
    scores[0, 1:] = -math.inf              # the first step of a search
    scores[1] = -math.inf                  # no beam at all
    scores[2, 2] = math.nan
    logits[0, 3] = math.nan                # rows of beams without a score are not read
    logits[2, 2] = math.inf
    logits[3, :, 5:] = -math.inf           # fewer tokens than continuations
    logits[4, 0] = -math.inf               # none allowed
    finished = torch.zeros((6, 5), dtype=torch.bool, device=dev)
    finished[5, 1] = finished[5, 4] = finished[3, 0] = finished[1, 0] = True
    logits[5, 1] = math.nan                # nor are those of beams that have ended
    for count in (1, 9, 30):
        check(ufb, logits, scores, count, finished, pad=7)
    finished[:] = True
    check(ufb, logits, scores, 6, finished, pad=998)


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])
def test_select_rows_that_are_not_finite(ufb, dev, dtype):
    logits, scores = inputs(dev, 3, 4, 777, dtype)
    logits[0, 1, 500], logits[1, 2, 0] = math.nan, math.inf
    logits[2, 0] = math.nan
    logits[2, 1], logits[2, 1, 776] = -math.inf, math.nan
    check(ufb, logits, scores, 12, status=51)


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])
def test_select_equal_values(ufb, dev, dtype):
    """Equal logits go by their tokens, equal rows by their beams."""
    for vocab in (5, 300, 40000):
        flat = torch.zeros((2, 3, vocab), dtype=dtype, device=dev)
        check(ufb, flat, torch.full((2, 3), -4.0, device=dev), 11)
        flat[0, 1] = -0.0
        flat[1, :, vocab // 2:] = 1.0
        check(ufb, flat, torch.full((2, 3), -4.0, device=dev), 5)
    logits, _ = inputs(dev, 1, 1, 20011, dtype, mul=1.0)
    same = logits.round().expand(4, 6, 20011)
    check(ufb, same, torch.full((4, 6), -2.5, device=dev), 40)


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])
def test_select_orders(ufb, dev, dtype):
    """Sorted rows, and the large values of a row all where one thread looks."""
    up = torch.linspace(-6, 6, 30001, device=dev, dtype=torch.float64).to(dtype)
    rows = torch.stack([up, up.flip(0)])[None].repeat(2, 1, 1)
    check(ufb, rows, torch.tensor([[-1.0, -1.5], [-3.0, -1.0]], device=dev), 20)
    for step in (256 * 4, 256 * 8, 2048 * 8):
        x, s = inputs(dev, 1, 2, 90000, dtype)
        x[..., 3::step] = (9 + torch.arange(x[..., 3::step].shape[-1], device=dev) * 0.0625).to(dtype)
        check(ufb, x, s, 64)


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])
def test_select_ranges(ufb, dev, dtype):
    """Logits of any size: far from zero together, and far from one another."""
    logits, scores = inputs(dev, 8, 3, 5003, dtype)
    lowest = torch.finfo(dtype).min
    logits[0] += 700.0
    logits[1] -= 900.0
    logits[2] = lowest                      # masked by the type's lowest value, all of it
    logits[3, :, 17:] = lowest
    logits[4, 0] = -20000.0
    logits[4, 0, 4000] = -19990.0
    logits[5] *= 2000.0 if dtype == torch.float16 else 1e30
    logits[6, :, ::2] = 0.0
    logits[6, :, 2501] = 60000.0
    logits[7, 1] = 650.0
    check(ufb, logits, scores, 21)
    check(ufb, logits, scores * 1e30, 3)
    check(ufb, logits, scores * 3e37, 3)    # scores that leave the range are no continuations
    check(ufb, logits, -scores, 3)
    scores[0, 1] = math.inf
    check(ufb, logits[:1, 1:2], scores[:1, 1:2], 3)


def test_select_is_accurate(ufb, dev):
    """ln sum exp of broad and of narrow rows is good to 2^-27 (the scores here are small)."""
    for mul in (0.01, 1.0, 8.0, 30.0):
        logits, _ = inputs(dev, 4, 2, 65537, torch.float32, seed=3, mul=mul)
        top = logits.max(-1, keepdim=True).values
        logits -= top                       # the best logits are 0
        row = logits.double()
        lse = torch.logsumexp(row, -1)
        # a score that leaves the first continuation near 0, where 32 bits are fine
        scores = lse.float()
        best, parents, _ = ufb.beam_select(logits, scores, 2)
        want = (scores.double() - lse).gather(1, parents.long())
        near = (best - want.float()).abs().double()[:, :1]
        assert float(near.max()) <= 2.0 ** -27 + 2.0 ** -24 * float(want.abs().max())
    assert ufb.device_status(0) == 0


def test_select_on_streams_and_in_graphs(ufb, dev):
    """Calls side by side, and replays of a captured call with other inputs."""
    sets = [inputs(dev, 5, 6, 30011, torch.bfloat16, seed=i) for i in range(4)]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = []
    for (x, s), stream in zip(sets, streams):
        with torch.cuda.stream(stream):
            got.append([ufb.beam_select(x, s, 12) for _ in range(3)])
    torch.cuda.synchronize()
    for (x, s), g in zip(sets, got):
        want = select_ref(x, s, 12)
        for r in g:
            compare(r, want)
    x, s = (t.clone() for t in sets[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = ufb.beam_select(x, s, 12)
    for i in (2, 1, 3):
        x.copy_(sets[i][0])
        s.copy_(sets[i][1])
        graph.replay()
        torch.cuda.synchronize()
        compare(r, select_ref(x, s, 12))
    assert ufb.device_status(0) == 0


def test_select_empty_and_refusals(ufb, dev):
    x, s = inputs(dev, 2, 3, 8, torch.float16)
    none = ufb.beam_select(x[:0], s[:0], 4)
    assert [t.shape for t in none] == [(0, 4)] * 3
    f = torch.zeros((2, 3), dtype=torch.bool, device=dev)
    for args in [(x[0], s, 2), (x.double(), s, 2), (x.cpu(), s, 2), (x, s[:1], 2), (x, s.half(), 2), (x, s.cpu(), 2),
                 (x, s, 0), (x, s, -1), (x, s, 65), (x, s, 1 << 40), (x, s, 2, f.int()), (x, s, 2, f[:1]),
                 (x, s, 2, f.cpu()), (x, s, 2, f, -1), (x[:, :0], s[:, :0], 2), (x[..., :0], s, 2),
                 (torch.zeros((1, 65, 4), device=dev), torch.zeros((1, 65), device=dev), 2)]:
        with pytest.raises(ufb.UfbError):
            ufb.beam_select(*args)
