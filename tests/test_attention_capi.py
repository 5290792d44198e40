"""CPU: argument checks of the latent-attention entry points (before any CUDA
call), the rotary table, and the refusals of the Python view without a GPU."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

EINVAL, ERANGE = -1, -2


@pytest.fixture(scope="module")
def att(ufb):
    import sys
    return sys.modules[ufb.__name__ + ".attention"]


class Heads(C.Structure):
    """ufb_heads as include/uf_b200.h has it."""
    _fields_ = [("data", C.c_void_p), ("token_stride", C.c_int64), ("head_stride", C.c_int64), ("heads", C.c_int32)]


def _cache(att, **over):
    a = 1 << 20  # a fake device address; no check reads through it
    f = dict(kv=a, scale=a, table=a, lengths=a, refs=a, work=a, layers=2, pages=8, heads=2, page_tokens=64,
             head_dim=128, slots=4, table_width=4)
    f.update(over)
    return att._Cache(*[f[n] for n, _ in att._Cache._fields_])


def _heads(att, data=1 << 24, token=512, head=128, heads=2):
    return Heads(data, token, head, heads)


def test_packed_heads_match_the_struct(att):
    """The Python view packs ufb_heads by itself."""
    h = Heads(1 << 40, 1 << 35, -7, 12)
    assert att._heads(1 << 40, 1 << 35, -7, 12) == bytes(h) and C.sizeof(Heads) == 32
    assert att._heads2(1, 2, 3, 4, 5, 6, 7, 8) == bytes(Heads(1, 2, 3, 4)) + bytes(Heads(5, 6, 7, 8))


def test_rotary_table(att):
    L = att._lib()
    pairs, extents, bases = (C.c_int32 * 2)(3, 5), (C.c_int32 * 2)(7, 11), (C.c_double * 2)(10000.0, 50.0)
    n = L.ufb_rotary_table(2, pairs, extents, bases, None)
    assert n == 2 * (3 * 7 + 5 * 11)
    t = np.empty(n, np.float32)
    assert L.ufb_rotary_table(2, pairs, extents, bases, t.ctypes.data) == n
    at = 0
    for p, e, b in zip(pairs, extents, bases):
        for pos in range(e):
            for i in range(p):
                angle = pos * b ** (-i / p)
                # one rounding to 32 bits of 64-bit values that agree to 2^-50 of the angle
                assert abs(t[at] - math.cos(angle)) <= 2.0 ** -25 + 2.0 ** -50 * angle
                assert abs(t[at + 1] - math.sin(angle)) <= 2.0 ** -25 + 2.0 ** -50 * angle
                at += 2
    for axes, pr, ex, bs in ((0, pairs, extents, bases), (5, pairs, extents, bases), (2, None, extents, bases),
                             (2, (C.c_int32 * 2)(0, 5), extents, bases), (2, pairs, (C.c_int32 * 2)(7, 0), bases),
                             (2, pairs, extents, (C.c_double * 2)(1.0, math.inf)),
                             (2, pairs, extents, (C.c_double * 2)(-1.0, 2.0))):
        assert L.ufb_rotary_table(axes, pr, ex, bs, None) == EINVAL
        assert L.ufb_last_error()


def test_rotary_refusals(att):
    L = att._lib()
    pairs, extents = (C.c_int32 * 2)(16, 16), (C.c_int32 * 2)(8, 8)
    base = dict(table=4096, axes=2, pairs=pairs, extents=extents, layout=0, inverse=0, positions=4096, tokens=3,
                head_dim=64, dtype=1, count=1, x=(Heads * 1)(_heads(att, 1 << 24, 256, 64, 4)),
                out=(Heads * 1)(_heads(att, 1 << 25, 256, 64, 4)))

    def call(**over):
        f = {**base, **over}
        return L.ufb_rotary(*[f[k] for k in ("table", "axes", "pairs", "extents", "layout", "inverse", "positions",
                                             "tokens", "head_dim", "dtype", "count", "x", "out")], None)

    one = lambda *a: (Heads * 1)(_heads(att, *a))
    for over in (dict(axes=0), dict(axes=5), dict(pairs=None), dict(dtype=3), dict(layout=2), dict(head_dim=40),
                 dict(head_dim=272), dict(head_dim=48), dict(count=0), dict(count=3), dict(table=None),
                 dict(positions=None), dict(x=None), dict(x=one(None, 256, 64, 4)), dict(x=one(1 << 24, 256, 64, 0)),
                 dict(x=one((1 << 24) + 8, 256, 64, 4)), dict(x=one(1 << 24, 260, 64, 4)),
                 dict(x=one(1 << 24, 256, 60, 4)), dict(x=one(1 << 24, 256, 32, 4)), dict(x=one(1 << 24, -256, 64, 4)),
                 dict(out=one(1 << 25, 256, 64, 3)), dict(out=one(1 << 24, 256, 64, 4)),
                 dict(out=one((1 << 24) + 512, 256, 64, 4))):
        assert call(**over) == EINVAL, over
        assert L.ufb_last_error()
    assert call(tokens=-1) == ERANGE
    assert call(tokens=0) == 0  # nothing to do, no CUDA call


def test_cache_refusals(att):
    L = att._lib()
    bad = [dict(kv=None), dict(refs=None), dict(work=None), dict(layers=0), dict(pages=0), dict(heads=0),
           dict(slots=0), dict(table_width=0), dict(page_tokens=48), dict(page_tokens=256), dict(head_dim=96),
           dict(kv=(1 << 20) + 64)]
    h = C.byref(_heads(att))
    for over in bad:
        c = C.byref(_cache(att, **over))
        assert L.ufb_kv_extend(c, 4096, 4096, 1, None) == EINVAL, over
        assert L.ufb_kv_release(c, 4096, 1, None) == EINVAL
        assert L.ufb_kv_fork(c, 4096, 4096, 1, None) == EINVAL
        assert L.ufb_kv_trim(c, 4096, 1, 4, 0, None) == EINVAL
        assert L.ufb_kv_compact(c, None) == EINVAL
        assert L.ufb_kv_append(c, 0, 4096, 4096, 1, 1, 1, 1, h, h, None) == EINVAL
        assert L.ufb_kv_read(c, 0, 4096, 1, 0, 4096, None) == EINVAL
        assert L.ufb_kv_attend(c, 0, 4096, 4096, 1, 1, 1, 1, h, h, None, 0, 0, 1, 1.0, 4096, 1 << 30, None) == EINVAL
    for over in (dict(table_width=1 << 25), dict(layers=32767), dict(heads=40000)):
        assert L.ufb_kv_compact(C.byref(_cache(att, **over)), None) == ERANGE, over
    c = C.byref(_cache(att))
    for n in (-1, 5):
        assert L.ufb_kv_release(c, 4096, n, None) == EINVAL
    assert L.ufb_kv_release(c, None, 1, None) == EINVAL
    assert L.ufb_kv_extend(c, 4096, None, 1, None) == EINVAL
    assert L.ufb_kv_trim(c, 4096, 1, 0, 0, None) == EINVAL
    assert L.ufb_kv_trim(c, 4096, 1, 1, -1, None) == EINVAL
    for call in (L.ufb_kv_extend(c, None, None, 0, None), L.ufb_kv_release(c, None, 0, None),
                 L.ufb_kv_fork(c, None, None, 0, None), L.ufb_kv_trim(c, None, 0, 1, 0, None)):
        assert call == 0  # an empty list is nothing to do
    assert L.ufb_kv_work_ints(0, 1) == EINVAL and L.ufb_kv_work_ints(8, 4) >= 8


def test_append_read_attend_refusals(att):
    L = att._lib()
    c = C.byref(_cache(att))
    k = _heads(att)

    def append(layer=0, slots=4096, offsets=4096, n=2, max_new=3, tokens=5, dtype=1, keys=k, values=k):
        return L.ufb_kv_append(c, layer, slots, offsets, n, max_new, tokens, dtype, C.byref(keys) if keys else None,
                               C.byref(values) if values else None, None)

    for over in (dict(layer=-1), dict(layer=2), dict(slots=None), dict(offsets=None), dict(n=5), dict(max_new=-1),
                 dict(max_new=6), dict(tokens=-1), dict(dtype=3), dict(keys=None), dict(values=None),
                 dict(keys=_heads(att, heads=3)), dict(values=_heads(att, token=516)), dict(keys=_heads(att, head=64))):
        assert append(**over) == EINVAL, over
    assert append(n=0, slots=None, offsets=None) == 0
    for args in ((2, 4096, 1, 0, 4096), (0, None, 1, 0, 4096), (0, 4096, 1, 3, 4096), (0, 4096, 1, 0, None),
                 (0, 4096, 1, 0, 4100)):
        assert L.ufb_kv_read(c, *args, None) == EINVAL, args
    assert L.ufb_kv_read(c, 0, 4096, -1, 0, 4096, None) == ERANGE
    q = _heads(att, token=1024, heads=4)

    def attend(q=q, out=q, dtype=1, window=0, sinks=0, scale=1.0, n=1, max_new=1, tokens=1):
        return L.ufb_kv_attend(c, 0, 4096, 4096, n, max_new, tokens, dtype, C.byref(q), C.byref(out), None, window,
                               sinks, 1, scale, None, 0, None)

    for over in (dict(dtype=0), dict(window=-1), dict(sinks=-1), dict(scale=math.inf), dict(scale=math.nan),
                 dict(q=_heads(att, token=1024, heads=3)), dict(out=_heads(att, token=1024, heads=6)),
                 dict(q=_heads(att, data=(1 << 24) + 2, token=1024, heads=4))):
        assert attend(**over) == EINVAL, over
    wide = _heads(att, token=258 * 128, heads=258)
    assert attend(q=wide, out=wide) == ERANGE
    assert attend(n=0) == 0 and attend(max_new=0, tokens=0) == 0


def test_python_view_needs_cuda(ufb):
    with pytest.raises(ufb.UfbError):
        ufb.Rotary((4,), (8,), device="cpu")
    with pytest.raises(ufb.UfbError):
        ufb.KVCache(1, 4, 1, 64, device="cpu")
    for pairs, extents in (((), ()), ((1,) * 5, (1,) * 5), ((4,), (8, 8))):
        with pytest.raises((ufb.UfbError, RuntimeError)):
            ufb.Rotary(pairs, extents, device="cuda:0")
    with pytest.raises(ufb.UfbError):
        ufb.Rotary((4,), (8,), layout="spiral", device="cuda:0")


def test_outputs_that_overlap_themselves(att):
    """Heads of one result, or of the two of a rotary, that share memory are refused; inputs may repeat."""
    L = att._lib()
    pairs, extents = (C.c_int32 * 1)(16), (C.c_int32 * 1)(8)

    def rotary(x, out, tokens=3):
        n = len(x)
        return L.ufb_rotary(4096, 1, pairs, extents, 0, 0, 4096, tokens, 64, 1, n, (Heads * n)(*x), (Heads * n)(*out), None)

    def at(place, token, head, heads):
        return Heads((1 << 24) + place * 2, token, head, heads)

    x, far = at(0, 0, 64, 4), 1 << 20
    for token, head in ((0, 64), (8, 64), (56, 4096), (192, 64), (64, 64), (128, 96), (104, 160), (200, 64)):
        assert rotary([x], [at(far, token, head, 4)]) == EINVAL, (token, head)
        assert b"overlap" in L.ufb_last_error()
    # the second result begins in the first
    assert rotary([x, at(0, 0, 64, 2)], [at(far, 256, 64, 4), at(far + 192, 256, 64, 2)]) == EINVAL
    assert b"overlap" in L.ufb_last_error()
    c, q = C.byref(_cache(att)), _heads(att, token=512, heads=4)
    bad = _heads(att, data=1 << 25, token=128, heads=4)
    assert L.ufb_kv_attend(c, 0, 4096, 4096, 1, 3, 3, 1, C.byref(q), C.byref(bad), None, 0, 0, 1, 1.0, 4096, 1 << 40,
                           None) == EINVAL
    assert b"overlap" in L.ufb_last_error()
