"""CPU: argument checks of reorder, share and attention over groups (before any CUDA call)."""
import ctypes as C

import pytest
from test_attention_capi import EINVAL, ERANGE, Heads, _cache, _heads, att  # noqa: F401


def test_reorder_refusals(att):  # noqa: F811
    L = att._lib()
    c = C.byref(_cache(att, slots=200))

    def reorder(slots=4096, parents=4096, n=12, width=4, cache=c):
        return L.ufb_kv_reorder(cache, slots, parents, n, width, None)

    for over in (dict(slots=None), dict(parents=None), dict(n=-4), dict(n=204), dict(n=13), dict(width=0), dict(width=-4),
                 dict(n=4, width=8), dict(cache=None), dict(cache=C.byref(_cache(att, refs=None)))):
        assert reorder(**over) == EINVAL, over
        assert L.ufb_last_error()
    assert reorder(n=130, width=65) == ERANGE
    assert reorder(n=0, slots=None, parents=None) == 0  # nothing to do, no CUDA call
    # room for what a reorder keeps of each stream
    assert L.ufb_kv_work_ints(8, 4) == 16 + 3 * 8 + 3 * 4


def test_group_refusals(att):  # noqa: F811
    L = att._lib()
    c = C.byref(_cache(att, slots=8))
    q = _heads(att, token=1024, heads=4)

    def groups(first=4096, offsets=4096, state=4096, n=2, most=3):
        return att._Groups(first, offsets, state, n, most)

    def share(g, n=4, max_new=2, tokens=5, slots=4096, offsets=4096):
        return L.ufb_kv_share(c, slots, offsets, n, max_new, tokens, C.byref(g) if g else None, None)

    def attend(g, workspace=None, room=0, layer=0, window=0):
        return L.ufb_kv_attend_groups(c, layer, 4096, 4096, 4, 2, 5, 1, C.byref(q), C.byref(q), None, window, 0, 1, 1.0,
                                      C.byref(g) if g else None, workspace, room, None)

    for g in (None, groups(first=None), groups(offsets=None), groups(state=None), groups(state=4100), groups(n=-1), groups(n=0), groups(n=5),
              groups(most=1), groups(most=6)):
        assert share(g) == EINVAL
        assert L.ufb_last_error()
    for over in (dict(slots=None), dict(offsets=None), dict(n=9), dict(max_new=6), dict(tokens=-1)):
        assert share(groups(), **over) == EINVAL, over
    assert share(groups(n=0, first=None, most=0), n=0, max_new=0, tokens=0) == 0
    for over in (dict(layer=2), dict(layer=-1), dict(window=-1)):
        assert attend(groups(), **over) == EINVAL, over
    assert L.ufb_kv_group_ints(2, 4, 5) == 4 + 12 * 2 + 4 + 4 * 5
    for args in ((-1, 4, 5), (2, -1, 5), (2, 4, -1), (2, 4, 1 << 31)):
        assert L.ufb_kv_group_ints(*args) == EINVAL
