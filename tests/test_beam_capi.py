"""CPU: argument checks of the selection over beams (before any CUDA call) and
the refusals of the Python view without a GPU."""
import ctypes as C
import sys

import pytest
import torch

EINVAL, ERANGE = -1, -2


@pytest.fixture(scope="module")
def fn(ufb):
    return sys.modules[ufb.__name__ + ".beams"]._entry()


BASE = dict(logits=1 << 20, dtype=2, stream_stride=400, beam_stride=100, scores=4096, finished=None, streams=3, beams=4,
            vocab=100, count=4, pad=0, out_scores=8192, parents=8192, tokens=8192, workspace=1 << 22, room=1 << 30)


def call(fn, **over):
    return fn(*{**BASE, **over}.values(), None)


def test_refusals(ufb, fn):
    L = ufb.library()
    for over in (dict(dtype=3), dict(dtype=-1), dict(streams=-1), dict(beams=0), dict(vocab=0), dict(count=0),
                 dict(count=-4), dict(pad=-1), dict(stream_stride=-1), dict(beam_stride=-8), dict(logits=None),
                 dict(scores=None), dict(out_scores=None), dict(parents=None), dict(tokens=None),
                 dict(logits=(1 << 20) + 1), dict(logits=(1 << 20) + 2, dtype=0)):
        assert call(fn, **over) == EINVAL, over
        assert L.ufb_last_error()
    for over in (dict(beams=65), dict(count=65), dict(vocab=(1 << 25) + 1), dict(streams=(1 << 24) + 1)):
        assert call(fn, **over) == ERANGE, over
    size = dict(dtype=2, streams=3, beams=4, vocab=100, count=4)
    for over, code in ((dict(dtype=3), EINVAL), (dict(streams=-1), EINVAL), (dict(count=0), EINVAL), (dict(beams=65), ERANGE)):
        assert L.ufb_beam_select_workspace(*{**size, **over}.values()) == code, over
    assert L.ufb_beam_select_workspace(*{**size, "streams": 0}.values()) == 0
    assert call(fn, streams=0, logits=None, scores=None) == 0  # nothing to do, no CUDA call


def test_python_view_needs_cuda(ufb):
    with pytest.raises(ufb.UfbError):
        ufb.beam_select(torch.zeros(1, 2, 8), torch.zeros(1, 2), 2)
    with pytest.raises(ufb.UfbError):
        ufb.beam_select([[[0.0]]], torch.zeros(1, 1), 1)
