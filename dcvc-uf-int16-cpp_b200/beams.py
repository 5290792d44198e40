"""A search over sequences: the best continuations of each stream's beams.

With KVCache.reorder (the cache's streams follow the choice) and KVCache.attend
over groups (the beams' common pages are read once) this makes a step of a beam
search that never waits for the host.  The arithmetic is in libufb200.so (C ABI in
include/uf_b200.h, which states the formulas).
"""
from __future__ import annotations

import ctypes as C

import torch

from . import UfbError, _check, library
from .attention import _DTYPES, _launch


_rooms = {}   # bytes of scratch by device and sizes


def _entry():
    L = library()
    fn = L.ufb_beam_select
    if fn.argtypes is None:
        vp, ci, i64 = C.c_void_p, C.c_int, C.c_int64
        fn.argtypes = [vp, ci, i64, i64, vp, vp, ci, ci, ci, ci, ci, vp, vp, vp, vp, i64, vp]
        L.ufb_beam_select_workspace.restype = i64
        L.ufb_beam_select_workspace.argtypes = [ci, ci, ci, ci, ci]
    return fn


def beam_select(logits, scores, count, finished=None, pad=0):
    """The best ``count`` continuations of every stream.

    ``logits`` [streams, beams, vocab] (float32, float16 or bfloat16), ``scores``
    [streams, beams] float32: the beams' summed log probabilities, -inf for places
    without a beam (at the first step one beam is enough).  A continuation's score is
    its beam's plus its token's log probability.  Beams marked in ``finished`` (bool,
    as scores) go on with ``pad`` at an unchanged score.  Returns (scores float32,
    parents int32, tokens int32), each [streams, count], best first; equal scores by
    the lower beam, then the larger logit, then the lower token.  Where a stream has
    fewer continuations the rest have score -inf, parent min(place, beams - 1) and
    token 0.  Up to 64 beams and 64 continuations.  No gradient."""
    if not isinstance(logits, torch.Tensor) or not logits.is_cuda or logits.dtype not in _DTYPES or logits.dim() != 3:
        raise UfbError(-1, "logits: CUDA tensor [streams, beams, vocab] of float32, float16 or bfloat16 required")
    streams, beams, vocab = logits.shape
    device = logits.device
    if not (isinstance(scores, torch.Tensor) and scores.device == device and scores.dtype == torch.float32 and
            scores.shape == (streams, beams)):
        raise UfbError(-1, f"scores: float32 tensor {[streams, beams]} on {device} required")
    if finished is not None and not (isinstance(finished, torch.Tensor) and finished.device == device and
                                     finished.dtype == torch.bool and finished.shape == (streams, beams)):
        raise UfbError(-1, f"finished: bool tensor {[streams, beams]} on {device} required")
    if count >> 31 or pad >> 31:
        raise UfbError(-1, "count and pad must be 32-bit numbers that are not negative")
    ss, bs, es = logits.stride()
    if es != 1 and vocab > 1:
        logits = logits.contiguous()
        ss, bs, es = logits.stride()
    if not scores.is_contiguous():
        scores = scores.contiguous()
    if finished is not None and not finished.is_contiguous():
        finished = finished.contiguous()
    fn = _entry()
    dtype = _DTYPES[logits.dtype]
    key = (device.index, dtype, streams, beams, vocab, count)
    room = _rooms.get(key)
    if room is None:
        with torch.cuda.device(device):
            room = library().ufb_beam_select_workspace(dtype, streams, beams, vocab, count)
        if room < 0:
            _check(room)
        _rooms[key] = room
    out = torch.empty((3, streams, count), dtype=torch.int32, device=device)
    work = torch.empty(room, dtype=torch.uint8, device=device)
    at, step = out.data_ptr(), streams * count * 4
    _launch(device, fn, logits.data_ptr(), dtype, ss, bs, scores.data_ptr(),
            None if finished is None else finished.data_ptr(), streams, beams, vocab, count, pad, at, at + step,
            at + 2 * step, work.data_ptr(), room)
    best, parents, tokens = out.unbind(0)
    return best.view(torch.float32), parents, tokens
