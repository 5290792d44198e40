"""Attention over latent tokens: rotary positions with several axes, a paged
cache of keys and values held in 8 bits, and attention over it.

Like the other operators of this package these take CUDA tensors, allocate
their results and launch on the current torch stream; the arithmetic is in
libufb200.so (C ABI in include/uf_b200.h, which states the formulas).  What only
the device can see (a position outside its axis, too few free pages) is reported
by ``device_status``.
"""
from __future__ import annotations

import ctypes as C
import struct

import torch

from . import UfbError, _check, library

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_QUERY_DTYPES = {torch.float16: 1, torch.bfloat16: 2}
_LAYOUTS = {"half": 0, "interleaved": 1}
_ATTEND_ZERO = 1024  # UFB_KV_ATTEND_ZERO


# ufb_heads (data, token stride, head stride, heads), one or two of them
_heads = struct.Struct("@Pqqi4x").pack
_heads2 = struct.Struct("@Pqqi4xPqqi4x").pack


class _Cache(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("kv", "scale", "table", "lengths", "refs", "work")] + [
        (n, C.c_int32) for n in ("layers", "pages", "heads", "page_tokens", "head_dim", "slots", "table_width")]


def _lib():
    L = library()
    if getattr(L, "_attention_ready", False):
        return L
    vp, ci, i64 = C.c_void_p, C.c_int, C.c_int64
    cache = heads = vp  # addresses; ufb_heads as packed bytes
    L.ufb_rotary_table.restype = i64
    L.ufb_rotary_table.argtypes = [ci, vp, vp, vp, vp]
    L.ufb_rotary.argtypes = [vp, ci, vp, vp, ci, ci, vp, i64, ci, ci, ci, heads, heads, vp]
    L.ufb_kv_work_ints.restype = i64
    L.ufb_kv_work_ints.argtypes = [C.c_int32, C.c_int32]
    L.ufb_kv_extend.argtypes = [cache, vp, vp, ci, vp]
    L.ufb_kv_release.argtypes = [cache, vp, ci, vp]
    L.ufb_kv_fork.argtypes = [cache, vp, vp, ci, vp]
    L.ufb_kv_trim.argtypes = [cache, vp, ci, ci, ci, vp]
    L.ufb_kv_compact.argtypes = [cache, vp]
    L.ufb_kv_append.argtypes = [cache, ci, vp, vp, ci, ci, i64, ci, heads, heads, vp]
    L.ufb_kv_read.argtypes = [cache, ci, vp, i64, ci, vp, vp]
    L.ufb_kv_attend_workspace.restype = i64
    L.ufb_capture_id.restype = i64
    L.ufb_capture_id.argtypes = [vp]
    L.ufb_kv_attend.argtypes = [cache, ci, vp, vp, ci, ci, i64, ci, heads, heads, vp, ci, ci, ci, C.c_float, vp, i64, vp]
    L._attention_ready = True
    return L


def _device(device) -> torch.device:
    d = torch.device(device)
    if d.type != "cuda":
        raise UfbError(-1, "a CUDA device is required")
    return torch.device("cuda", torch.cuda.current_device()) if d.index is None else d


# A decoding step makes these calls for every layer and its kernels take a few
# microseconds, so the wrappers below keep to few and cheap host operations.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_capturing = getattr(torch._C, "_cuda_isCurrentStreamCapturing", None) or torch.cuda.is_current_stream_capturing


def _launch(device, fn, *args):
    """fn(*args, current stream of the device), with that device current."""
    index = device.index
    if _current_device() == index:
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _raw_stream(index))
    if rc:
        _check(rc)


def _check_ints(layer, window=0, sinks=0):
    # ctypes would cut larger numbers to 32 bits
    if layer >> 31 or window >> 31 or sinks >> 31:
        raise UfbError(-1, "layer, window and sinks must be 32-bit numbers that are not negative")


def _refuse_heads(device, what, dtypes):
    names = ", ".join(str(d).replace("torch.", "") for d in dtypes)
    raise UfbError(-1, f"{what}: [tokens, heads, head_dim] tensor of {names} on {device} required")


def _head_tensor(t, device, what: str, dtypes=_DTYPES):
    """[tokens, heads, dim] on the device, rows of 16-byte multiples (copied if
    not): the tensor, its sizes, dtype code, address and strides."""
    if not isinstance(t, torch.Tensor) or t.device != device:
        _refuse_heads(device, what, dtypes)
    shape, code = t.shape, dtypes.get(t.dtype)
    if code is None or len(shape) != 3:
        _refuse_heads(device, what, dtypes)
    tokens, heads, dim = shape
    ts, hs, es = t.stride()
    lanes = 4 if code == 0 else 8
    # a stride over one element or none is free: any value does
    if tokens <= 1:
        ts = heads * dim
    if heads <= 1:
        hs = dim
    at = t.data_ptr()
    if es != 1 or ts % lanes or hs % lanes or at % 16 or (heads > 1 and hs < dim) or (tokens > 1 and ts < dim):
        t = t.clone(memory_format=torch.contiguous_format)
        ts, hs, at = heads * dim, dim, t.data_ptr()
    return t, tokens, heads, dim, code, at, ts, hs


class _Turn(torch.autograd.Function):
    """Rotary.apply of inputs that require a gradient: theirs is the inverse turn."""

    @staticmethod
    def forward(ctx, rotary, positions, inverse, q, k):
        ctx.rotary, ctx.inverse = rotary, inverse
        ctx.save_for_backward(positions)
        ctx.set_materialize_grads(False)
        return rotary._turn(positions, q, k, inverse)

    @staticmethod
    def backward(ctx, *grads):
        (positions,) = ctx.saved_tensors
        wanted = [g if need else None for g, need in zip(grads, ctx.needs_input_grad[3:])]
        given = [g for g in wanted if g is not None]
        if not given:
            return None, None, None, None, None
        turned = ctx.rotary.apply(positions, *given, inverse=not ctx.inverse)
        back = iter(turned if len(given) == 2 else (turned,))
        return (None, None, None, *(None if g is None else next(back) for g in (*wanted, None)[:2]))


class Rotary:
    """Rotary positions over several axes, for example (time, height, width).

    ``pairs[a]`` of a head's dimension pairs turn with the position on axis a,
    pair i by ``position * bases[a] ** (-i / pairs[a])``; positions lie in
    ``[0, extents[a])``.  Elements past ``2 * sum(pairs)`` are copied.  layout
    "half" pairs element j with j + sum(pairs), "interleaved" 2j with 2j + 1.
    The table of cosines and sines is computed once, in 64 bits, and kept on the
    device."""

    def __init__(self, pairs, extents, bases=10000.0, layout="half", device="cuda"):
        L = _lib()
        self.device = _device(device)
        pairs, extents = [int(p) for p in pairs], [int(e) for e in extents]
        bases = [float(bases)] * len(pairs) if isinstance(bases, (int, float)) else [float(b) for b in bases]
        if not 1 <= len(pairs) <= 4 or len(extents) != len(pairs) or len(bases) != len(pairs):
            raise UfbError(-1, "rotary positions have 1 to 4 axes, each with pairs, an extent and a base")
        if layout not in _LAYOUTS:
            raise UfbError(-1, "rotary layout must be 'half' or 'interleaved'")
        self.pairs, self.extents, self.bases, self.layout = pairs, extents, bases, layout
        self._pairs = (C.c_int32 * len(pairs))(*pairs)
        self._extents = (C.c_int32 * len(pairs))(*extents)
        b = (C.c_double * len(pairs))(*bases)
        n = L.ufb_rotary_table(len(pairs), self._pairs, self._extents, b, None)
        if n < 0:
            _check(int(n))
        host = torch.empty(n, dtype=torch.float32)
        L.ufb_rotary_table(len(pairs), self._pairs, self._extents, b, host.data_ptr())
        self.table = host.to(self.device)
        self._fn, self._table, self._layout = L.ufb_rotary, self.table.data_ptr(), _LAYOUTS[layout]
        self._axes, self._pairs_at, self._extents_at = len(pairs), C.addressof(self._pairs), C.addressof(self._extents)

    def apply(self, positions, q, k=None, inverse=False):
        """Turn q (and k in the same launch) by the tokens' positions
        ([tokens, axes] int32); inverse turns back, which is the gradient with
        respect to the input: results of inputs that require one carry it.
        Returns new tensors: q, or (q, k)."""
        if torch.is_grad_enabled() and (getattr(q, "requires_grad", False) or getattr(k, "requires_grad", False)):
            return _Turn.apply(self, positions, inverse, q, k)
        return self._turn(positions, q, k, inverse)

    def _turn(self, positions, q, k, inverse):
        if not (isinstance(positions, torch.Tensor) and positions.device == self.device and
                positions.dtype == torch.int32 and positions.dim() == 2 and positions.shape[1] == self._axes):
            raise UfbError(-1, f"positions: int32 tensor [tokens, {self._axes}] on {self.device} required")
        if not positions.is_contiguous():
            positions = positions.contiguous()
        tokens = positions.shape[0]
        device = self.device
        q, qt, qn, dim, code, qa, qts, qhs = _head_tensor(q, device, "rotary input")
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        if qt != tokens:
            raise UfbError(-1, "rotary inputs and positions differ in tokens")
        if k is None:
            n, most = 1, qn
            x, y = _heads(qa, qts, qhs, qn), _heads(out.data_ptr(), qn * dim, dim, qn)
        else:
            k, kt, kn, kdim, kcode, ka, kts, khs = _head_tensor(k, device, "rotary input")
            if kt != tokens or kdim != dim or kcode != code:
                raise UfbError(-1, "rotary inputs differ in tokens, head_dim or dtype")
            out2 = torch.empty_like(k, memory_format=torch.contiguous_format)
            n, most = 2, min(qn, kn)
            x = _heads2(qa, qts, qhs, qn, ka, kts, khs, kn)
            y = _heads2(out.data_ptr(), qn * dim, dim, qn, out2.data_ptr(), kn * dim, dim, kn)
        if tokens and most:
            _launch(device, self._fn, self._table, self._axes, self._pairs_at, self._extents_at, self._layout,
                    1 if inverse else 0, positions.data_ptr(), tokens, dim, code, n, x, y)
        return out if k is None else (out, out2)


class KVPlan:
    """Streams of one step and how many tokens each brings (KVCache.plan)."""

    def __init__(self, cache, slots, counts):
        slots, counts = [int(s) for s in slots], [int(c) for c in counts]
        if len(slots) != len(counts):
            raise UfbError(-1, "a plan needs one count for each slot")
        if len(set(slots)) != len(slots):
            raise UfbError(-1, "a slot may appear once in a plan")
        if any(s < 0 or s >= cache.slots for s in slots):
            raise UfbError(-1, "slot out of range")
        if any(c < 0 for c in counts):
            raise UfbError(-1, "token counts must not be negative")
        self.cache, self.n, self.tokens = cache, len(slots), sum(counts)
        if self.tokens > 2 ** 31 - 1:
            raise UfbError(-2, "too many tokens")
        self.max_new = max(counts, default=0)
        offsets = [0]
        for c in counts:
            offsets.append(offsets[-1] + c)
        ints = torch.tensor(slots + offsets, dtype=torch.int32).to(cache.device)
        self.slots, self.offsets = ints[:self.n], ints[self.n:]
        self._slots, self._offsets = self.slots.data_ptr(), self.offsets.data_ptr()


class KVForkPlan:
    """Branches src[i] -> dst[i] of one fork (KVCache.fork_plan)."""

    def __init__(self, cache, src, dst):
        src, dst = [int(s) for s in src], [int(d) for d in dst]
        if len(src) != len(dst):
            raise UfbError(-1, "fork needs one destination for each source")
        if any(s < 0 or s >= cache.slots for s in src + dst):
            raise UfbError(-1, "slot out of range")
        if len(set(dst)) != len(dst) or set(dst) & set(src):
            raise UfbError(-1, "fork destinations must differ from each other and from the sources")
        self.cache, self.n = cache, len(src)
        ints = torch.tensor(src + dst, dtype=torch.int32).to(cache.device)
        self.src, self.dst = ints[:self.n], ints[self.n:]
        self._src, self._dst = self.src.data_ptr(), self.dst.data_ptr()


class KVCache:
    """Keys and values of many streams and layers in 8 bits, in pages of
    ``page_tokens`` tokens with one scale for each page, head and side (key or
    value).  ``slots`` streams hold up to ``table_width`` pages each.

    The state is ordinary tensors on the device -- ``kv`` [layers, pages, 2,
    heads, page_tokens, head_dim] int8, ``scale`` [layers, pages, 2, heads],
    ``table`` [slots, table_width] (-1: no page), ``lengths`` [slots], ``refs``
    [pages] -- and no call waits for it on the host.  Calls on one cache belong
    on one stream at a time (or are ordered by events), like writes to any tensor.
    They are operators of inference: their results carry no gradient.

        plan = cache.plan(slots, counts)      # who brings how many tokens
        cache.extend(plan)                    # pages for them, once a step
        cache.append(layer, plan, k, v)       # in every layer
        out = cache.attend(layer, plan, q, window=..., sinks=...)

    When the pages do not suffice, extend changes nothing (status 31), and append
    and attend leave out the streams that were to grow (status 31 again, zeros for
    their queries) until an extend of theirs is granted, one of no tokens too.
    """

    def __init__(self, layers, pages, heads, head_dim, page_tokens=64, slots=1, table_width=None, device="cuda"):
        self.device = _device(device)
        self.layers, self.pages, self.heads, self.head_dim = int(layers), int(pages), int(heads), int(head_dim)
        self.page_tokens, self.slots = int(page_tokens), int(slots)
        self.table_width = int(pages if table_width is None else table_width)
        if self.page_tokens not in (16, 32, 64, 128):
            raise UfbError(-1, "page_tokens must be 16, 32, 64 or 128")
        if self.head_dim not in (64, 128):
            raise UfbError(-1, "head_dim must be 64 or 128")
        if min(self.layers, self.pages, self.heads, self.slots, self.table_width) <= 0:
            raise UfbError(-1, "empty cache")
        d = self.device
        self.kv = torch.zeros((self.layers, self.pages, 2, self.heads, self.page_tokens, self.head_dim),
                              dtype=torch.int8, device=d)
        self.scale = torch.zeros((self.layers, self.pages, 2, self.heads), dtype=torch.float32, device=d)
        self.table = torch.full((self.slots, self.table_width), -1, dtype=torch.int32, device=d)
        self.lengths = torch.zeros(self.slots, dtype=torch.int32, device=d)
        self.refs = torch.zeros(self.pages, dtype=torch.int32, device=d)
        L = self._L = _lib()
        n = L.ufb_kv_work_ints(self.pages, self.slots)
        if n < 0:
            _check(int(n))
        self._work = torch.zeros(n, dtype=torch.int32, device=d)
        self._struct = _Cache(*[t.data_ptr() for t in (self.kv, self.scale, self.table, self.lengths, self.refs,
                                                       self._work)],
                              self.layers, self.pages, self.heads, self.page_tokens, self.head_dim, self.slots,
                              self.table_width)
        self._ref = C.addressof(self._struct)
        self._default_scale = self.head_dim ** -0.5
        self._append, self._attend = L.ufb_kv_append, L.ufb_kv_attend
        self._workspaces, self._captures = {}, {}
        self._spare = self._new_workspace()

    # -- streams and their pages

    def plan(self, slots, counts):
        """The streams of a step and the tokens each brings; kept over layers and steps."""
        return KVPlan(self, slots, counts)

    def fork_plan(self, src, dst):
        """Branches src[i] -> dst[i]; kept over calls."""
        return KVForkPlan(self, src, dst)

    def _own(self, plan, kind=KVPlan):
        if not isinstance(plan, kind) or plan.cache is not self:
            raise UfbError(-1, f"a {kind.__name__} of this cache is required")
        return plan

    def extend(self, plan):
        """Grow the plan's streams by its counts and give them the pages for it."""
        self._own(plan)
        _launch(self.device, self._L.ufb_kv_extend, self._ref, plan._slots, plan._offsets, plan.n)

    def release(self, plan):
        """Drop the pages of the plan's streams; their lengths become 0."""
        self._own(plan)
        _launch(self.device, self._L.ufb_kv_release, self._ref, plan._slots, plan.n)

    def trim(self, plan, window, sinks=0):
        """Drop the pages that no later query of the plan's streams sees."""
        self._own(plan)
        _check_ints(0, window, sinks)
        _launch(self.device, self._L.ufb_kv_trim, self._ref, plan._slots, plan.n, int(window), int(sinks))

    def fork(self, plan):
        """Make the plan's destinations branches of its sources, whose tokens have
        been appended in every layer: full pages are shared from here on."""
        self._own(plan, KVForkPlan)
        _launch(self.device, self._L.ufb_kv_fork, self._ref, plan._src, plan._dst, plan.n)

    def compact(self):
        """Move the live pages to the lowest ids."""
        _launch(self.device, self._L.ufb_kv_compact, self._ref)

    # -- contents

    def append(self, layer, plan, k, v):
        """Store k and v [tokens, heads, head_dim] as the newest tokens of the plan's streams."""
        self._own(plan)
        _check_ints(layer)
        device = self.device
        k, kt, kn, kd, code, ka, kts, khs = _head_tensor(k, device, "keys")
        v, vt, vn, vd, vcode, va, vts, vhs = _head_tensor(v, device, "values")
        if not (kt == vt == plan.tokens and kn == vn == self.heads and kd == vd == self.head_dim and code == vcode):
            raise UfbError(-1, f"keys and values must be {[plan.tokens, self.heads, self.head_dim]} of one dtype")
        _launch(device, self._append, self._ref, layer, plan._slots, plan._offsets, plan.n, plan.max_new, kt, code,
                _heads(ka, kts, khs, kn), _heads(va, vts, vhs, vn))

    def read(self, layer, pages, dtype=torch.float32):
        """The values of listed pages (int32 tensor): [n, 2, heads, page_tokens, head_dim]."""
        if not (isinstance(pages, torch.Tensor) and pages.device == self.device and pages.dtype == torch.int32 and
                pages.dim() == 1):
            raise UfbError(-1, f"pages: int32 list on {self.device} required")
        if dtype not in _DTYPES:
            raise UfbError(-1, "unsupported dtype")
        _check_ints(layer)
        if not pages.is_contiguous():
            pages = pages.contiguous()
        n = pages.shape[0]
        out = torch.empty((n, 2, self.heads, self.page_tokens, self.head_dim), dtype=dtype, device=self.device)
        _launch(self.device, self._L.ufb_kv_read, self._ref, layer, pages.data_ptr(), n, _DTYPES[dtype],
                out.data_ptr())
        return out

    def _new_workspace(self):
        with torch.cuda.device(self.device):
            n = self._L.ufb_kv_attend_workspace()
        if n < 0:
            _check(int(n))
        t = torch.zeros(n, dtype=torch.uint8, device=self.device)
        return t.data_ptr(), n, t

    def _workspace(self):
        # zeroed once and left zeroed by every call; streams may overlap, so each has its own
        index = self.device.index
        key = _raw_stream(index)
        if _current_device() == index:
            capturing = _capturing()
        else:
            with torch.cuda.device(index):
                capturing = _capturing()
        w = self._workspaces.get(key)
        if w is None:
            if not capturing:
                w = self._new_workspace()
            elif self._spare is None:
                raise UfbError(-1, "this stream has no attention scratch yet: call attend on it once before capturing")
            else:
                # zeros made here would be zeroed by this graph's replays only, and
                # the stream's own calls may come first
                w, self._spare = self._spare, None
            self._workspaces[key] = w
        return self._captured(key) if capturing else w

    def _captured(self, key):
        # a graph may be replayed beside its stream's calls and other graphs of it, so
        # each capture has its own, from the graph's memory and zeroed by its replays;
        # kept here until the stream's next capture, so that nothing else of the graph gets it
        capture = self._L.ufb_capture_id(key)
        if capture < 0:
            _check(capture)
        held = self._captures.get(key)
        if held is None or held[0] != capture:
            t = torch.empty(self._workspaces[key][1], dtype=torch.uint8, device=self.device)
            t[:_ATTEND_ZERO].zero_()
            held = self._captures[key] = (capture, (t.data_ptr(), t.numel(), t))
        return held[1]

    def attend(self, layer, plan, q, window=0, sinks=0, causal=True, scale=None, lse=False):
        """Attention of the plan's newest tokens (q [tokens, query heads, head_dim],
        float16 or bfloat16) over their streams.  A query at position a sees key
        j when j <= a (all keys when not causal) and, with a window, j > a -
        window or j < sinks.  scale defaults to head_dim ** -0.5.  A query that
        sees nothing gives zeros.  Returns out, or (out, lse [tokens, query
        heads] float32).  Every CUDA stream has its own scratch, and so has every
        capture, in its graph's memory: graphs may be replayed beside each other
        and beside other calls.  One stream may capture without an earlier call
        on it; others call attend once before."""
        self._own(plan)
        _check_ints(layer, window, sinks)
        device = self.device
        q, tokens, heads, dim, code, qa, qts, qhs = _head_tensor(q, device, "queries", _QUERY_DTYPES)
        if tokens != plan.tokens or dim != self.head_dim or heads == 0 or heads % self.heads:
            raise UfbError(-1, f"queries must be [{plan.tokens}, a multiple of {self.heads}, {self.head_dim}]")
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        l = torch.empty((tokens, heads), dtype=torch.float32, device=device) if lse else None
        w = self._workspace()
        _launch(device, self._attend, self._ref, layer, plan._slots, plan._offsets, plan.n, plan.max_new, tokens, code,
                _heads(qa, qts, qhs, heads), _heads(out.data_ptr(), heads * dim, dim, heads),
                None if l is None else l.data_ptr(), window, sinks, 1 if causal else 0,
                self._default_scale if scale is None else scale, w[0], w[1])
        return (out, l) if lse else out
