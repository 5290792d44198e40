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

import torch

from . import UfbError, _check, _stream, library

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_LAYOUTS = {"half": 0, "interleaved": 1}


class _Heads(C.Structure):
    _fields_ = [("data", C.c_void_p), ("token_stride", C.c_int64), ("head_stride", C.c_int64), ("heads", C.c_int32)]


class _Cache(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("kv", "scale", "table", "lengths", "refs", "work")] + [
        (n, C.c_int32) for n in ("layers", "pages", "heads", "page_tokens", "head_dim", "slots", "table_width")]


def _lib():
    L = library()
    if getattr(L, "_attention_ready", False):
        return L
    vp, ci, i64 = C.c_void_p, C.c_int, C.c_int64
    cache, heads = C.POINTER(_Cache), C.POINTER(_Heads)
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
    L.ufb_kv_attend.argtypes = [cache, ci, vp, vp, ci, ci, i64, ci, heads, heads, vp, ci, ci, ci, C.c_float, vp, i64, vp]
    L._attention_ready = True
    return L


def _device(device) -> torch.device:
    d = torch.device(device)
    if d.type != "cuda":
        raise UfbError(-1, "a CUDA device is required")
    return torch.device("cuda", torch.cuda.current_device()) if d.index is None else d


def _head_tensor(t, device, what: str, dtypes=_DTYPES):
    """[tokens, heads, dim] on the device, rows of 16-byte multiples (copied if not)."""
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.device == device and t.dtype in dtypes and t.dim() == 3):
        names = ", ".join(str(d).replace("torch.", "") for d in dtypes)
        raise UfbError(-1, f"{what}: [tokens, heads, head_dim] tensor of {names} on {device} required")
    lanes = 16 // t.element_size()
    tokens, heads, dim = t.shape
    # a stride over one element or none is free: any value does
    ts = t.stride(0) if tokens > 1 else heads * dim
    hs = t.stride(1) if heads > 1 else dim
    if t.stride(2) != 1 or ts % lanes or hs % lanes or t.data_ptr() % 16 or (heads > 1 and hs < dim) or \
            (tokens > 1 and ts < dim):
        t = t.contiguous() if not t.is_contiguous() else t.clone()
        ts, hs = heads * dim, dim
    return t, _Heads(t.data_ptr(), ts, hs, heads)


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

    def apply(self, positions, q, k=None, inverse=False):
        """Turn q (and k in the same launch) by the tokens' positions
        ([tokens, axes] int32); inverse turns back, which is the gradient with
        respect to the input.  Returns new tensors: q, or (q, k)."""
        axes = len(self.pairs)
        if not (isinstance(positions, torch.Tensor) and positions.device == self.device and
                positions.dtype == torch.int32 and positions.dim() == 2 and positions.shape[1] == axes):
            raise UfbError(-1, f"positions: int32 tensor [tokens, {axes}] on {self.device} required")
        positions = positions.contiguous()
        xs = [q] if k is None else [q, k]
        ins, outs, keep = [], [], []
        for x in xs:
            x, h = _head_tensor(x, self.device, "rotary input")
            if x.shape[0] != positions.shape[0] or x.shape[2] != xs[0].shape[2] or x.dtype != xs[0].dtype:
                raise UfbError(-1, "rotary inputs and positions differ in tokens, head_dim or dtype")
            out = torch.empty(x.shape, dtype=x.dtype, device=self.device)
            keep.append((x, out))
            ins.append(h)
            outs.append(_Heads(out.data_ptr(), x.shape[1] * x.shape[2], x.shape[2], x.shape[1]))
        if positions.shape[0] and min(x.shape[1] for x in xs) > 0:
            n = len(xs)
            with torch.cuda.device(self.device):
                _check(_lib().ufb_rotary(self.table.data_ptr(), axes, self._pairs, self._extents,
                                         _LAYOUTS[self.layout], int(bool(inverse)), positions.data_ptr(),
                                         positions.shape[0], xs[0].shape[2], _DTYPES[xs[0].dtype], n,
                                         (_Heads * n)(*ins), (_Heads * n)(*outs), _stream(self.table)))
        return keep[0][1] if k is None else (keep[0][1], keep[1][1])


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


class KVCache:
    """Keys and values of many streams and layers in 8 bits, in pages of
    ``page_tokens`` tokens with one scale for each page, head and side (key or
    value).  ``slots`` streams hold up to ``table_width`` pages each.

    The state is ordinary tensors on the device -- ``kv`` [layers, pages, 2,
    heads, page_tokens, head_dim] int8, ``scale`` [layers, pages, 2, heads],
    ``table`` [slots, table_width] (-1: no page), ``lengths`` [slots], ``refs``
    [pages] -- and no call waits for it on the host.  Calls on one cache belong
    on one stream at a time (or are ordered by events), like writes to any tensor.

        plan = cache.plan(slots, counts)      # who brings how many tokens
        cache.extend(plan)                    # pages for them, once a step
        cache.append(layer, plan, k, v)       # in every layer
        out = cache.attend(layer, plan, q, window=..., sinks=...)
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
        n = _lib().ufb_kv_work_ints(self.pages, self.slots)
        if n < 0:
            _check(int(n))
        self._work = torch.zeros(n, dtype=torch.int32, device=d)
        self._struct = _Cache(*[t.data_ptr() for t in (self.kv, self.scale, self.table, self.lengths, self.refs,
                                                       self._work)],
                              self.layers, self.pages, self.heads, self.page_tokens, self.head_dim, self.slots,
                              self.table_width)
        self._workspaces = {}

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

    def _call(self, name, *args):
        with torch.cuda.device(self.device):
            _check(getattr(_lib(), name)(C.byref(self._struct), *args, _stream(self.kv)))

    def extend(self, plan):
        """Grow the plan's streams by its counts and give them the pages for it."""
        self._own(plan)
        self._call("ufb_kv_extend", plan.slots.data_ptr(), plan.offsets.data_ptr(), plan.n)

    def release(self, plan):
        """Drop the pages of the plan's streams; their lengths become 0."""
        self._own(plan)
        self._call("ufb_kv_release", plan.slots.data_ptr(), plan.n)

    def trim(self, plan, window, sinks=0):
        """Drop the pages that no later query of the plan's streams sees."""
        self._own(plan)
        self._call("ufb_kv_trim", plan.slots.data_ptr(), plan.n, int(window), int(sinks))

    def fork(self, plan):
        """Make the plan's destinations branches of its sources."""
        self._own(plan, KVForkPlan)
        self._call("ufb_kv_fork", plan.src.data_ptr(), plan.dst.data_ptr(), plan.n)

    def compact(self):
        """Move the live pages to the lowest ids."""
        self._call("ufb_kv_compact")

    # -- contents

    def append(self, layer, plan, k, v):
        """Store k and v [tokens, heads, head_dim] as the newest tokens of the plan's streams."""
        self._own(plan)
        shape = (plan.tokens, self.heads, self.head_dim)
        k, kh = _head_tensor(k, self.device, "keys")
        v, vh = _head_tensor(v, self.device, "values")
        if k.shape != shape or v.shape != shape or k.dtype != v.dtype:
            raise UfbError(-1, f"keys and values must be {list(shape)} of one dtype")
        self._call("ufb_kv_append", int(layer), plan.slots.data_ptr(), plan.offsets.data_ptr(), plan.n, plan.max_new,
                   plan.tokens, _DTYPES[k.dtype], C.byref(kh), C.byref(vh))

    def read(self, layer, pages, dtype=torch.float32):
        """The values of listed pages (int32 tensor): [n, 2, heads, page_tokens, head_dim]."""
        if not (isinstance(pages, torch.Tensor) and pages.device == self.device and pages.dtype == torch.int32 and
                pages.dim() == 1):
            raise UfbError(-1, f"pages: int32 list on {self.device} required")
        if dtype not in _DTYPES:
            raise UfbError(-1, "unsupported dtype")
        pages = pages.contiguous()
        out = torch.empty((pages.numel(), 2, self.heads, self.page_tokens, self.head_dim), dtype=dtype,
                          device=self.device)
        self._call("ufb_kv_read", int(layer), pages.data_ptr(), pages.numel(), _DTYPES[dtype], out.data_ptr())
        return out

    def _workspace(self):
        # zeroed once and left zeroed by every call; streams may overlap, so each has its own
        key = torch.cuda.current_stream(self.device).cuda_stream
        w = self._workspaces.get(key)
        if w is None:
            with torch.cuda.device(self.device):
                n = _lib().ufb_kv_attend_workspace()
            if n < 0:
                _check(int(n))
            w = self._workspaces[key] = torch.zeros(n, dtype=torch.uint8, device=self.device)
        return w

    def attend(self, layer, plan, q, window=0, sinks=0, causal=True, scale=None, lse=False):
        """Attention of the plan's newest tokens (q [tokens, query heads, head_dim],
        float16 or bfloat16) over their streams.  A query at position a sees key
        j when j <= a (all keys when not causal) and, with a window, j > a -
        window or j < sinks.  scale defaults to head_dim ** -0.5.  A query that
        sees nothing gives zeros.  Returns out, or (out, lse [tokens, query
        heads] float32)."""
        self._own(plan)
        q, qh = _head_tensor(q, self.device, "queries", (torch.float16, torch.bfloat16))
        if q.shape[0] != plan.tokens or q.shape[2] != self.head_dim or q.shape[1] == 0 or q.shape[1] % self.heads:
            raise UfbError(-1, f"queries must be [{plan.tokens}, a multiple of {self.heads}, {self.head_dim}]")
        out = torch.empty(q.shape, dtype=q.dtype, device=self.device)
        oh = _Heads(out.data_ptr(), q.shape[1] * q.shape[2], q.shape[2], q.shape[1])
        l = torch.empty(q.shape[:2], dtype=torch.float32, device=self.device) if lse else None
        w = self._workspace()
        self._call("ufb_kv_attend", int(layer), plan.slots.data_ptr(), plan.offsets.data_ptr(), plan.n, plan.max_new,
                   plan.tokens, _DTYPES[q.dtype], C.byref(qh), C.byref(oh), None if l is None else l.data_ptr(),
                   int(window), int(sinks), int(bool(causal)),
                   float(self.head_dim ** -0.5 if scale is None else scale), w.data_ptr(), w.numel())
        return (out, l) if lse else out
