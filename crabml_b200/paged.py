"""Python handles on include/crabml_paged.h: the plan of a step over several sequences, a layer's cache in pages of 16 or 8 bits, the append and the attention.

    plan = PagePlan(dev, page_size=64, n_pages=n, table=pages_of_each_sequence, pos0=lengths, counts=new_tokens, n_slots=max_sequences)
    for layer in layers:                                          # rows of qkv: the new tokens, sequence after sequence
        q = append(plan, layer.cache, qkv, 0, qkv, H * d, qkv, (H + G) * d, H, freq=freq)
        y = attention(plan, layer.cache, q, H, d ** -0.5)

Results are queued on the device's stream: a library that is handed one (torch.as_tensor(y)) has to be ordered with it, see CudaTensor.__cuda_array_interface__.
"""
from __future__ import annotations

import ctypes as C
import operator
import struct

import numpy as np

from . import capi
from .capi import TensorError
from .tensor import CudaTensor, TensorStrider, _Buf


def _whole(what, a, kind):
    """an array of whole numbers that `kind` can hold, or a refusal: none is cut off or wrapped on its way"""
    a = np.asarray(a)
    if a.size and (a.dtype.kind not in "iu" or int(a.min()) < np.iinfo(kind).min or int(a.max()) > np.iinfo(kind).max):
        raise TensorError(f"page_plan: {what} are not whole numbers of {np.dtype(kind).itemsize * 8} bits")
    return np.ascontiguousarray(a, kind)


def _number(call, what, x, bits=32):
    """a whole number that the C call's argument can hold, or a refusal"""
    try:
        n = int(x) if isinstance(x, float) and x.is_integer() else operator.index(x)
    except TypeError:
        raise TensorError(f"{call}: {what} is {x!r}, not a whole number") from None
    if not -(1 << bits - 1) <= n < 1 << bits - 1:
        raise TensorError(f"{call}: {what} is {n}, beyond {bits} bits")
    return n


_TWO, _SIX = struct.Struct("=2i").pack, struct.Struct("=6i").pack      # one look at all of a call's numbers: it is made for every layer of a token


class PagePlan:
    """What the sequences of a step have in the cache (pos0), bring along (counts) and own (table: rows of page numbers, an array or lists of any lengths; slots:
    their open blocks, sequence i slot i where it is None).  Checked once; every layer's append and attention take it.

    A position below what a sequence has had takes it back (rejected drafts): to the start of any block, or, with 8-bit pages, to a token of the block that its next token
    falls into or of the one before, counted from the furthest it has reached; include/crabml_paged.h has the rule."""

    def __init__(self, device, page_size, n_pages, table, pos0, counts, n_slots=0, slots=None):
        self.device, self.handle = device, None
        counts, pos0 = _whole("counts", counts, np.int32).reshape(-1), _whole("positions", pos0, np.int64).reshape(-1)
        n = len(counts)
        if not isinstance(table, np.ndarray):
            rows, width = [list(r) for r in table], max([len(r) for r in table], default=0)
            table = np.full((len(rows), width), -1, np.int32)       # a page that is needed and was not given is refused
            for i, r in enumerate(rows):
                table[i, :len(r)] = _whole("page numbers", r, np.int32)
        if len(pos0) != n or table.ndim != 2 or len(table) != n or (slots is not None and len(slots) != n):
            raise TensorError(f"page_plan: {n} counts, {len(pos0)} positions, table {table.shape}" + ("" if slots is None else f", {len(slots)} slots"))
        table, slots = _whole("page numbers", table, np.int32), None if slots is None else _whole("slots", slots, np.int32).reshape(-1)
        d = capi.cc_page_plan_desc(n, _number("page_plan", "page_size", page_size), table.shape[1], _number("page_plan", "n_pages", n_pages, 64),
                                   _number("page_plan", "n_slots", n_slots, 64), *(None if a is None else a.ctypes.data for a in (pos0, counts, table, slots)))
        h = C.c_void_p()
        device.check(device.lib.cc_page_plan_create(device.handle, C.byref(d), C.byref(h)))
        self.handle = h
        self.tokens = int(device.lib.cc_page_plan_tokens(h))

    def __del__(self):
        try:
            if self.handle and self.device.handle:
                self.device.lib.cc_page_plan_release(self.handle)
        except Exception:
            pass


class PagedCache:
    """One layer's pages: k, v [pages, heads, page size, size] in F16, or in I8 with factors [pages, heads] and open blocks [2 * slots, heads, page size, size]"""

    def __init__(self, k, v, k_scale=None, v_scale=None, k_open=None, v_open=None):
        self._tensors = {"k": k, "v": v, "k_scale": k_scale, "v_scale": v_scale, "k_open": k_open, "v_open": v_open}
        self._c = capi.cc_paged_cache(**{n: t._view() for n, t in self._tensors.items() if t is not None})

    k = property(lambda self: self._tensors["k"])
    v = property(lambda self: self._tensors["v"])
    k_scale = property(lambda self: self._tensors["k_scale"])
    v_scale = property(lambda self: self._tensors["v_scale"])
    k_open = property(lambda self: self._tensors["k_open"])
    v_open = property(lambda self: self._tensors["v_open"])

    @classmethod
    def alloc(cls, device, n_pages, n_kv, page_size, dk, dv=None, dtype=capi.I8, n_slots=0):
        dv = dk if dv is None else dv
        t = [CudaTensor.alloc([n_pages, n_kv, page_size, d], dtype, device) for d in (dk, dv)]
        if dtype == capi.I8:
            t += [CudaTensor.alloc([n_pages, n_kv], capi.F32, device) for _ in range(2)]
            t += [CudaTensor.alloc([2 * n_slots, n_kv, page_size, d], capi.F16, device) for d in (dk, dv)]
        return cls(*t)


def _v(t):
    return C.byref(t._view()) if t is not None else None


def append(plan, cache, q_src, q_col0, k_src, k_col0, v_src, v_col0, n_heads=0, freq=None, pairing=capi.ROPE_NEIGHBOURS, offset=0, mag=1.0):
    """keys and values of the plan's tokens, turned by their positions, into the pages -> the turned queries [T, n_heads * dk] (q_src None: None)"""
    dev, h = plan.device, C.c_void_p()
    try:
        _SIX(q_col0, k_col0, v_col0, n_heads, pairing, offset)
    except struct.error:
        q_col0, k_col0, v_col0, n_heads, pairing, offset = (_number("paged_append", what, x) for what, x in (
            ("q_col0", q_col0), ("k_col0", k_col0), ("v_col0", v_col0), ("n_heads", n_heads), ("pairing", pairing), ("offset", offset)))
    dev.check(dev.lib.cc_paged_append(dev.handle, plan.handle, C.byref(cache._c), _v(q_src), q_col0, _v(k_src), k_col0, _v(v_src), v_col0, n_heads, _v(freq), pairing, offset,
                                      float(mag), C.byref(h)))
    return None if q_src is None else CudaTensor(_Buf(dev, h), TensorStrider([plan.tokens, n_heads * cache.k.shape()[3]]), dev)


def attention(plan, cache, q, n_heads, scale, window=0, softcap=0.0, sink=None):
    """-> [T, n_heads * dv]"""
    dev, h = plan.device, C.c_void_p()
    try:
        _TWO(n_heads, window)
    except struct.error:
        n_heads, window = _number("paged_attention", "n_heads", n_heads), _number("paged_attention", "window", window)
    dev.check(dev.lib.cc_paged_attention(dev.handle, plan.handle, C.byref(cache._c), _v(q), n_heads, float(scale), window, float(softcap), _v(sink), C.byref(h)))
    return CudaTensor(_Buf(dev, h), TensorStrider([plan.tokens, n_heads * cache.v.shape()[3]]), dev)
