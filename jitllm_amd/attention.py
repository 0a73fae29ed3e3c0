"""The key-value cache in pages and the attention that reads it: host mirror of the jl_kv_* calls.

What a decode step runs between the q|k|v projection and the output projection of
``jitllm_amd.projections``::

    tables = BlockTables(ctx, requests, blocksPerRequest, pages, pageTokens, maxRows)
    caches = [PagedKvCache(ctx, KvType.F16, pages, kvHeads, headDim, pageTokens) for _ in layers]
    rope = Rope.of_base(ctx, headDim, 500000.0)
    attention = PagedAttention(ctx, maxRows, heads, kvHeads, headDim)
    ...
    tables.plan(fresh)                                   # once a step
    for cache, layer in zip(caches, layers):             # in every layer
        projections.fusedQKV(xb, qkv, layer.wq, layer.wk, layer.wv, rows)
        cache.append(Rows(qkv, w, dim), Rows(qkv, w, dim + kv), tables.positions, tables.slots, rows, rope=rope,
                     q=Rows(qkv, w), heads=heads)
        attention.attend(cache, Rows(qkv, w), rows, tables.positions, tables.table, att, requests=requests,
                         rowRequests=tables.rowRequests)
        projections.projection(att, x, layer.wo, ...)

Every array lies on the device, so the calls of a step can be captured into a graph once and replayed while
the lengths grow.  The reference's own paged cache (J/backend/tornado/kernels/TransformerPagedKvKernels.java)
is planned on the host; these calls plan, write and read on the device.
"""
from __future__ import annotations

import ctypes as C
import enum
import math

import numpy as np

from . import _lib as L
from .runtime import Context, DeviceBuffer, HalfFloatArray


class KvType(enum.IntEnum):
    """What a cache keeps of an element (jl_kv_type)."""
    F16 = L.JL_KV_F16
    Q8_0 = L.JL_KV_Q8_0


class RopeStyle(enum.IntEnum):
    """Which elements of a head turn together: 2i and 2i + 1, or i and i + rotated / 2 (jl_rope_style)."""
    PAIRS = L.JL_ROPE_PAIRS
    HALVES = L.JL_ROPE_HALVES


class IntArray(DeviceBuffer):
    """int32 device array."""

    def __init__(self, ctx: Context, size: int):
        super().__init__(ctx, int(size) * 4)
        self.size = int(size)

    def set(self, values: np.ndarray) -> None:
        values = np.ascontiguousarray(values, dtype=np.int32).reshape(-1)
        if values.size != self.size:
            raise ValueError(f"{values.size} values for an IntArray of {self.size}")
        self.upload(values)

    def get(self) -> np.ndarray:
        return self.download(np.int32, self.size)


class Rows:
    """Rows of a device array that lie ``stride`` elements apart, the first ``offset`` elements in: the q, k
    or v part of the rows that a fused projection leaves side by side."""

    __slots__ = ("array", "stride", "offset")

    def __init__(self, array, stride: int, offset: int = 0):
        self.array, self.stride, self.offset = array, stride, offset


def _place(who: str, value, rows: int, width: int, itemsize: int = 0):
    """(address, stride) of ``rows`` rows of ``width`` elements; raises where they are not the array's, or its
    elements not of ``itemsize`` bytes (0: of any).  An array in place of Rows: its rows lie behind one another."""
    if value.__class__ is Rows:
        array, stride, offset = value.array, value.stride, value.offset
    else:
        array, stride, offset = value, width, 0
    size = array.size
    if stride < width or offset < 0 or (rows > 0 and offset + (rows - 1) * stride + width > size):
        raise ValueError(f"{who}: {rows} rows of {width} elements, {stride} apart from {offset} on, in an array of {size}")
    if itemsize == 0:
        itemsize = array.nbytes // max(size, 1)
    elif array.nbytes != itemsize * size:
        raise ValueError(f"{who}: an array of {size} elements in {array.nbytes} bytes, of {itemsize} each is taken")
    return (array.ptr.value or 0) + itemsize * offset, stride


def _ints(who: str, array, count: int) -> int:
    if array.nbytes < 4 * count:
        raise ValueError(f"{who}: {count} int32 values in an array of {array.nbytes} bytes")
    return array.ptr.value or 0


class Rope:
    """A rotation: ``rotated`` values of every head turn, pair i by position * frequencies[i] radians.

    ``frequencies`` is a device array of ``rotated / 2`` doubles, so that any scaling of them is the caller's;
    ``of_base`` makes the plain ones."""

    def __init__(self, ctx: Context, frequencies, rotated: int, style: RopeStyle = RopeStyle.PAIRS):
        if frequencies.nbytes < 4 * rotated:
            raise ValueError(f"{rotated // 2} frequencies in an array of {frequencies.nbytes} bytes")
        self.ctx, self.frequencies, self.rotated, self.style = ctx, frequencies, int(rotated), RopeStyle(style)
        self._args = (frequencies.ptr.value, self.rotated, int(self.style))

    @classmethod
    def of(cls, ctx: Context, frequencies, style: RopeStyle = RopeStyle.PAIRS) -> "Rope":
        values = np.ascontiguousarray(frequencies, dtype=np.float64).reshape(-1)
        memory = ctx.raw_buffer(values.nbytes)
        memory.upload(values)
        return cls(ctx, memory, 2 * values.size, style)

    @classmethod
    def of_base(cls, ctx: Context, rotated: int, base: float, style: RopeStyle = RopeStyle.PAIRS) -> "Rope":
        return cls.of(ctx, float(base) ** (-np.arange(0, rotated, 2, dtype=np.float64) / rotated), style)


_NO_ROPE = (None, 0, int(RopeStyle.PAIRS))


class PagedKvCache:
    """One layer's keys and values in pages (jl_kv_cache).  ``memory``: a device array that holds the pages
    and stays the caller's; without one the cache allocates them."""

    def __init__(self, ctx: Context, kvType: KvType, pages: int, kvHeads: int, headDim: int, pageTokens: int, memory=None):
        self.ctx, self._lib = ctx, ctx._lib
        self.type = KvType(kvType)
        self.pages, self.kvHeads, self.headDim, self.pageTokens = int(pages), int(kvHeads), int(headDim), int(pageTokens)
        self.memory = memory
        h = C.c_void_p()
        if memory is None:
            L.check(self._lib.jl_kv_cache_create(ctx.handle, self.type, pages, kvHeads, headDim, pageTokens, C.byref(h)))
        else:
            want = self.bytes_for(self.type, pages, kvHeads, headDim, pageTokens)
            if memory.nbytes < want:
                raise ValueError(f"{memory.nbytes} bytes for a cache of {want}")
            L.check(self._lib.jl_kv_cache_wrap(ctx.handle, memory.ptr, self.type, pages, kvHeads, headDim, pageTokens, C.byref(h)))
        self.handle = h

    @staticmethod
    def bytes_for(kvType: KvType, pages: int, kvHeads: int, headDim: int, pageTokens: int) -> int:
        return L.load().jl_kv_cache_bytes(int(kvType), pages, kvHeads, headDim, pageTokens)

    @property
    def nbytes(self) -> int:
        return self.bytes_for(self.type, self.pages, self.kvHeads, self.headDim, self.pageTokens)

    def free(self) -> None:
        if self.handle and self.ctx.handle:
            L.check(self._lib.jl_kv_cache_free(self.handle))
        self.handle = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass

    def append(self, k, v, positions, slots, rows: int, rope: Rope | None = None, q=None, qOut=None, heads: int = 0,
               qNorm=None, kNorm=None, eps: float = 0.0) -> None:
        """Turns q and k (normalised first where ``qNorm`` / ``kNorm`` are given) and writes k and v to
        ``slots`` (jl_kv_append).  ``q`` is turned into ``qOut``, or in place without one."""
        width = self.kvHeads * self.headDim
        k, ldk = _place("k", k, rows, width, 4)
        v, ldv = _place("v", v, rows, width, 4)
        if q is None:
            q = ldq = out = ldOut = heads = 0
        else:
            width = heads * self.headDim
            out, ldOut = _place("qOut", q if qOut is None else qOut, rows, width, 4)
            q, ldq = _place("q", q, rows, width, 4)
        for name, norm in (("qNorm", qNorm), ("kNorm", kNorm)) if qNorm is not None or kNorm is not None else ():
            if norm is not None and not norm.size == self.headDim == norm.nbytes // 4:
                raise ValueError(f"{name} has {norm.size} weights in {norm.nbytes} bytes, a head {self.headDim} values")
        frequencies, rotated, style = rope._args if rope is not None else _NO_ROPE
        status = self._lib.jl_kv_append(
            self.ctx.handle, self.handle, q, heads, ldq, k, ldk, v, ldv, out, ldOut, _ints("positions", positions, rows),
            _ints("slots", slots, rows), rows, frequencies, rotated, style, qNorm.ptr if qNorm is not None else None,
            kNorm.ptr if kNorm is not None else None, eps)
        if status:
            L.check(status)

    def read(self, slots, rows: int, k=None, v=None) -> None:
        """Decodes the k and v at ``slots`` into rows of kvHeads x headDim values, binary16 or fp32 by the
        arrays' elements (jl_kv_read)."""
        need = rows * self.kvHeads * self.headDim
        half = None
        for name, array in (("k", k), ("v", v)):
            if array is None:
                continue
            if array.size < need:
                raise ValueError(f"{name} has {array.size} elements, {need} are read")
            size = array.nbytes // max(1, array.size)
            if half is not None and half != (size == 2):
                raise ValueError("k and v are read into elements of one type")
            half = size == 2
        L.check(self._lib.jl_kv_read(self.ctx.handle, self.handle, _ints("slots", slots, rows), rows,
                                     k.ptr if k is not None else None, v.ptr if v is not None else None, int(bool(half))))


class BlockTables:
    """The pages of a batch's requests, and the rows of a step (jl_kv_plan).

    Device arrays: ``table`` [requests x blocksPerRequest], ``lengths`` [requests], ``rowStarts``
    [requests + 1], ``slots``, ``positions`` and ``rowRequests`` [maxRows], and the free pages, a ring
    ``pageRing`` [pages] with ``freePages`` = {head, count}.  ``arrays`` gives some or all of them; those not
    given are allocated, and start with no tokens and every page free."""

    def __init__(self, ctx: Context, requests: int, blocksPerRequest: int, pages: int, pageTokens: int, maxRows: int, arrays=None):
        self.ctx, self._lib = ctx, ctx._lib
        self.requests, self.blocksPerRequest, self.pages = int(requests), int(blocksPerRequest), int(pages)
        self.pageTokens, self.maxRows = int(pageTokens), int(maxRows)
        sizes = {"table": requests * blocksPerRequest, "lengths": requests, "rowStarts": requests + 1, "slots": maxRows,
                 "positions": maxRows, "rowRequests": maxRows, "pageRing": pages, "freePages": 2}
        start = {"table": lambda n: np.full(n, -1), "pageRing": np.arange, "freePages": lambda n: np.array([0, pages])}
        given = dict(arrays or {})
        for name, size in sizes.items():
            array = given.pop(name, None)
            if array is None:
                array = IntArray(ctx, size)
                if size:
                    array.set(start.get(name, np.zeros)(size))
            elif array.nbytes < 4 * size:
                raise ValueError(f"{name}: {array.nbytes} bytes for {size} int32 values")
            setattr(self, name, array)
        if given:
            raise ValueError(f"no such arrays: {', '.join(sorted(given))}")

    def plan(self, fresh, past=None, freeIn=None) -> None:
        """One step: ``fresh`` [requests] new tokens of each request (negative: it has ended).  Lengths and
        free pages move on in place; ``past`` / ``freeIn`` give others to start from."""
        n = self.requests
        status = self._lib.jl_kv_plan(
            self.ctx.handle, _ints("past", self.lengths if past is None else past, n), _ints("fresh", fresh, n), n, self.pages, self.pageTokens,
            self.pageRing.ptr, _ints("freeIn", self.freePages if freeIn is None else freeIn, 2), self.freePages.ptr, self.table.ptr,
            self.blocksPerRequest, self.lengths.ptr, self.rowStarts.ptr, self.slots.ptr, self.positions.ptr, self.rowRequests.ptr, self.maxRows)
        if status:
            L.check(status)


class PagedAttention:
    """Attention of one new token a row over paged caches of one shape, with the workspace it joins in
    (jl_kv_attention).  One object for every layer; calls that may run at the same time need one each.
    ``maxRows`` is the caller's own note: the workspace is the same for any number of rows, and no call is
    held to it (jl_kv_attention takes up to 65535)."""

    def __init__(self, ctx: Context, maxRows: int, heads: int, kvHeads: int, headDim: int):
        self.ctx, self._lib = ctx, ctx._lib
        self.maxRows, self.heads, self.kvHeads, self.headDim = int(maxRows), int(heads), int(kvHeads), int(headDim)
        self.width, self.scale = self.heads * self.headDim, 1 / math.sqrt(self.headDim) if headDim > 0 else 0.0
        nbytes = self._lib.jl_kv_attention_workspace_bytes(heads, kvHeads, headDim)
        if not nbytes:
            raise ValueError(f"{heads} query heads over {kvHeads} of k and v, {headDim} values each")
        self.workspace = ctx.raw_buffer(nbytes)
        L.check(self._lib.jl_kv_attention_workspace_init(ctx.handle, self.workspace.ptr, nbytes))

    def attend(self, cache: PagedKvCache, q, rows: int, positions, table, out, requests: int, rowRequests=None,
               scale: float | None = None, window: int = 0, blocksPerRequest: int | None = None) -> None:
        """``out[row] = softmax(scale * q[row] . k) v`` over the tokens up to ``positions[row]`` (the last
        ``window`` of them where that is positive) of request ``rowRequests[row]``, or of request ``row``.
        ``scale``: 1 / sqrt(headDim) unless given.  ``out``: a FloatArray or a HalfFloatArray.  ``requests`` are
        all of the table's rows, unless ``blocksPerRequest`` says how many entries a row has."""
        if cache.kvHeads != self.kvHeads or cache.headDim != self.headDim:
            raise ValueError(f"a cache of {cache.kvHeads} heads of {cache.headDim}, attention over {self.kvHeads} of {self.headDim}")
        width = self.width
        array = out.array if out.__class__ is Rows else out
        half = array.nbytes == 2 * array.size
        q, ldq = _place("q", q, rows, width, 4)
        out, ldOut = _place("out", out, rows, width, 2 if half else 4)
        entries = table.nbytes // 4
        if blocksPerRequest is None:
            blocksPerRequest = entries // requests if requests > 0 else 1
            if requests > 0 and blocksPerRequest * requests != entries:
                raise ValueError(f"a block table of {entries} entries for {requests} requests: blocksPerRequest?")
        elif blocksPerRequest * requests > entries:
            raise ValueError(f"{requests} x {blocksPerRequest} entries of a block table of {entries}")
        status = self._lib.jl_kv_attention(
            self.ctx.handle, cache.handle, q, self.heads, ldq, rows, _ints("positions", positions, rows),
            _ints("rowRequests", rowRequests, rows) if rowRequests is not None else None, table.ptr, requests,
            blocksPerRequest, self.scale if scale is None else scale, window, out, half, ldOut,
            self.workspace.ptr, self.workspace.nbytes)
        if status:
            L.check(status)
