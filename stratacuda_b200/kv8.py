"""Attention over a paged key/value cache held in 8 bits (include/strata_cuda.h, strata_kv8_*).

The reference keeps F32 caches of at most 2048 cells (src/model.js:13). Here a cache holds one byte
per value with a scale for each block of 64 tokens and head, in pages that sequences take from one
pool, so that sessions can be longer and more of them fit. Three operators work on it:

* ``append`` — quantise new key and value rows into the sequences' pages;
* ``select`` — choose, for each token and key/value head, the blocks with the largest bound on the
  logits, from two 8-bit marks per block and channel;
* ``attend`` — softmax attention over all blocks or over the chosen ones, F32 in and out, for single
  tokens of many sequences and for prompt chunks.

``Kv8Cache`` owns its buffers on a CudaBackend and works on its stream. ``DeviceCache`` is a view of
caller-owned device memory (torch tensors, or plain addresses) on a stream of the caller's.
"""
from __future__ import annotations

import ctypes as C
import math
import struct
import threading

import numpy as np

from . import _lib as L
from .backend import Buffer, StrataError, StrataRangeError

BLOCK = L.KV8_BLOCK


def padded(dim: int) -> int:
    """Channels that a page stores for heads of `dim`."""
    return 64 if dim <= 64 else 128 if dim <= 128 else 256


def sizes(kv_heads: int, dim: int, pages: int, sequences: int, blocks: int) -> dict:
    """Elements of a cache's parts: codes and marks in bytes, the others in 4-byte elements."""
    p = padded(dim)
    return dict(codes=pages * kv_heads * 2 * p * BLOCK, marks=pages * kv_heads * 2 * p, scales=pages * kv_heads * 2,
                open=sequences * 2 * BLOCK * kv_heads * dim, table=sequences * blocks, workspace=L.KV8_WORKSPACE_BYTES // 4)


def _int32(**values) -> None:
    for name, x in values.items():
        if not -(1 << 31) <= x < 1 << 31:
            raise StrataRangeError(L.ERR_RANGE, f"{name} must be a 32-bit integer")


class Kv8Cache:
    """One layer's cache on a CudaBackend. `pages` defaults to a page for every block of every
    sequence, in order; with fewer, the caller hands pages out with ``write_table``."""

    def __init__(self, backend, kv_heads: int, dim: int, sequences: int, blocks: int, pages: int | None = None, workspace=None):
        if getattr(backend, "kind", None) != "cuda":
            raise StrataRangeError(L.ERR_RANGE, "an 8-bit cache needs the CUDA backend")
        _int32(kv_heads=kv_heads, dim=dim, sequences=sequences, blocks=blocks, pages=sequences * blocks if pages is None else pages)
        self.b = backend
        self.kv_heads, self.dim, self.sequences, self.blocks = kv_heads, dim, sequences, blocks
        self.pages = sequences * blocks if pages is None else pages
        n = sizes(kv_heads, dim, self.pages, sequences, blocks)
        self._owned = []

        def keep(length, type="f32"):
            buf = backend.alloc(length, type, zero=True)
            self._owned.append(buf)
            return buf

        try:
            self.codes, self.marks = keep(n["codes"] // 4, "u32"), keep(n["marks"] // 4, "u32")
            self.scales, self.open, self.table = keep(n["scales"]), keep(n["open"]), keep(n["table"], "i32")
            # caches whose calls follow one another on the backend's stream may share one workspace
            self.workspace = keep(n["workspace"], "u32") if workspace is None else workspace
            if pages is None:
                self.write_table(np.arange(self.pages, dtype=np.int32).reshape(sequences, blocks))
            else:
                self.write_table(np.full((sequences, blocks), -1, np.int32))
        except BaseException:  # nobody else has them
            self.free()
            raise

    def write_table(self, table) -> None:
        """The page of every block of every sequence, int [sequences][blocks]; -1 where there is none yet."""
        table = np.ascontiguousarray(table, np.int32)
        if table.shape != (self.sequences, self.blocks):
            raise StrataError(L.ERR_LAYOUT, f"the page table is [{self.sequences}][{self.blocks}]")
        self.b.write(self.table, table.ravel())

    def _struct(self) -> L.StrataKv8Cache:
        return L.StrataKv8Cache(self.kv_heads, self.dim, self.pages, self.sequences, self.blocks, self.codes.handle, self.marks.handle,
                                self.scales.handle, self.open.handle, self.table.handle, self.workspace.handle)

    def append(self, k, v, sequence, start, segments: int = 1, count: int = 1, row_stride: int = 0) -> None:
        """Append rows k and v [segments * count][kv_heads * dim] (strata_kv8_append)."""
        _int32(segments=segments, count=count)
        self.b._check(self.b.lib.strata_kv8_append(self.b.ctx, C.byref(self._struct()), k.handle, v.handle, row_stride, segments, count,
                                                   sequence.handle, start.handle))

    def select(self, q, heads: int, picks, sequence, start, segments: int = 1, count: int = 1, top: int = 32, first: int = 1, last: int = 2,
               row_stride: int = 0) -> None:
        """picks [segments * count][kv_heads][top] (i32): the chosen blocks (strata_kv8_select)."""
        _int32(segments=segments, count=count, heads=heads, top=top, first=first, last=last)
        self.b._check(self.b.lib.strata_kv8_select(self.b.ctx, C.byref(self._struct()), q.handle, row_stride, heads, segments, count,
                                                   sequence.handle, start.handle, top, first, last, picks.handle))

    def attend(self, q, heads: int, y, sequence, start, segments: int = 1, count: int = 1, picks=None, top: int = 0,
               scale: float | None = None, row_stride: int = 0) -> None:
        """y [segments * count][heads * dim]: attention over all blocks, or those in `picks` (strata_kv8_attend).
        `scale` defaults to 1 / sqrt(dim)."""
        _int32(segments=segments, count=count, heads=heads, top=top)
        self.b._check(self.b.lib.strata_kv8_attend(self.b.ctx, C.byref(self._struct()), q.handle, row_stride, heads, segments, count,
                                                   sequence.handle, start.handle, 0 if picks is None else picks.handle, top,
                                                   1 / math.sqrt(self.dim) if scale is None else scale, y.handle))

    def free(self) -> None:
        for buf in self._owned:
            self.b.free(buf)
        self._owned = []


class _Types:
    """torch's element types, once a tensor has been seen."""
    int8 = int32 = float32 = None

    @classmethod
    def known(cls):
        if cls.int8 is None:
            import torch
            cls.int8, cls.int32, cls.float32 = torch.int8, torch.int32, torch.float32
        return cls


def _memory(x, what: str, need: int, device):
    """Device address of a tensor's elements, `need` or more that follow one another."""
    if x.get_device() < 0 or (device is not None and x.get_device() != device):
        raise StrataError(L.ERR_LAYOUT, f"{what} must be on the cache's CUDA device, not on {x.device}")
    if not x.is_contiguous():
        raise StrataError(L.ERR_LAYOUT, f"{what} must be contiguous (rows of k, v and q may be row_stride apart)")
    if x.numel() < need:
        raise StrataError(L.ERR_LAYOUT, f"{what} needs {need} elements, the tensor has {x.numel()}")
    return x.data_ptr()


def _address(x, what: str, need: int, dtype: str, device):
    """Device address of `need` elements: of a tensor of that type or a Buffer that has them, or as given."""
    if x is None or isinstance(x, int):
        return x or 0
    if isinstance(x, Buffer):
        if x.length < need:
            raise StrataError(L.ERR_LAYOUT, f"{what} needs {need} elements, the buffer has {x.length}")
        return x.device_ptr
    if x.dtype is not getattr(_Types.known(), dtype):
        raise StrataError(L.ERR_LAYOUT, f"{what} must be a tensor of torch.{dtype}, not {x.dtype}")
    return _memory(x, what, need, device)


def _words(x, what: str, need: int, device):
    """The same of `need` 32-bit words, in a tensor of any type."""
    if hasattr(x, "element_size"):
        return _memory(x, what, -(-4 * need // x.element_size()), device)
    return _address(x, what, need, "int32", device)


def _strided(x, what: str, rows: int, width: int, row_stride: int, device):
    """The same of `rows` rows of `width` floats, `row_stride` apart."""
    if x is None or isinstance(x, (int, Buffer)) or x.is_contiguous():
        return _address(x, what, (rows - 1) * row_stride + width, "float32", device)
    # a view of some columns of longer rows
    if x.dim() != 2 or x.stride(1) != 1 or x.stride(0) != row_stride or x.shape[0] < max(rows, 1) or x.shape[1] < width:
        raise StrataError(L.ERR_LAYOUT, f"{what} must be {rows} rows of {width} elements, {row_stride} apart")
    return _address(x[0], what, width, "float32", device)


class _Message(threading.local):
    """Where a thread's calls leave the reason for a refusal."""

    def __init__(self):
        self.text = C.create_string_buffer(256)
        self.at = C.addressof(self.text)


_message = _Message()
_pack = L.KV8_CALL.pack


class DeviceCache:
    """A cache in caller-owned device memory: torch tensors, Buffers or addresses of the layouts in
    include/strata_cuda.h. Tensors are checked for their type, device, order and size and Buffers for their size; addresses
    are the caller's word. Calls go to `stream` (a cudaStream_t as an integer; 0 is the default
    stream) of the current device, allocate nothing and do not synchronise. `status`, where given, is
    a zeroed 32-bit device word that device-side errors are added to. The parts must stay alive."""

    def __init__(self, kv_heads: int, dim: int, pages: int, sequences: int, blocks: int, codes, marks, scales, open, table, workspace,
                 status=None):
        self.lib = L.load()
        self.kv_heads, self.dim = kv_heads, dim
        self.parts = (codes, marks, scales, open, table, workspace, status)
        _int32(kv_heads=kv_heads, dim=dim, pages=pages, sequences=sequences, blocks=blocks)
        self._device = d = codes.get_device() if hasattr(codes, "get_device") else None
        n = sizes(kv_heads, dim, pages, sequences, blocks)

        def codes_at(x, what):  # a Buffer has them four to an element
            return _address(x, what, n[what] // 4 if isinstance(x, Buffer) else n[what], "int8", d)

        self._cache = L.StrataKv8CacheDev(kv_heads, dim, pages, sequences, blocks, codes_at(codes, "codes"), codes_at(marks, "marks"),
                                          _address(scales, "scales", n["scales"], "float32", d),
                                          _address(open, "open", n["open"], "float32", d), _address(table, "table", n["table"], "int32", d),
                                          _words(workspace, "workspace", n["workspace"], d), _words(status, "status", 1, d))
        self._at = C.addressof(self._cache)
        self._scale = 1 / math.sqrt(dim) if dim > 0 else 0.0

    def _call(self, rows, v, row_stride, sequence, start, picks, y, stream, op, segments, count, heads=0, top=0, first=0, last=0, scale=0.0) -> None:
        try:
            call = _pack(self._at, rows, v, row_stride, sequence, start, picks, y, stream, _message.at, 256, op, segments, count, heads,
                                   top, first, last, scale)
        except (struct.error, OverflowError) as e:
            raise StrataRangeError(L.ERR_RANGE, f"an argument is not a number of its type: {e}") from None
        rc = self.lib.strata_kv8_call_dev(call)
        if rc != L.OK:
            raise (StrataRangeError if rc == L.ERR_RANGE else StrataError)(rc, _message.text.value.decode(errors="replace"))

    # most calls' tensors are as they should be: these look at that at once, and leave the rest to _address
    def _floats(self, x, what: str, need: int):
        try:
            if x.dtype is _Types.float32 and x.get_device() == self._device and x.numel() >= need and x.is_contiguous():
                return x.data_ptr()
        except AttributeError:  # an address or a Buffer
            pass
        return _address(x, what, need, "float32", self._device)

    def _ints(self, x, what: str, need: int):
        try:
            if x.dtype is _Types.int32 and x.get_device() == self._device and x.numel() >= need and x.is_contiguous():
                return x.data_ptr()
        except AttributeError:  # an address or a Buffer
            pass
        return _address(x, what, need, "int32", self._device)

    def append(self, k, v, sequence, start, segments: int = 1, count: int = 1, row_stride: int = 0, stream: int = 0) -> None:
        n, w = segments * count, self.kv_heads * self.dim
        self._call(_strided(k, "k", n, w, row_stride, self._device) if row_stride else self._floats(k, "k", n * w),
                   _strided(v, "v", n, w, row_stride, self._device) if row_stride else self._floats(v, "v", n * w), row_stride,
                   self._ints(sequence, "sequence", segments), self._ints(start, "start", segments), 0, 0, stream, L.KV8_APPEND, segments, count)

    def select(self, q, heads: int, picks, sequence, start, segments: int = 1, count: int = 1, top: int = 32, first: int = 1, last: int = 2,
               row_stride: int = 0, stream: int = 0) -> None:
        n, w = segments * count, heads * self.dim
        self._call(_strided(q, "q", n, w, row_stride, self._device) if row_stride else self._floats(q, "q", n * w), 0, row_stride,
                   self._ints(sequence, "sequence", segments), self._ints(start, "start", segments),
                   self._ints(picks, "picks", n * self.kv_heads * top), 0, stream, L.KV8_SELECT, segments, count, heads, top, first, last)

    def attend(self, q, heads: int, y, sequence, start, segments: int = 1, count: int = 1, picks=None, top: int = 0,
               scale: float | None = None, row_stride: int = 0, stream: int = 0) -> None:
        n, w = segments * count, heads * self.dim
        self._call(_strided(q, "q", n, w, row_stride, self._device) if row_stride else self._floats(q, "q", n * w), 0, row_stride,
                   self._ints(sequence, "sequence", segments), self._ints(start, "start", segments),
                   0 if picks is None else self._ints(picks, "picks", n * self.kv_heads * top), self._floats(y, "y", n * w), stream,
                   L.KV8_ATTEND, segments, count, heads, top, 0, 0, self._scale if scale is None else scale)
