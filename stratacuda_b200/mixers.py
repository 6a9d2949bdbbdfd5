"""Token mixers over runs of many sequences (include/strata_cuda.h, strata_delta_* and strata_qk_rope).

The reference walks the gated delta rule token after token and makes its inputs, and the queries and keys of attention, in five
dispatches each (src/engine.js, src/prefill.js). Here one call takes several tokens of several sequences:

* ``inputs`` — a delta-rule layer's convolution with each sequence's history, SiLU and the norms of its q and k heads;
* ``rule`` — the gated delta rule on each sequence's state, chunked on the tensor cores for prompts, token by token for decode;
* ``QkRope.apply`` — the norms of queries and keys for each head with the position's rotation in the same pass.

A call works on ``segments`` runs of ``count`` rows. Run i is sequence[i]'s (-1: an idle slot) and has lengths[i] tokens (all
of its rows without ``lengths``); both are read on the device.

``DeltaNet`` and ``QkRope`` work on Buffers of a CudaBackend and its stream. ``DeviceDeltaNet`` and ``DeviceQkRope`` are the same
on caller-owned device memory (torch tensors, or plain addresses) and a stream of the caller's.
"""
from __future__ import annotations

import ctypes as C
import struct

import numpy as np

from . import _lib as L
from .backend import StrataError, StrataRangeError
from .kv8 import _Types, _address, _int32, _message, _strided, _words


def sizes(key_heads: int, value_heads: int, dim: int, sequences: int, taps: int = 4) -> dict:
    """Elements (of 4 bytes) of a delta-rule layer's parts."""
    channels = (2 * key_heads + value_heads) * dim
    return dict(state=sequences * dim * value_heads * dim, history=sequences * channels * (taps - 1), weight=channels * taps,
                workspace=L.DELTA_WORKSPACE_BYTES // 4)


def borrow_workspace(backend):
    """The workspace that users of a backend share, whose calls follow one another on its stream: made for the first of them, freed when the
    last one gives it back (``return_workspace``)."""
    shared = getattr(backend, "_delta_workspace", None)
    if shared is None:
        shared = backend._delta_workspace = [backend.alloc(L.DELTA_WORKSPACE_BYTES // 4, "u32", zero=False), 0]
    shared[1] += 1
    return shared[0]


def return_workspace(backend) -> None:
    shared = backend._delta_workspace
    shared[1] -= 1
    if not shared[1]:
        backend._delta_workspace = None
        backend.free(shared[0])


def _cuda(backend):
    if getattr(backend, "kind", None) != "cuda":
        raise StrataRangeError(L.ERR_RANGE, "the token mixers over runs need the CUDA backend")
    return backend


def _handle(buf) -> int:
    return 0 if buf is None else buf.handle


def _strides(**values) -> None:
    for name, x in values.items():
        if not isinstance(x, (int, np.integer)) or not 0 <= x < 1 << 64:
            raise StrataRangeError(L.ERR_RANGE, f"{name} must be an integer in [0, 2^64)")


class DeltaNet:
    """One layer's delta rule for `sequences` sequences on a CudaBackend: `state` and `history` (zeroed ones of its own where
    None), the convolution's `weight` (None: only ``rule`` is used), and a `workspace`, which calls that follow one another on the
    backend's stream may share."""

    def __init__(self, backend, key_heads: int, value_heads: int, dim: int, sequences: int, taps: int = 4, state=None, history=None,
                 weight=None, workspace=None):
        self.b = _cuda(backend)
        _int32(key_heads=key_heads, value_heads=value_heads, dim=dim, sequences=sequences, taps=taps)
        self.key_heads, self.value_heads, self.dim, self.sequences, self.taps = key_heads, value_heads, dim, sequences, taps
        n = sizes(key_heads, value_heads, dim, sequences, taps)
        self._owned = []

        def keep(given, what, type="f32"):
            if given is not None:
                return given
            buf = backend.alloc(n[what], type, zero=True)
            self._owned.append(buf)
            return buf

        try:
            self.state = keep(state, "state")
            self.history = keep(history, "history") if taps > 1 else None
            self.workspace = keep(workspace, "workspace", "u32")
        except BaseException:  # nobody else has them
            self.free()
            raise
        self.weight = weight

    def _struct(self) -> L.StrataDeltaNet:
        return L.StrataDeltaNet(self.key_heads, self.value_heads, self.dim, self.taps, self.sequences, self.state.handle,
                                _handle(self.history), _handle(self.weight), self.workspace.handle)

    def inputs(self, x, q, k, v, sequence, segments: int = 1, count: int = 1, lengths=None, row_stride: int = 0, q_scale: float = 0.0,
               epsilon: float = 1e-6) -> None:
        """q, k, v from projection rows x (strata_delta_inputs). `q_scale` 0 is 1 / sqrt(dim)."""
        _int32(segments=segments, count=count)
        _strides(row_stride=row_stride)
        self.b._check(self.b.lib.strata_delta_inputs(self.b.ctx, C.byref(self._struct()), x.handle, row_stride, segments, count,
                                                     sequence.handle, _handle(lengths), q_scale, epsilon, q.handle, k.handle, v.handle))

    def rule(self, q, k, v, decay, beta, y, sequence, segments: int = 1, count: int = 1, lengths=None, q_stride: int = 0, k_stride: int = 0,
             v_stride: int = 0) -> None:
        """y, and the sequences' new states, from rows q, k, v, decay and beta (strata_delta_rule)."""
        _int32(segments=segments, count=count)
        _strides(q_stride=q_stride, k_stride=k_stride, v_stride=v_stride)
        self.b._check(self.b.lib.strata_delta_rule(self.b.ctx, C.byref(self._struct()), q.handle, q_stride, k.handle, k_stride, v.handle,
                                                   v_stride, decay.handle, beta.handle, segments, count, sequence.handle, _handle(lengths),
                                                   y.handle))

    def free(self) -> None:
        for buf in self._owned:
            self.b.free(buf)
        self._owned = []


class QkRope:
    """Norm weights of queries and keys, and a rotation's tables, on a CudaBackend. `sequences` bounds the numbers that `sequence`
    may hold."""

    def __init__(self, backend, heads: int, kv_heads: int, dim: int, rotary: int, cells: int, q_weight, k_weight, cos=None, sin=None,
                 sequences: int = 0x7FFFFFFF):
        self.b = _cuda(backend)
        _int32(heads=heads, kv_heads=kv_heads, dim=dim, rotary=rotary, cells=cells, sequences=sequences)
        self.parts = (q_weight, k_weight, cos, sin)
        self._weights = L.StrataQkRopeWeights(heads, kv_heads, dim, rotary, cells, sequences, q_weight.handle, k_weight.handle, _handle(cos),
                                              _handle(sin))

    def apply(self, q, k, yq, yk, start, segments: int = 1, count: int = 1, sequence=None, lengths=None, q_stride: int = 0,
              q_head_stride: int = 0, k_stride: int = 0, epsilon: float = 1e-6) -> None:
        """yq, yk: the normed and rotated heads of rows q and k (strata_qk_rope)."""
        _int32(segments=segments, count=count)
        _strides(q_stride=q_stride, q_head_stride=q_head_stride, k_stride=k_stride)
        self.b._check(self.b.lib.strata_qk_rope(self.b.ctx, C.byref(self._weights), q.handle, q_stride, q_head_stride, k.handle, k_stride,
                                                segments, count, _handle(sequence), start.handle, _handle(lengths), epsilon, yq.handle,
                                                yk.handle))


class _Device:
    """What both views of caller-owned memory do with tensors, Buffers and addresses."""

    _device = _cuda = None

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

    def _rows(self, x, what: str, rows: int, width: int, stride: int):
        return _strided(x, what, rows, width, stride, self._device) if stride else self._floats(x, what, rows * width)

    def _where(self):
        """The parts' device, if a tensor among them tells. The only device there is is the current one: nothing to look at in calls."""
        self._device = next((x.get_device() for x in self.parts if hasattr(x, "get_device")), None)
        if self._device is not None:
            import torch
            self._cuda = None if self._device == 0 and torch.cuda.device_count() == 1 else torch.cuda
        return self._device

    def _here(self) -> None:
        """Calls go to a stream of the current device: refused where that is not the one that holds the parts. (A launch refuses a stream of
        another device than the current one.)"""
        if self._cuda is not None and (now := self._cuda.current_device()) != self._device:
            raise StrataError(L.ERR_LAYOUT, f"the parts are on device {self._device}, the current device is {now}: its default stream, or "
                                            "another of its streams, is where the call would go")

    def _run(self, entry, pack, *values) -> None:
        try:
            call = pack(*values)
        except (struct.error, OverflowError) as e:
            raise StrataRangeError(L.ERR_RANGE, f"an argument is not a number of its type: {e}") from None
        rc = entry(call)
        if rc != L.OK:
            raise (StrataRangeError if rc == L.ERR_RANGE else StrataError)(rc, _message.text.value.decode(errors="replace"))


_pack_inputs, _pack_rule, _pack_rope = L.DELTA_INPUTS_CALL.pack, L.DELTA_RULE_CALL.pack, L.QK_ROPE_CALL.pack


class DeviceDeltaNet(_Device):
    """A delta-rule layer in caller-owned device memory: torch tensors, Buffers or addresses of the layouts in
    include/strata_cuda.h. Tensors are checked for their type, device, order and size and Buffers for their size; addresses are the
    caller's word. ``inputs`` needs `weight` and (with taps > 1) `history`, ``rule`` needs `state` and `workspace`. Calls go to
    `stream` (a cudaStream_t as an integer; 0 is the default stream) of the current device, which has to be the parts', allocate
    nothing and do not synchronise. `status`, where given, is a zeroed 32-bit device word that device-side errors are added to. The parts must stay
    alive."""

    def __init__(self, key_heads: int, value_heads: int, dim: int, sequences: int, taps: int = 4, state=None, history=None, weight=None,
                 workspace=None, status=None):
        lib = L.load()
        self._inputs, self._rule = lib.strata_delta_inputs_dev, lib.strata_delta_rule_dev
        _int32(key_heads=key_heads, value_heads=value_heads, dim=dim, sequences=sequences, taps=taps)
        self.parts = (state, history, weight, workspace, status)
        d = self._where()
        n = sizes(key_heads, value_heads, dim, sequences, taps)
        self.kd, self.vd, self.value_heads = key_heads * dim, value_heads * dim, value_heads
        self._net = L.StrataDeltaNetDev(key_heads, value_heads, dim, taps, sequences, _address(state, "state", n["state"], "float32", d),
                                        _address(history, "history", n["history"], "float32", d),
                                        _address(weight, "weight", n["weight"], "float32", d), _words(workspace, "workspace", n["workspace"], d),
                                        _words(status, "status", 1, d))
        self._at = C.addressof(self._net)

    def inputs(self, x, q, k, v, sequence, segments: int = 1, count: int = 1, lengths=None, row_stride: int = 0, q_scale: float = 0.0,
               epsilon: float = 1e-6, stream: int = 0) -> None:
        n = segments * count
        self._here()
        self._run(self._inputs, _pack_inputs, self._at, self._rows(x, "x", n, 2 * self.kd + self.vd, row_stride), row_stride,
                  self._ints(sequence, "sequence", segments), 0 if lengths is None else self._ints(lengths, "lengths", segments),
                  self._floats(q, "q", n * self.kd), self._floats(k, "k", n * self.kd), self._floats(v, "v", n * self.vd), stream, _message.at,
                  256, segments, count, q_scale, epsilon)

    def rule(self, q, k, v, decay, beta, y, sequence, segments: int = 1, count: int = 1, lengths=None, q_stride: int = 0, k_stride: int = 0,
             v_stride: int = 0, stream: int = 0) -> None:
        n = segments * count
        self._here()
        self._run(self._rule, _pack_rule, self._at, self._rows(q, "q", n, self.kd, q_stride), self._rows(k, "k", n, self.kd, k_stride),
                  self._rows(v, "v", n, self.vd, v_stride), q_stride, k_stride, v_stride, self._floats(decay, "decay", n * self.value_heads),
                  self._floats(beta, "beta", n * self.value_heads), self._ints(sequence, "sequence", segments),
                  0 if lengths is None else self._ints(lengths, "lengths", segments), self._floats(y, "y", n * self.vd), stream, _message.at,
                  256, segments, count)


class DeviceQkRope(_Device):
    """Norm weights and a rotation's tables in caller-owned device memory, as in DeviceDeltaNet. `sequences` bounds the numbers
    that `sequence` may hold."""

    def __init__(self, heads: int, kv_heads: int, dim: int, rotary: int, cells: int, q_weight, k_weight, cos=None, sin=None,
                 sequences: int = 0x7FFFFFFF, status=None):
        self._entry = L.load().strata_qk_rope_dev
        _int32(heads=heads, kv_heads=kv_heads, dim=dim, rotary=rotary, cells=cells, sequences=sequences)
        self.parts = (q_weight, k_weight, cos, sin, status)
        d = self._where()
        self.heads, self.dim, self.kw = heads, dim, kv_heads * dim
        self._weights = L.StrataQkRopeWeightsDev(heads, kv_heads, dim, rotary, cells, sequences,
                                                 _address(q_weight, "q_weight", dim, "float32", d), _address(k_weight, "k_weight", dim, "float32", d),
                                                 _address(cos, "cos", cells * (rotary // 2), "float32", d),
                                                 _address(sin, "sin", cells * (rotary // 2), "float32", d), _words(status, "status", 1, d))
        self._at = C.addressof(self._weights)

    def apply(self, q, k, yq, yk, start, segments: int = 1, count: int = 1, sequence=None, lengths=None, q_stride: int = 0,
              q_head_stride: int = 0, k_stride: int = 0, epsilon: float = 1e-6, stream: int = 0) -> None:
        n, apart = segments * count, q_head_stride or self.dim
        self._here()
        reach = (self.heads - 1) * apart + self.dim  # from a row's first head to the end of its last
        if q_stride:
            pq = _strided(q, "q", n, reach, q_stride, self._device)
        else:
            pq = self._floats(q, "q", (n - 1) * self.heads * apart + reach)
        self._run(self._entry, _pack_rope, self._at, pq, self._rows(k, "k", n, self.kw, k_stride), q_stride, q_head_stride, k_stride,
                  0 if sequence is None else self._ints(sequence, "sequence", segments), self._ints(start, "start", segments),
                  0 if lengths is None else self._ints(lengths, "lengths", segments), self._floats(yq, "yq", n * self.heads * self.dim),
                  self._floats(yk, "yk", n * self.kw), stream, _message.at, 256, segments, count, epsilon)
