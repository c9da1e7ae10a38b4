"""Layer operators of language models on device-resident data: the gated
delta rule, the norm block and dropout, over the C-ABI of
``include/cchip_operators.h`` (which states what each computes).

A handle is made once for its shapes, checks the arguments of each call and
keeps the workspace, one for each stream it is called on. A call only issues
work on ``stream`` (a ``runtime.Stream``, an object with ``cuda_stream``, a
raw pointer, or None for the default stream) and may be captured into a HIP
graph once its handle has been called on that stream (or ``reserve`` has);
the arrays it is given have to live until the stream is past it.

Arrays are ``Array``, ``backend_hip.Resident`` or anything with ``data_ptr()``,
``get_device()``, ``dtype``, ``shape`` and ``stride()``, such as a tensor of
a GPU framework; their last dimension is contiguous, the others may have any
stride. A wrong shape, type or stride raises ``ValueError`` before any device
work.
"""

from __future__ import annotations

import ctypes

from . import _lib
from ._lib import check, lib
from .backend_hip import Resident
from .runtime import Buffer, Device, Stream

CODES = {"f32": 0, "bf16": 5, "f16": 6}
SIZES = {"f32": 4, "bf16": 2, "f16": 2, "i32": 4, "i64": 8, "u8": 1}
NORMS = {"none": 0, "rms": 1, "layer": 2}
GATES = {"none": 0, "sigmoid": 1, "silu": 2}


def _contiguous(shape):
    out, n = [], 1
    for d in reversed(shape):
        out.append(n)
        n *= d
    return tuple(reversed(out))


class Array:
    """A device buffer read as elements of ``dtype`` (a name of ``SIZES``), with
    a shape, strides and a first element, both counted in elements."""

    __slots__ = ("buf", "dtype", "shape", "strides", "first")

    def __init__(self, buf, dtype, shape, strides=None, first=0):
        if dtype not in SIZES:
            raise ValueError("Array: unknown dtype %r" % (dtype,))
        self.buf = buf
        self.dtype = dtype
        self.shape = tuple(shape)
        self.strides = _contiguous(self.shape) if strides is None else tuple(strides)
        self.first = first
        if len(self.strides) != len(self.shape):
            raise ValueError("Array: %d strides for %d dimensions" % (len(self.strides), len(self.shape)))
        if all(self.shape):
            ends = [(d - 1) * s for d, s in zip(self.shape, self.strides)]
            low, high = first + sum(min(e, 0) for e in ends), first + sum(max(e, 0) for e in ends)
            if low < 0 or (high + 1) * SIZES[dtype] > buf.nbytes:
                raise ValueError("Array: %s elements %d .. %d do not lie in a buffer of %d bytes" % (dtype, low, high, buf.nbytes))

    @staticmethod
    def empty(dtype, shape):
        n = 1
        for d in shape:
            n *= d
        return Array(Buffer.alloc(n * SIZES[dtype]), dtype, shape)

    def data_ptr(self):
        return (self.buf.ptr or 0) + self.first * SIZES[self.dtype]

    def stride(self):
        return self.strides

    def get_device(self):
        return None  # the current device's, as every Buffer

    def free(self):
        self.buf.free()


_NAMES = {"float32": "f32", "bfloat16": "bf16", "float16": "f16", "int32": "i32", "int64": "i64", "uint8": "u8"}
_dtypes = {}  # an array's dtype object -> its name here


def _dtype_name(d):
    n = _dtypes.get(d)
    if n is None:
        s = d if isinstance(d, str) else getattr(d, "name", None) or str(d)
        s = s.rsplit(".", 1)[-1]
        n = _dtypes[d] = s if s in SIZES else _NAMES.get(s, s)
    return n


def _as_array(x):
    if isinstance(x, Resident):
        return Array(x.buf, x.dtype.name, x.shape)
    return x


def _stream_ptr(stream):
    if stream is None or isinstance(stream, int):
        return stream
    if isinstance(stream, Stream):
        return stream.ptr
    return stream.cuda_stream


def _dims(shape):
    return "[" + ", ".join(str(d) for d in shape) + "]"


class _Operator:
    _who = ""

    def __init__(self):
        self._device = Device.current() if Device.available() else None
        self._workspace_bytes = 0
        self._workspaces = {}

    def _check(self, name, x, dtype, shape):
        """The array's pointer and strides, or ValueError."""
        if type(x) is Resident:
            x = _as_array(x)
        if x.shape != shape and tuple(x.shape) != shape:
            raise ValueError("%s: %s has shape %s, expected %s" % (self._who, name, _dims(x.shape), _dims(shape)))
        if _dtypes.get(x.dtype) != dtype and _dtype_name(x.dtype) != dtype:
            raise ValueError("%s: %s has dtype %s, expected %s" % (self._who, name, _dtype_name(x.dtype), dtype))
        d = x.get_device()
        if d is not None and d != self._device:
            raise ValueError("%s: %s is not on device %s" % (self._who, name, self._device))
        return x.data_ptr(), x.stride()

    def _whole(self, name, x, dtype, shape):
        """The pointer of an array without gaps; None for None."""
        if x is None:
            return None
        p, st = self._check(name, x, dtype, shape)
        if st != _contiguous(shape) and any(a != b for a, b, d in zip(st, _contiguous(shape), shape) if d > 1):
            raise ValueError("%s: %s is not contiguous" % (self._who, name))
        return p

    def _workspace(self, stream):
        if not self._workspace_bytes:
            return None
        w = self._workspaces.get(stream)
        if w is None:
            w = self._workspaces[stream] = Buffer.alloc(self._workspace_bytes)
        return w.ptr

    def reserve(self, stream=None):
        """Allocate the workspace of a stream before the first call on it."""
        self._workspace(_stream_ptr(stream))

    def free(self):
        """Free the workspaces; the streams have to be done with them."""
        for w in self._workspaces.values():
            w.free()
        self._workspaces.clear()

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


class GatedDelta(_Operator):
    """The gated delta rule over ``[batch, tokens, heads, dim]`` arrays.

    ``u = beta (v - exp(g) S^T k)``, ``S = exp(g) S + k u^T``,
    ``o = scale S^T q`` for each token of each sequence and value head; scale
    is ``key_dim ** -0.5`` unless given. ``sequences``: that many sequences
    packed into a batch of 1, which every call says the bounds of
    (``offsets``, i32, ``sequences + 1`` values from 0 to ``tokens``).
    ``states``: whether sequences begin from or end in f32 states
    ``[sequence, value head, key_dim, value_dim]`` that the caller holds.
    """

    _who = "GatedDelta"

    def __init__(self, dtype, batch, tokens, key_heads, value_heads, key_dim, value_dim, scale=None, sequences=None,
                 states=True):
        super().__init__()
        if dtype not in CODES:
            raise ValueError("GatedDelta: dtype %r is not f32, bf16 or f16" % (dtype,))
        if sequences is not None and sequences < 1:
            raise ValueError("GatedDelta: sequences must be >= 1")
        self.dtype = dtype
        self._desc = _lib.GatedDeltaDesc(CODES[dtype], batch, tokens, sequences or 0, key_heads, value_heads, key_dim,
                                         value_dim, 1 if states else 0,
                                         key_dim ** -0.5 if scale is None and key_dim > 0 else scale or 0.0)
        w, s = ctypes.c_size_t(), ctypes.c_size_t()
        check(lib().cchip_gated_delta_sizes(self._desc, ctypes.byref(w), ctypes.byref(s)))
        self._workspace_bytes, self._saved_bytes = w.value, s.value
        self._qk = (batch, tokens, key_heads, key_dim)
        self._v = (batch, tokens, value_heads, value_dim)
        self._gates = (batch, tokens, value_heads)
        self._state = (sequences or batch, value_heads, key_dim, value_dim)
        self._offsets = None if sequences is None else (sequences + 1,)

    def saved_bytes(self):
        """Bytes of what a forward pass saves for its backward pass."""
        return self._saved_bytes

    def saved(self):
        """A fresh array for what a forward pass saves."""
        return Array.empty("u8", (self._saved_bytes,))

    def _heads(self, io, name, x, shape):
        p, st = self._check(name, x, self.dtype, shape)
        if len(shape) == 4 and shape[3] > 1 and st[3] != 1:
            raise ValueError("GatedDelta: the last dimension of %s is not contiguous" % name)
        h = getattr(io, name)
        h.data, h.batch, h.token, h.head = p, st[0], st[1], st[2]

    def _io(self, q, k, v, g, beta, offsets, saved):
        io = _lib.GatedDeltaIO()
        self._heads(io, "q", q, self._qk)
        self._heads(io, "k", k, self._qk)
        self._heads(io, "v", v, self._v)
        self._heads(io, "g", g, self._gates)
        self._heads(io, "beta", beta, self._gates)
        if self._offsets is None:
            if offsets is not None:
                raise ValueError("GatedDelta: offsets without packed sequences")
        else:
            if offsets is None:
                raise ValueError("GatedDelta: packed sequences need offsets")
            io.offsets = self._whole("offsets", offsets, "i32", self._offsets)
        if saved is not None:
            if saved.shape != (self._saved_bytes,):
                raise ValueError("GatedDelta: saved has shape %s, expected %s" % (_dims(saved.shape), _dims((self._saved_bytes,))))
            io.saved = self._whole("saved", saved, "u8", (self._saved_bytes,))
        return io

    def forward(self, q, k, v, g, beta, o, *, state=None, state_out=None, offsets=None, saved=None, stream=None):
        """Write ``o``, and the sequences' last states to ``state_out`` if given
        (it may be ``state``, where they begin; without one, at zero).
        ``saved`` is written for a backward pass if given."""
        io = self._io(q, k, v, g, beta, offsets, saved)
        self._heads(io, "o", o, self._v)
        io.state = self._whole("state", state, "f32", self._state)
        io.state_out = self._whole("state_out", state_out, "f32", self._state)
        s = _stream_ptr(stream)
        check(lib().cchip_gated_delta_forward(self._desc, io, self._workspace(s), self._workspace_bytes, s))

    def backward(self, q, k, v, g, beta, do, saved, dq, dk, dv, dg, dbeta, *, dstate_out=None, dstate=None, offsets=None,
                 stream=None):
        """From the gradients of ``o`` and of the last states (None: zero) write
        those of q, k, v, g, beta, and of the first states to ``dstate`` if
        given. ``saved`` is what ``forward`` wrote for the same inputs."""
        if saved is None:
            raise ValueError("GatedDelta: the backward pass needs what the forward pass saved")
        io = self._io(q, k, v, g, beta, offsets, saved)
        self._heads(io, "d_o", do, self._v)
        self._heads(io, "dq", dq, self._qk)
        self._heads(io, "dk", dk, self._qk)
        self._heads(io, "dv", dv, self._v)
        self._heads(io, "dg", dg, self._gates)
        self._heads(io, "dbeta", dbeta, self._gates)
        io.dstate_out = self._whole("dstate_out", dstate_out, "f32", self._state)
        io.dstate = self._whole("dstate", dstate, "f32", self._state)
        s = _stream_ptr(stream)
        check(lib().cchip_gated_delta_backward(self._desc, io, self._workspace(s), self._workspace_bytes, s))


class _RowOperator(_Operator):
    def _rows(self, name, x, needed=False):
        if x is None:
            if needed:
                raise ValueError("%s: no %s" % (self._who, name))
            return _lib.Rows(None, 0)
        p, st = self._check(name, x, self.dtype, self._shape)
        if self._shape[1] > 1 and st[1] != 1:
            raise ValueError("%s: rows of %s are not contiguous" % (self._who, name))
        return _lib.Rows(p, st[0])

    def _step(self, step):
        return self._whole("step", step, "i64", ())


class Dropout(_RowOperator):
    """Dropout of ``[rows, cols]`` arrays by the counter-based generator, its
    mask drawn when needed and never stored: the same ``seed`` and ``offset``
    give the same mask. ``step``, a one-element i64 array without dimensions,
    is added to ``offset`` on the device."""

    _who = "Dropout"

    def __init__(self, dtype, rows, cols, p, scale=1.0):
        super().__init__()
        if dtype not in CODES:
            raise ValueError("Dropout: dtype %r is not f32, bf16 or f16" % (dtype,))
        if not 0.0 <= p <= 1.0:
            raise ValueError("Dropout: p = %r is not in 0 .. 1" % (p,))
        self.dtype = dtype
        self.p = p
        self.scale = scale
        self._shape = (rows, cols)

    def forward(self, x, out, *, seed, offset=0, residual=None, step=None, stream=None):
        """``out = residual + scale drop(x)``; out may be x or residual."""
        drop = _lib.DropDesc(self.p, seed & 0xFFFFFFFFFFFFFFFF, offset & 0xFFFFFFFFFFFFFFFF, self._step(step))
        check(lib().cchip_dropout(CODES[self.dtype], self._shape[0], self._shape[1], drop, self.scale,
                                  self._rows("x", x, True), self._rows("residual", residual), self._rows("out", out, True),
                                  _stream_ptr(stream)))

    def backward(self, dout, dx, *, seed, offset=0, step=None, stream=None):
        """``dx = scale drop(dout)`` with the forward pass's mask; the residual's
        gradient is ``dout`` itself."""
        self.forward(dout, dx, seed=seed, offset=offset, step=step, stream=stream)


_PARAMS = ("post_weight", "post_bias", "channel_scale", "pre_weight", "pre_bias")


class NormBlock(_RowOperator):
    """What stands between a block's output ``y`` and the next block's input,
    on each row: ``h = residual + scale channel_scale drop(norm(y) act(gate))``
    and ``n = norm(h)``, each norm with a weight and a bias.

    ``norm`` and ``pre`` (the norm of h): "rms", "layer" or "none"; ``gate``:
    "silu", "sigmoid" or "none". Parameters are vectors of ``width`` of
    ``weight_dtype`` ("f32" or ``dtype``); one that is not given is 1 or 0."""

    _who = "NormBlock"

    def __init__(self, dtype, rows, width, norm="rms", pre="rms", gate="none", dropout=0.0, scale=1.0, eps=1e-6,
                 weight_dtype="f32"):
        super().__init__()
        if dtype not in CODES or weight_dtype not in CODES:
            raise ValueError("NormBlock: dtypes %r and %r are not f32, bf16 or f16" % (dtype, weight_dtype))
        if norm not in NORMS or pre not in NORMS or gate not in GATES:
            raise ValueError("NormBlock: unknown norm %r, pre %r or gate %r" % (norm, pre, gate))
        if not 0.0 <= dropout <= 1.0:
            raise ValueError("NormBlock: dropout = %r is not in 0 .. 1" % (dropout,))
        self.dtype = dtype
        self.weight_dtype = weight_dtype
        self.p = dropout
        self._shape = (rows, width)
        self._desc = _lib.NormBlockDesc(CODES[dtype], CODES[weight_dtype], rows, width, NORMS[norm], NORMS[pre], GATES[gate],
                                        scale, eps)
        w = ctypes.c_size_t()
        check(lib().cchip_norm_block_workspace(self._desc, ctypes.byref(w)))
        self._workspace_bytes = w.value

    def _vectors(self, given):
        p = _lib.NormParams()
        for n, x in given.items():
            if n not in _PARAMS:
                raise ValueError("NormBlock: unknown parameter %s" % n)
            setattr(p, n, self._whole(n, x, self.weight_dtype, self._shape[1:]))
        return p

    def _drop(self, seed, offset, step):
        return _lib.DropDesc(self.p, seed & 0xFFFFFFFFFFFFFFFF, offset & 0xFFFFFFFFFFFFFFFF, self._step(step))

    def forward(self, y, h, n=None, *, gate=None, residual=None, seed=0, offset=0, step=None, stream=None, **params):
        """Write ``h``, and ``n`` if there is a norm of it. h may be residual or
        y, n may be y. ``params``: post_weight, post_bias, channel_scale,
        pre_weight, pre_bias. ``seed``, ``offset`` and ``step`` as for Dropout."""
        check(lib().cchip_norm_block_forward(self._desc, self._drop(seed, offset, step), self._vectors(params),
                                             self._rows("y", y, True), self._rows("gate", gate),
                                             self._rows("residual", residual), self._rows("h", h, True),
                                             self._rows("n", n), _stream_ptr(stream)))

    def backward(self, y, dh, dy, *, dn=None, h=None, gate=None, dgate=None, dresidual=None, grads=None, seed=0, offset=0,
                 step=None, stream=None, **params):
        """From y, gate, the forward pass's h (where it is normed again) and the
        gradients of h and n, write those of y, gate and residual and, for each
        name in ``grads``, of that parameter, summed over the rows."""
        s = _stream_ptr(stream)
        check(lib().cchip_norm_block_backward(self._desc, self._drop(seed, offset, step), self._vectors(params),
                                              self._vectors(grads or {}), self._rows("y", y, True), self._rows("gate", gate),
                                              self._rows("h", h), self._rows("dh", dh, True), self._rows("dn", dn),
                                              self._rows("dy", dy, True), self._rows("dgate", dgate),
                                              self._rows("dresidual", dresidual), self._workspace(s), self._workspace_bytes,
                                              s))
