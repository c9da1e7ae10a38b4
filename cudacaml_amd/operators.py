"""Layer operators of language models on device-resident data: the gated
delta rule, attention, the norm and rotation of its heads, the embedding, the
norm block and dropout, over the C-ABI of ``include/cchip_operators.h`` (which
states what each computes).

A handle is made once for its shapes, checks the arguments of each call and
keeps the workspaces, one for each direction and stream it is called on; they
stay where they are until ``free``. A call only issues work on ``stream`` (a
``runtime.Stream``, an object with ``cuda_stream``, a raw pointer, or None for
the default stream) and may be captured into a HIP graph once the handle has
its workspace there (``reserve``, or an earlier call); the arrays it is given
have to live until the stream is past it.

A graph uses the workspace that its call was captured with: the handle has to
outlive the graph, and a replay must not run while another replay or a call
on the capture stream uses the same workspace. A call with a ``workspace`` of
the caller's own (u8, ``workspace_bytes`` at least, aligned to 16 bytes) is
free of both.

Arrays are ``Array``, ``backend_hip.Resident`` or anything with ``data_ptr()``,
``get_device()``, ``dtype``, ``shape`` and ``stride()``, such as a tensor of
a GPU framework; their last dimension is contiguous, the others may have any
stride (tokens of heads one of 0 to 2^23 elements). A wrong shape, type or
stride raises ``ValueError`` before any device work.
"""

from __future__ import annotations

import ctypes
import functools
import struct

from . import _lib
from ._lib import check, lib
from .backend_hip import Resident
from .runtime import Buffer, Device, Stream

CODES = {"f32": 0, "bf16": 5, "f16": 6}
SIZES = {"f32": 4, "bf16": 2, "f16": 2, "i32": 4, "i64": 8, "u8": 1}
NORMS = {"none": 0, "rms": 1, "layer": 2}
GATES = {"none": 0, "sigmoid": 1, "silu": 2}


@functools.lru_cache(maxsize=1024)
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


def _stream_ptr(stream):
    if stream is None or isinstance(stream, int):
        return stream
    if isinstance(stream, Stream):
        return stream.ptr
    return stream.cuda_stream


def _stream_on(who, device, stream):
    """The same for a handle of one device of several: a call while another is
    current is refused, as its kernels would run there."""
    if Device.current() != device:
        raise ValueError("%s: made for device %d, called on device %d" % (who, device, Device.current()))
    return _stream_ptr(stream)


def _dims(shape):
    return "[" + ", ".join(str(d) for d in shape) + "]"


_NO_ROWS = (0, 0)


class _Operator:
    _who = ""
    _on = staticmethod(_stream_ptr)

    def __init__(self):
        self._device = Device.current() if Device.available() else None
        if self._device is not None and Device.count() > 1:
            self._on = functools.partial(_stream_on, self._who, self._device)
        self._workspaces = {}

    def _view(self, name, x, dtype, shape):
        """The array's pointer and strides, or ValueError."""
        if x is None:
            raise ValueError("%s: no %s" % (self._who, name))
        if type(x) is Resident:
            x = Array(x.buf, x.dtype.name, x.shape)
        try:
            have, d, device, p, st = x.shape, x.dtype, x.get_device(), x.data_ptr(), x.stride()
        except AttributeError:
            raise ValueError("%s: %s is no array on a device" % (self._who, name)) from None
        if have != shape and tuple(have) != shape:
            raise ValueError("%s: %s has shape %s, expected %s" % (self._who, name, _dims(have), _dims(shape)))
        if _dtypes.get(d) != dtype and _dtype_name(d) != dtype:
            raise ValueError("%s: %s has dtype %s, expected %s" % (self._who, name, _dtype_name(d), dtype))
        if device != self._device and device is not None:
            raise ValueError("%s: %s is not on device %s" % (self._who, name, self._device))
        return p, st

    def _whole(self, name, x, dtype, shape):
        """The pointer of an array without gaps; 0 for None."""
        if x is None:
            return 0
        p, st = self._view(name, x, dtype, shape)
        if st != _contiguous(shape) and any(a != b for a, b, d in zip(st, _contiguous(shape), shape) if d > 1):
            raise ValueError("%s: %s is not contiguous" % (self._who, name))
        return p

    _forward_bytes = 0
    _backward_bytes = 0

    def workspace_bytes(self, backward=False):
        """Bytes of workspace that a call of a direction needs."""
        return self._backward_bytes if backward else self._forward_bytes

    def _workspace(self, stream, backward=False, given=None):
        """The pointer and bytes of a call's workspace: the one given, or the
        stream's own for this direction. That one is never replaced, as a
        captured graph may hold it."""
        n = self.workspace_bytes(backward)
        if given is not None:
            have = given.shape[0] if len(given.shape) == 1 else 0
            return self._whole("workspace", given, "u8", (have,)), have
        if not n:
            return None, 0
        w = self._workspaces.get((stream, backward))
        if w is None:
            w = self._workspaces[stream, backward] = Buffer.alloc(n)
        return w.ptr, n

    def free(self):
        """Free the workspaces; streams and captured graphs have to be done
        with them."""
        for w in self._workspaces.values():
            w.free()
        self._workspaces.clear()

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


def _check_dtype(who, *names):
    for n in names:
        if n not in CODES:
            raise ValueError("%s: dtype %r is not f32, bf16 or f16" % (who, n))


class _HeadOperator(_Operator):
    """Operators on ``[batch, tokens, heads, dim]`` arrays, whose shapes
    ``_shapes`` has by name."""

    def _words(self, **given):
        """Pointer and three strides of each array. The loop does in one go what
        _view does with words to say: a call on small arrays costs little more
        than looking at them."""
        words, device, dtype, shapes = [], self._device, self.dtype, self._shapes
        for name, x in given.items():
            shape = shapes[name]
            try:
                st = x.stride()
                plain = x.shape == shape and _dtypes[x.dtype] == dtype and x.get_device() == device
                p = x.data_ptr()
            except (AttributeError, KeyError):
                plain = False
            if not plain:
                p, st = self._view(name, x, dtype, shape)
            if len(st) == 4:
                if st[3] != 1 and shape[3] > 1:
                    raise ValueError("%s: the last dimension of %s is not contiguous" % (self._who, name))
                st = st[:3]
            words.append(p)
            words += st
        return words

    def _bounds(self, offsets):
        if (offsets is None) != (self._offsets is None):
            raise ValueError("%s: packed sequences need offsets" % self._who if offsets is None else
                             "%s: offsets without packed sequences" % self._who)
        return self._whole("offsets", offsets, "i32", self._offsets)

    _saved_bytes = 0

    def saved_bytes(self):
        """Bytes of what a forward pass saves for its backward pass."""
        return self._saved_bytes

    def saved(self):
        """A fresh array for what a forward pass saves."""
        return Array.empty("u8", (self._saved_bytes,))

    def _kept(self, saved):
        return self._whole("saved", saved, "u8", (self._saved_bytes,))

    def reserve(self, stream=None, backward=False):
        """Allocate a stream's workspace for forward calls, and that for
        backward calls, ahead of the first of them."""
        for back in (False, True)[:1 + bool(backward)]:
            self._workspace(self._on(stream), back)


class GatedDelta(_HeadOperator):
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
    # cchip_gated_delta_io: twelve cchip_heads of four words, six pointers
    _forward_io = struct.Struct("24q192x6q")
    _backward_io = struct.Struct("20q32x24q6q")

    def __init__(self, dtype, batch, tokens, key_heads, value_heads, key_dim, value_dim, scale=None, sequences=None,
                 states=True):
        super().__init__()
        _check_dtype("GatedDelta", dtype)
        if sequences is not None and sequences < 1:
            raise ValueError("GatedDelta: sequences must be >= 1")
        self.dtype = dtype
        self._desc = _lib.GatedDeltaDesc(CODES[dtype], batch, tokens, sequences or 0, key_heads, value_heads, key_dim,
                                         value_dim, 1 if states else 0,
                                         key_dim ** -0.5 if scale is None and key_dim > 0 else scale or 0.0)
        sizes = [ctypes.c_size_t() for _ in range(3)]
        check(lib().cchip_gated_delta_sizes(self._desc, *sizes))
        self._forward_bytes, self._backward_bytes, self._saved_bytes = (x.value for x in sizes)
        qk, v, gates = (batch, tokens, key_heads, key_dim), (batch, tokens, value_heads, value_dim), (batch, tokens, value_heads)
        self._shapes = dict(q=qk, k=qk, dq=qk, dk=qk, v=v, o=v, do=v, dv=v, g=gates, beta=gates, dg=gates, dbeta=gates)
        self._state = (sequences or batch, value_heads, key_dim, value_dim)
        self._offsets = None if sequences is None else (sequences + 1,)

    def forward(self, q, k, v, g, beta, o, *, state=None, state_out=None, offsets=None, saved=None, workspace=None,
                stream=None):
        """Write ``o``, and the sequences' last states to ``state_out`` if given
        (it may be ``state``, where they begin; without one, at zero).
        ``saved`` is written for a backward pass if given."""
        words = self._words(q=q, k=k, v=v, g=g, beta=beta, o=o)
        s = self._on(stream)
        io = self._forward_io.pack(*words, self._bounds(offsets), self._whole("state", state, "f32", self._state),
                                   self._whole("state_out", state_out, "f32", self._state), 0, 0, self._kept(saved))
        w, n = (None, 0) if saved is not None or not self._forward_bytes else self._workspace(s, False, workspace)
        rc = lib().cchip_gated_delta_forward(self._desc, io, w, n, s)
        if rc:
            check(rc)

    def backward(self, q, k, v, g, beta, do, saved, dq, dk, dv, dg, dbeta, *, dstate_out=None, dstate=None, offsets=None,
                 workspace=None, stream=None):
        """From the gradients of ``o`` and of the last states (None: zero) write
        those of q, k, v, g, beta, and of the first states to ``dstate`` if
        given. ``saved`` is what ``forward`` wrote for the same inputs."""
        if saved is None:
            raise ValueError("GatedDelta: the backward pass needs what the forward pass saved")
        words = self._words(q=q, k=k, v=v, g=g, beta=beta, do=do, dq=dq, dk=dk, dv=dv, dg=dg, dbeta=dbeta)
        s = self._on(stream)
        io = self._backward_io.pack(*words, self._bounds(offsets), 0, 0,
                                    self._whole("dstate_out", dstate_out, "f32", self._state),
                                    self._whole("dstate", dstate, "f32", self._state), self._kept(saved))
        check(lib().cchip_gated_delta_backward(self._desc, io, *self._workspace(s, True, workspace), s))


class Attention(_HeadOperator):
    """Causal attention over ``[batch, tokens, heads, head_dim]`` queries and
    ``[batch, tokens, kv_heads, head_dim]`` keys and values; heads ``h`` of
    ``heads`` go with key head ``h // (heads // kv_heads)``. scale is
    ``head_dim ** -0.5`` unless given.

    ``sequences``: that many sequences packed into a batch of 1, which every
    call says the bounds of (``offsets``, i32, ``sequences + 1`` values from 0
    to ``tokens``). ``keys``: k and v are caches of that many tokens a row, of
    which every call says how many they hold (``lengths``, i32, ``[batch]``),
    the queries' own ``tokens``, the last, among them: single tokens and
    chunks of a prompt. Without either, prompts and training."""

    _who = "Attention"
    # cchip_attention_io: eight cchip_heads of four words, three pointers
    _forward_io = struct.Struct("16q128x3q")
    _backward_io = struct.Struct("32q3q")

    def __init__(self, dtype, batch, tokens, heads, kv_heads, head_dim, scale=None, sequences=None, keys=None):
        super().__init__()
        _check_dtype("Attention", dtype)
        if sequences is not None and sequences < 1:
            raise ValueError("Attention: sequences must be >= 1")
        if keys is not None and keys < 1:
            raise ValueError("Attention: keys must be >= 1")
        self.dtype = dtype
        self._desc = _lib.AttentionDesc(CODES[dtype], batch, tokens, sequences or 0, keys or 0, heads, kv_heads, head_dim,
                                        head_dim ** -0.5 if scale is None and head_dim > 0 else scale or 0.0)
        sizes = [ctypes.c_size_t() for _ in range(3)]
        check(lib().cchip_attention_sizes(self._desc, *sizes))
        self._forward_bytes, self._backward_bytes, self._saved_bytes = (x.value for x in sizes)
        q, k = (batch, tokens, heads, head_dim), (batch, keys or tokens, kv_heads, head_dim)
        self._shapes = dict(q=q, o=q, do=q, dq=q, k=k, v=k, dk=k, dv=k)
        self._offsets = None if sequences is None else (sequences + 1,)
        self._lengths = None if keys is None else (batch,)

    def forward(self, q, k, v, o, *, offsets=None, lengths=None, saved=None, workspace=None, stream=None):
        """Write ``o``, and ``saved`` for a backward pass if given."""
        words = self._words(q=q, k=k, v=v, o=o)
        if (lengths is None) != (self._lengths is None):
            raise ValueError("Attention: a cache needs lengths" if lengths is None else "Attention: lengths without a cache")
        s = self._on(stream)
        io = self._forward_io.pack(*words, self._bounds(offsets), self._whole("lengths", lengths, "i32", self._lengths),
                                   self._kept(saved))
        w, n = self._workspace(s, False, workspace) if self._forward_bytes else (None, 0)
        rc = lib().cchip_attention_forward(self._desc, io, w, n, s)
        if rc:
            check(rc)

    def backward(self, q, k, v, o, do, saved, dq, dk, dv, *, offsets=None, workspace=None, stream=None):
        """From ``o`` and its gradient ``do`` write those of q, k and v. ``saved``
        is what ``forward`` wrote for the same inputs."""
        if self._lengths is not None:
            raise ValueError("Attention: there is no backward pass over a cache")
        if saved is None:
            raise ValueError("Attention: the backward pass needs what the forward pass saved")
        words = self._words(q=q, k=k, v=v, o=o, do=do, dq=dq, dk=dk, dv=dv)
        s = self._on(stream)
        io = self._backward_io.pack(*words, self._bounds(offsets), 0, self._kept(saved))
        check(lib().cchip_attention_backward(self._desc, io, *self._workspace(s, True, workspace), s))


class HeadNorm(_HeadOperator):
    """The norm of each head of q ``[batch, tokens, heads, head_dim]`` and k
    ``[batch, tokens, kv_heads, head_dim]`` ("rms", with a weight of
    ``head_dim`` for each of the two, or "none") and the rotation of its first
    ``rotary`` elements (all unless given) by the token's position: pairs are
    the halves of these or, ``interleaved``, neighbours.

    Every call is given the ``frequencies``, radians a position of each of the
    ``rotary // 2`` pairs (f32), and may be given ``positions`` (i32,
    ``[batch, tokens]``; without them rows count from 0). ``keys``: forward
    calls also write k and v to caches ``[batch, keys, kv_heads, head_dim]``
    at the tokens' positions (those outside the cache nowhere)."""

    _who = "HeadNorm"
    _io = struct.Struct("44q6q")  # cchip_head_norm_io: eleven cchip_heads, six pointers
    _NONE = (0, 0, 0, 0)

    def __init__(self, dtype, batch, tokens, heads, kv_heads, head_dim, norm="rms", rotary=None, interleaved=False, eps=1e-6,
                 weight_dtype="f32", keys=None):
        super().__init__()
        _check_dtype("HeadNorm", dtype, weight_dtype)
        if norm not in ("rms", "none"):
            raise ValueError("HeadNorm: unknown norm %r" % (norm,))
        if keys is not None and keys < 1:
            raise ValueError("HeadNorm: keys must be >= 1")
        self.dtype = dtype
        self.weight_dtype = weight_dtype
        rotary = head_dim // 2 * 2 if rotary is None else rotary
        self._desc = _lib.HeadNormDesc(CODES[dtype], CODES[weight_dtype], batch, tokens, keys or 0, heads, kv_heads, head_dim,
                                       rotary, 1 if interleaved else 0, NORMS[norm], eps)
        w = ctypes.c_size_t()
        check(lib().cchip_head_norm_workspace(self._desc, ctypes.byref(w)))
        self._backward_bytes = w.value
        q, k = (batch, tokens, heads, head_dim), (batch, tokens, kv_heads, head_dim)
        self._shapes = dict(q=q, q_out=q, dq_out=q, dq=q, k=k, v=k, k_out=k, dk_out=k, dk=k)
        self._cache = keys is not None
        if self._cache:
            self._shapes["k_cache"] = self._shapes["v_cache"] = (batch, keys, kv_heads, head_dim)
        self._positions = (batch, tokens)
        self._frequencies = (rotary // 2,)
        self._vector = (head_dim,)

    def reserve(self, stream=None):
        """Allocate a stream's workspace ahead of the first backward call on it."""
        self._workspace(self._on(stream), True)

    def _tables(self, frequencies, positions, q_weight, k_weight):
        return (self._whole("positions", positions, "i32", self._positions),
                self._whole("frequencies", frequencies, "f32", self._frequencies),
                self._whole("q_weight", q_weight, self.weight_dtype, self._vector),
                self._whole("k_weight", k_weight, self.weight_dtype, self._vector))

    def forward(self, q, k, q_out, k_out=None, *, frequencies=None, positions=None, q_weight=None, k_weight=None, v=None,
                k_cache=None, v_cache=None, stream=None):
        """Write ``q_out`` and ``k_out``, which may be q and k; with caches those
        are written from k and ``v``, and k_out need not be given."""
        none = self._NONE
        if self._cache:
            words = self._words(q=q, k=k, v=v, q_out=q_out)
            out = self._words(k_out=k_out) if k_out is not None else none
            io = self._io.pack(*words, *out, *self._words(k_cache=k_cache, v_cache=v_cache), *none, *none, *none, *none,
                               *self._tables(frequencies, positions, q_weight, k_weight), 0, 0)
        else:
            if not v is k_cache is v_cache is None:
                raise ValueError("HeadNorm: a cache for an operator made without keys")
            words = self._words(q=q, k=k)
            io = self._io.pack(*words, *none, *self._words(q_out=q_out, k_out=k_out), *none, *none, *none, *none, *none, *none,
                               *self._tables(frequencies, positions, q_weight, k_weight), 0, 0)
        rc = lib().cchip_head_norm_forward(self._desc, io, self._on(stream))
        if rc:
            check(rc)

    def backward(self, q, k, dq_out, dk_out, dq, dk, *, frequencies=None, positions=None, q_weight=None, k_weight=None,
                 grads=None, workspace=None, stream=None):
        """From q, k and the gradients of what ``forward`` wrote the gradients of
        q and k (they may be ``dq_out`` and ``dk_out``) and, for each name in
        ``grads`` ("q_weight", "k_weight"), of that weight, summed over tokens
        and heads."""
        none, s = self._NONE, self._on(stream)
        grads = grads or {}
        for n in grads:
            if n not in ("q_weight", "k_weight"):
                raise ValueError("HeadNorm: unknown parameter %s" % n)
        words = self._words(q=q, k=k), self._words(dq_out=dq_out, dk_out=dk_out, dq=dq, dk=dk)
        io = self._io.pack(*words[0], *none, *none, *none, *none, *none, *words[1],
                           *self._tables(frequencies, positions, q_weight, k_weight),
                           *(self._whole(n, grads.get(n), self.weight_dtype, self._vector) for n in ("q_weight", "k_weight")))
        w, n = self._workspace(s, True, workspace) if grads else (None, 0)
        check(lib().cchip_head_norm_backward(self._desc, io, w, n, s))


class _RowOperator(_Operator):
    def _rows(self, name, x):
        """An array's pointer and the distance of its rows; zeros for None."""
        if x is None:
            return _NO_ROWS
        try:
            st = x.stride()
            plain = x.shape == self._shape and _dtypes[x.dtype] == self.dtype and x.get_device() == self._device
            p = x.data_ptr()
        except (AttributeError, KeyError):
            plain = False
        if not plain:
            p, st = self._view(name, x, self.dtype, self._shape)
        if st[1] != 1 and self._shape[1] > 1:
            raise ValueError("%s: rows of %s are not contiguous" % (self._who, name))
        return p, st[0]

    def _needed(self, name, x):
        if x is None:
            raise ValueError("%s: no %s" % (self._who, name))
        return self._rows(name, x)

    def _seed(self, seed, offset, step):
        return (seed & 0xFFFFFFFFFFFFFFFF, offset & 0xFFFFFFFFFFFFFFFF,
                0 if step is None else self._whole("step", step, "i64", ()))


class Embedding(_RowOperator):
    """Rows of a table ``[vocab, width]`` by the tokens' ``ids`` (i32,
    ``[tokens]``), times ``scale``, and the table's gradient. Ids outside 0 ..
    vocab - 1 have rows of zeros and no gradient. The table and its gradient
    are of ``weight_dtype`` ("f32" or ``dtype``, which it is unless given)."""

    _who = "Embedding"
    _io = struct.Struct("10q")  # cchip_embedding_io

    def __init__(self, dtype, tokens, vocab, width, scale=1.0, weight_dtype=None):
        super().__init__()
        weight_dtype = weight_dtype or dtype
        _check_dtype("Embedding", dtype, weight_dtype)
        self.dtype = dtype
        self.weight_dtype = weight_dtype
        self._desc = _lib.EmbeddingDesc(CODES[dtype], CODES[weight_dtype], tokens, vocab, width, scale)
        w = ctypes.c_size_t()
        check(lib().cchip_embedding_workspace(self._desc, ctypes.byref(w)))
        self._backward_bytes = w.value
        self._ids = (tokens,)
        self._shape = (tokens, width)
        self._table = (vocab, width)

    def reserve(self, stream=None):
        """Allocate a stream's workspace ahead of the first backward call on it."""
        self._workspace(self._on(stream), True)

    def _words_of(self, ids):
        if ids is None:
            raise ValueError("Embedding: no ids")
        return self._whole("ids", ids, "i32", self._ids)

    def _table_of(self, name, x):
        p, st = self._view(name, x, self.weight_dtype, self._table)
        if st[1] != 1 and self._table[1] > 1:
            raise ValueError("Embedding: rows of %s are not contiguous" % name)
        return p, st[0]

    def forward(self, ids, weight, out, *, stream=None):
        """``out[t] = scale weight[ids[t]]``."""
        io = self._io.pack(self._words_of(ids), *self._table_of("weight", weight), *self._needed("out", out), 0, 0, 0, 0, 0)
        rc = lib().cchip_embedding_forward(self._desc, io, self._on(stream))
        if rc:
            check(rc)

    def backward(self, ids, dout, dweight, *, accumulate=False, workspace=None, stream=None):
        """Write the table's gradient, of all words, or with ``accumulate`` add
        to the rows of those there are."""
        s = self._on(stream)
        io = self._io.pack(self._words_of(ids), 0, 0, 0, 0, *self._needed("dout", dout), *self._table_of("dweight", dweight),
                           1 if accumulate else 0)
        check(lib().cchip_embedding_backward(self._desc, io, *self._workspace(s, True, workspace), s))


def _check_p(who, p):
    if not 0.0 <= p <= 1.0:
        raise ValueError("%s: p = %r is not in 0 .. 1" % (who, p))


class Dropout(_RowOperator):
    """Dropout of ``[rows, cols]`` arrays by the counter-based generator, its
    mask drawn when needed and never stored: the same ``seed`` and ``offset``
    give the same mask. ``step``, an i64 array without dimensions, is added
    to ``offset`` on the device."""

    _who = "Dropout"
    _io = struct.Struct("3Q6q")  # cchip_dropout_io

    def __init__(self, dtype, rows, cols, p, scale=1.0):
        super().__init__()
        _check_dtype("Dropout", dtype)
        _check_p("Dropout", p)
        self.dtype = dtype
        self._desc = _lib.DropoutDesc(CODES[dtype], rows, cols, p, scale)
        self._shape = (rows, cols)

    def forward(self, x, out, *, seed, offset=0, residual=None, step=None, stream=None):
        """``out = residual + scale drop(x)``; out may be x or residual."""
        io = self._io.pack(*self._seed(seed, offset, step), *self._needed("x", x), *self._rows("residual", residual),
                           *self._needed("out", out))
        check(lib().cchip_dropout_run(self._desc, io, self._on(stream)))

    def backward(self, dout, dx, *, seed, offset=0, step=None, stream=None):
        """``dx = scale drop(dout)`` with the forward pass's mask; the residual's
        gradient is ``dout`` itself."""
        self.forward(dout, dx, seed=seed, offset=offset, step=step, stream=stream)


_PARAMS = {"post_weight": 0, "post_bias": 1, "channel_scale": 2, "pre_weight": 3, "pre_bias": 4}


class NormBlock(_RowOperator):
    """What stands between a block's output ``y`` and the next block's input,
    on each row: ``h = residual + scale channel_scale drop(norm(y) act(gate))``
    and ``n = norm(h)``, each norm with a weight and a bias.

    ``norm`` and ``pre`` (the norm of h): "rms", "layer" or "none"; ``gate``:
    "silu", "sigmoid" or "none". Parameters are vectors of ``width`` of
    ``weight_dtype`` ("f32" or ``dtype``); one that is not given is 1 or 0."""

    _who = "NormBlock"
    _io = struct.Struct("3Q10q20q")  # cchip_norm_block_io

    def __init__(self, dtype, rows, width, norm="rms", pre="rms", gate="none", dropout=0.0, scale=1.0, eps=1e-6,
                 weight_dtype="f32"):
        super().__init__()
        _check_dtype("NormBlock", dtype, weight_dtype)
        _check_p("NormBlock", dropout)
        if norm not in NORMS or pre not in NORMS or gate not in GATES:
            raise ValueError("NormBlock: unknown norm %r, pre %r or gate %r" % (norm, pre, gate))
        self.dtype = dtype
        self.weight_dtype = weight_dtype
        self._shape = (rows, width)
        self._vector = (width,)
        self._desc = _lib.NormBlockDesc(CODES[dtype], CODES[weight_dtype], rows, width, NORMS[norm], NORMS[pre], GATES[gate],
                                        scale, eps, dropout)
        w = ctypes.c_size_t()
        check(lib().cchip_norm_block_workspace(self._desc, ctypes.byref(w)))
        self._backward_bytes = w.value

    def reserve(self, stream=None):
        """Allocate a stream's workspace ahead of the first backward call on it."""
        self._workspace(self._on(stream), True)

    def _vectors(self, given):
        p = [0, 0, 0, 0, 0]
        for n, x in given.items():
            if n not in _PARAMS:
                raise ValueError("NormBlock: unknown parameter %s" % n)
            p[_PARAMS[n]] = self._whole(n, x, self.weight_dtype, self._vector)
        return p

    def forward(self, y, h, n=None, *, gate=None, residual=None, seed=0, offset=0, step=None, stream=None, **params):
        """Write ``h``, and ``n`` if there is a norm of it. h may be residual or
        y, n may be y. ``params``: post_weight, post_bias, channel_scale,
        pre_weight, pre_bias. ``seed``, ``offset`` and ``step`` as for Dropout."""
        io = self._io.pack(*self._seed(seed, offset, step), *self._vectors(params), 0, 0, 0, 0, 0,
                           *self._needed("y", y), *self._rows("gate", gate), *self._rows("residual", residual),
                           *self._needed("h", h), *self._rows("n", n), 0, 0, 0, 0, 0, 0, 0, 0, 0, 0)
        check(lib().cchip_norm_block_forward(self._desc, io, self._on(stream)))

    def backward(self, y, dh, dy, *, dn=None, h=None, gate=None, dgate=None, dresidual=None, grads=None, seed=0, offset=0,
                 step=None, workspace=None, stream=None, **params):
        """From y, gate, the forward pass's h (where it is normed again) and the
        gradients of h and n, write those of y, gate and residual and, for each
        name in ``grads``, of that parameter, summed over the rows."""
        s = self._on(stream)
        io = self._io.pack(*self._seed(seed, offset, step), *self._vectors(params), *self._vectors(grads or {}),
                           *self._needed("y", y), *self._rows("gate", gate), 0, 0, *self._rows("h", h), 0, 0,
                           *self._needed("dh", dh), *self._rows("dn", dn), *self._needed("dy", dy),
                           *self._rows("dgate", dgate), *self._rows("dresidual", dresidual))
        w, n = self._workspace(s, True, workspace) if grads else (None, 0)
        check(lib().cchip_norm_block_backward(self._desc, io, w, n, s))
