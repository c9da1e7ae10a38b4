"""The layer operators without a device: the ABI, what the handles refuse, the
generator against the array DSL's, and the 64-bit references' gradients
against differences."""

import ctypes
import os
import re
import subprocess

import numpy as np
import pytest
import torch

import operator_reference as R
from cudacaml_amd import _lib
from cudacaml_amd import operators as O

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "cchip_operators.h")


def test_every_declared_operator_is_exported_and_bound():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = {m.group(1) for m in re.finditer(r"\b(cchip_[a-z_0-9]+)\s*\(", text)}
    assert names == set(_lib.OPERATOR_SIGNATURES)
    lib = ctypes.CDLL(_lib.LIB_PATH)
    assert not [n for n in names if not hasattr(lib, n)]


def test_structures_have_the_headers_sizes(tmp_path):
    """The header is strict C99, and what Python packs is what C reads."""
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "cchip_operators.h"\n'
                   "int main(void) { printf(\"%zu %zu %zu %zu %zu %zu %zu\\n\", sizeof(cchip_gated_delta), "
                   "sizeof(cchip_gated_delta_io), offsetof(cchip_gated_delta_io, offsets), sizeof(cchip_dropout), "
                   "sizeof(cchip_dropout_io), sizeof(cchip_norm_block), sizeof(cchip_norm_block_io)); return 0; }\n")
    exe = str(tmp_path / "sizes")
    subprocess.run(["gcc", "-std=c99", "-pedantic", "-Wall", "-Wextra", "-Werror", "-I" + os.path.join(ROOT, "include"),
                    "-o", exe, str(src)], check=True)
    got = [int(x) for x in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(_lib.GatedDeltaDesc), O.GatedDelta._forward_io.size, 12 * 32,
                   ctypes.sizeof(_lib.DropoutDesc), O.Dropout._io.size, ctypes.sizeof(_lib.NormBlockDesc),
                   O.NormBlock._io.size]
    assert O.GatedDelta._backward_io.size == O.GatedDelta._forward_io.size


BAD_DELTA = [
    (dict(dtype="f64"), "dtype"),
    (dict(key_heads=3), "multiple"),
    (dict(key_heads=0), "multiple"),
    (dict(key_dim=129), "key_dim"),
    (dict(key_dim=0), "key_dim"),
    (dict(value_dim=0), "value_dim"),
    (dict(value_dim=4097), "value_dim"),
    (dict(batch=-1), "negative"),
    (dict(tokens=1 << 31), "2\\^31"),
    (dict(sequences=2), "batch of 1"),
    (dict(sequences=0), "sequences"),
    (dict(scale=float("nan")), "finite"),
    (dict(batch=1 << 30, tokens=1 << 20), "launch"),
]


@pytest.mark.parametrize("change,why", BAD_DELTA)
def test_gated_delta_refuses_its_shapes(change, why):
    shape = dict(dtype="bf16", batch=2, tokens=100, key_heads=2, value_heads=4, key_dim=64, value_dim=64)
    O.GatedDelta(**shape)
    with pytest.raises(ValueError, match=why):
        O.GatedDelta(**{**shape, **change})


def test_sizes_grow_with_what_is_kept():
    a = O.GatedDelta("bf16", 1, 640, 2, 4, 64, 64)
    b = O.GatedDelta("bf16", 1, 1280, 2, 4, 64, 64)
    assert b.saved_bytes() == 2 * a.saved_bytes() > 0
    # a step needs no workspace, and packed sequences a slot each at the most
    assert O.GatedDelta("bf16", 7, 8, 2, 4, 64, 64)._forward_bytes == 0
    one = O.GatedDelta("bf16", 1, 64, 2, 4, 64, 64).saved_bytes()
    assert O.GatedDelta("bf16", 1, 640, 2, 4, 64, 64, sequences=3).saved_bytes() == 13 * one


def _delta_arrays(b=2, t=10, hk=2, hv=4, dk=16, dv=8, dtype=torch.float32):
    z = lambda *s: torch.zeros(s, dtype=dtype)  # noqa: E731
    return dict(q=z(b, t, hk, dk), k=z(b, t, hk, dk), v=z(b, t, hv, dv), g=z(b, t, hv), beta=z(b, t, hv), o=z(b, t, hv, dv))


@pytest.mark.parametrize("name,bad,why", [
    ("q", torch.zeros(2, 10, 2, 8), "shape"),
    ("v", torch.zeros(2, 10, 4, 8, dtype=torch.float64), "dtype"),
    ("k", torch.zeros(2, 10, 16, 2).transpose(2, 3), "contiguous"),
    ("g", torch.zeros(2, 10, 4), "device"),
])
def test_gated_delta_refuses_arrays(name, bad, why):
    """Wrong shapes, types and strides, and memory of the host, which the
    operator must never hand to a kernel."""
    op = O.GatedDelta("f32", 2, 10, 2, 4, 16, 8)
    x = _delta_arrays()
    op._device = -1 if why != "device" else 0  # as if these were the device's
    x[name] = bad
    with pytest.raises(ValueError, match=why):
        op.forward(*x.values())


def test_gated_delta_refuses_calls():
    x = _delta_arrays()
    op = O.GatedDelta("f32", 2, 10, 2, 4, 16, 8, states=False)
    op._device = -1
    grads = [x[n] for n in ("q", "k", "v", "g", "beta")]
    with pytest.raises(ValueError, match="saved"):
        op.backward(*grads, x["o"], None, *grads)
    with pytest.raises(ValueError, match="offsets"):
        op.forward(*x.values(), offsets=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="shape"):
        op.forward(*x.values(), saved=torch.zeros(16, dtype=torch.uint8))
    packed = O.GatedDelta("f32", 1, 10, 2, 4, 16, 8, sequences=3)
    packed._device = -1
    with pytest.raises(ValueError, match="offsets"):
        packed.forward(*_delta_arrays(b=1).values())


def _call(fn, *args):
    rc = fn(*args)
    return rc, _lib.lib().cchip_last_error().decode()


def test_c_entries_refuse_before_any_device_work():
    """Null pointers, misaligned and overlapping tensors, states that the
    operator was made without, and a workspace that is too small."""
    L = _lib.lib()
    d = _lib.GatedDeltaDesc(0, 2, 100, 0, 2, 4, 16, 8, 0, 1.0)
    F = O.GatedDelta._forward_io
    t = lambda p=4096, h=8: (p, 100 * 4 * h, 4 * h, h)  # noqa: E731
    good = [*t(h=16), *t(h=16), *t(), *t(h=1), *t(h=1), *t()]

    def forward(words, tail=(0,) * 6, ws=None, n=0, desc=d):
        return _call(L.cchip_gated_delta_forward, desc, F.pack(*words, *tail), ws, n, None)

    rc, msg = forward(good)
    assert rc == 1 and re.match(r"gated delta: the workspace needs \d+ bytes aligned to 16, has 0$", msg)
    for at, value, why in [(0, 0, "no q"), (8, 4098, "v is not aligned"), (21, 0, "o overlap"), (22, 0, "o overlap"),
                           (23, 4, "o overlap"), (6, 1 << 24, "tokens of k"), (2, -64, "tokens of q")]:
        words = list(good)
        words[at] = value
        rc, msg = forward(words)
        assert rc == 1 and why in msg, (at, msg)
    rc, msg = forward(good, tail=(0, 4096, 0, 0, 0, 0))
    assert rc == 1 and "without states" in msg
    rc, msg = forward(good, tail=(4096, 0, 0, 0, 0, 0))
    assert rc == 1 and "offsets without packed" in msg
    rc, msg = forward(good, tail=(0, 0, 0, 0, 0, 4100))
    assert rc == 1 and "saved is not aligned" in msg
    rc, msg = _call(L.cchip_gated_delta_backward, d, bytes(F.size), None, 0, None)
    assert rc == 1
    rc, msg = _call(L.cchip_gated_delta_forward, None, None, None, 0, None)
    assert rc == 1 and "no descriptor" in msg


def test_gated_delta_refuses_results_that_share_elements():
    """Against all heads written out, for strides of all orders: what is
    refused does overlap, and what is taken does not but by several steps along
    one axis against several along others."""
    L, F = _lib.lib(), O.GatedDelta._forward_io
    b, t, h, dv = 2, 3, 4, 5
    d = _lib.GatedDeltaDesc(0, b, t, 0, 1, h, 5, dv, 0, 1.0)
    x = lambda at, n: (at << 20, 3 * n, n, dv if n > h else 1)  # noqa: E731
    ins = [*x(1, dv), *x(2, dv), *x(3, h * dv), *x(4, h), *x(5, h)]
    rng, refused, taken = np.random.default_rng(5), 0, 0
    steps = [(60, 20, 5), (15, 5, 30), (20, 40, 5), (60, 20, -5), (60, 19, 5), (5, 10, 30), (100, 0, 5), (100, 33, 11), (40, 60, 10)]
    steps += [tuple(int(v) for v in rng.integers(0, 70, 3)) for _ in range(300)]
    for s in steps:
        heads = np.add.outer(np.add.outer(np.arange(b) * s[0], np.arange(t) * s[1]), np.arange(h) * s[2]).ravel()
        gaps = np.diff(np.sort(heads))
        # `saved` off its alignment: what is taken is refused for that
        rc, msg = _call(L.cchip_gated_delta_forward, d, F.pack(*ins, 6 << 20, *s, 0, 0, 0, 0, 0, 4100), None, 0, None)
        assert rc == 1
        if "overlap" in msg:
            refused += 1
            assert (gaps < dv).any(), s
        else:
            taken += 1
            assert "saved is not aligned" in msg
            if (gaps < dv).any():
                assert all(abs(v) >= dv for v in s), s
    assert refused > 50 and taken > 5


def test_gated_delta_refuses_misaligned_words():
    L = _lib.lib()
    t = lambda p, h=8: (p << 20, 100 * 4 * h, 4 * h, h)  # noqa: E731
    some = [w for i, h in enumerate((8, 8, 8, 1, 1, 8)) for w in t(i + 1, h)]
    for sequences, tail, why in [(0, (0, 4098, 0, 0, 0, 4096), "state is"), (0, (0, 0, 4097, 0, 0, 4096), "state_out is"),
                                 (1, (4098, 0, 0, 0, 0, 4096), "offsets is")]:
        d = _lib.GatedDeltaDesc(0, 1, 100, sequences, 4, 4, 8, 8, 1, 1.0)
        rc, msg = _call(L.cchip_gated_delta_forward, d, O.GatedDelta._forward_io.pack(*some, *tail), None, 0, None)
        assert rc == 1 and why + " not aligned" in msg, msg
    back = [w for i, h in enumerate((8, 8, 8, 1, 1)) for w in t(i + 1, h)] + [w for i, h in enumerate((8, 8, 8, 8, 1, 1)) for w in t(i + 7, h)]
    d = _lib.GatedDeltaDesc(0, 1, 100, 0, 4, 4, 8, 8, 1, 1.0)
    for tail, why in [((0, 0, 0, 4098, 0, 4096), "dstate_out is"), ((0, 0, 0, 0, 4099, 4096), "dstate is")]:
        rc, msg = _call(L.cchip_gated_delta_backward, d, O.GatedDelta._backward_io.pack(*back, *tail), None, 0, None)
        assert rc == 1 and why + " not aligned" in msg, msg


def test_nothing_to_do_is_no_error():
    """No rows, no columns, no sequences: no launch, so no device is needed."""
    L = _lib.lib()
    d = _lib.GatedDeltaDesc(0, 0, 100, 0, 2, 4, 16, 8, 1, 1.0)
    assert _call(L.cchip_gated_delta_forward, d, bytes(O.GatedDelta._forward_io.size), None, 0, None)[0] == 0
    assert _call(L.cchip_dropout_run, _lib.DropoutDesc(0, 0, 7, 0.5, 1.0), bytes(O.Dropout._io.size), None)[0] == 0
    n = _lib.NormBlockDesc(0, 0, 0, 8, 1, 1, 0, 1.0, 1e-6, 0.0)
    assert _call(L.cchip_norm_block_forward, n, bytes(O.NormBlock._io.size), None)[0] == 0


@pytest.mark.parametrize("kw,why", [
    (dict(dtype="i32"), "dtype"), (dict(weight_dtype="f16"), "parameters"), (dict(width=0), "width"),
    (dict(width=32769), "width"), (dict(rows=1 << 32), "rows"), (dict(norm="batch"), "unknown"),
    (dict(gate="tanh"), "unknown"), (dict(dropout=1.5), "not in 0"), (dict(dropout=float("nan")), "not in 0"),
    (dict(eps=-1.0), "eps"), (dict(scale=float("inf")), "finite"),
])
def test_norm_block_refuses_its_shapes(kw, why):
    with pytest.raises(ValueError, match=why):
        O.NormBlock(**{**dict(dtype="bf16", rows=4, width=8), **kw})


def test_norm_block_refuses_calls():
    z = lambda *s: torch.zeros(s)  # noqa: E731
    op = O.NormBlock("f32", 4, 8)
    op._device = -1
    with pytest.raises(ValueError, match="if and only if"):
        op.forward(z(4, 8), z(4, 8))
    with pytest.raises(ValueError, match="a gate is given"):
        op.forward(z(4, 8), z(4, 8), z(4, 8), gate=z(4, 8))
    with pytest.raises(ValueError, match="unknown parameter"):
        op.forward(z(4, 8), z(4, 8), z(4, 8), weight=z(8))
    with pytest.raises(ValueError, match="rows of y are not contiguous"):
        op.forward(z(8, 4).t(), z(4, 8), z(4, 8))
    with pytest.raises(ValueError, match="rows of h overlap"):
        op.forward(z(4, 8), z(1, 8).expand(4, 8), z(4, 8))
    with pytest.raises(ValueError, match="h and dn"):
        op.backward(z(4, 8), z(4, 8), z(4, 8))
    dh = z(4, 8)
    with pytest.raises(ValueError, match="written over"):
        op.backward(z(4, 8), dh, dh, dn=z(4, 8), h=z(4, 8))
    plain = O.NormBlock("f32", 4, 8, norm="none", pre="none")
    plain._device = -1
    with pytest.raises(ValueError, match="post norm that there is not"):
        plain.forward(z(4, 8), z(4, 8), post_weight=z(8))
    with pytest.raises(ValueError, match="gate that there is not"):
        plain.backward(z(4, 8), z(4, 8), z(4, 8), dgate=z(4, 8))


def test_dropout_refuses():
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError, match="not in 0"):
            O.Dropout("f32", 4, 8, p)
    op = O.Dropout("f32", 4, 8, 0.5)
    op._device = -1
    with pytest.raises(ValueError, match="no out"):
        op.forward(torch.zeros(4, 8), None, seed=1)
    with pytest.raises(ValueError, match="rows of out overlap"):
        op.forward(torch.zeros(4, 8), torch.zeros(1, 8).expand(4, 8), seed=1)


def test_rows_are_written_in_place_row_for_row_only():
    """A result over an input by other strides or a few elements on would be
    read by threads after others wrote it; h and n have a place each."""
    z = lambda *s: torch.zeros(s)  # noqa: E731
    op = O.Dropout("f32", 4, 8, 0.5)
    op._device = -1
    w = z(200)
    at = lambda first, row: w.as_strided((4, 8), (row, 1), first)  # noqa: E731
    for out in (at(0, 9), at(3, 8), at(7, 8)):
        with pytest.raises(ValueError, match="out is written over x, and not row for row"):
            op.forward(at(0, 8), out, seed=1)
        with pytest.raises(ValueError, match="out is written over residual"):
            op.forward(z(4, 8), out, residual=at(0, 8), seed=1)
    op = O.NormBlock("f32", 4, 8, gate="silu")
    op._device = -1
    with pytest.raises(ValueError, match="h is written over residual"):
        op.forward(z(4, 8), at(0, 9), z(4, 8), gate=z(4, 8), residual=at(0, 8))
    with pytest.raises(ValueError, match="n is written over y"):
        op.forward(at(4, 8), z(4, 8), at(0, 8), gate=z(4, 8))
    with pytest.raises(ValueError, match="n is written over h"):
        op.forward(z(4, 8), at(0, 8), at(0, 8), gate=z(4, 8))
    back = dict(dn=z(4, 8), h=z(4, 8), gate=z(4, 8))
    with pytest.raises(ValueError, match="dgate is written over dy"):
        op.backward(z(4, 8), z(4, 8), at(0, 8), dgate=at(0, 8), **back)
    with pytest.raises(ValueError, match="dresidual is written over h"):
        op.backward(z(4, 8), z(4, 8), z(4, 8), dresidual=at(5, 8), **{**back, "h": at(0, 8)})


def test_what_is_no_array_is_refused():
    """None, and arrays of the host, by name."""
    delta, block, drop = O.GatedDelta("f32", 2, 10, 2, 4, 16, 8), O.NormBlock("f32", 4, 8), O.Dropout("f32", 4, 8, 0.5)
    for op in (delta, block, drop):
        op._device = -1
    x = _delta_arrays()
    z = torch.zeros(4, 8)
    for name in x:
        with pytest.raises(ValueError, match="GatedDelta: no %s$" % name):
            delta.forward(*{**x, name: None}.values())
        with pytest.raises(ValueError, match="GatedDelta: %s is no array on a device" % name):
            delta.forward(*{**x, name: x[name].numpy()}.values())
    with pytest.raises(ValueError, match="no array on a device"):
        delta.forward(*x.values(), state=np.zeros((2, 4, 16, 8), np.float32))
    with pytest.raises(ValueError, match="NormBlock: no y"):
        block.forward(None, z, z.clone())
    with pytest.raises(ValueError, match="NormBlock: h is no array on a device"):
        block.forward(z, z.numpy(), z.clone())
    with pytest.raises(ValueError, match="Dropout: x is no array on a device"):
        drop.forward(z.numpy(), z, seed=1)


def test_a_call_on_another_device_is_refused(monkeypatch):
    """The arrays are on the handle's device; kernels would run on the one
    that is current."""
    now = [-1]
    monkeypatch.setattr(O.Device, "available", staticmethod(lambda: True))
    monkeypatch.setattr(O.Device, "count", staticmethod(lambda: 2))
    monkeypatch.setattr(O.Device, "current", staticmethod(lambda: now[0]))
    op = O.Dropout("f32", 4, 8, 0.5)  # on device -1, where the host's tensors are
    assert op._on(5) == 5
    now[0] = 3
    with pytest.raises(ValueError, match="made for device -1, called on device 3"):
        op.forward(torch.zeros(4, 8), torch.zeros(4, 8), seed=1)


def test_arrays_lie_in_their_buffers():
    class Memory:
        ptr, nbytes = 4096, 64

    O.Array(Memory(), "f32", (4, 4))
    O.Array(Memory(), "bf16", (4, 4), strides=(8, 1), first=4)
    with pytest.raises(ValueError, match="do not lie"):
        O.Array(Memory(), "f32", (4, 5))
    with pytest.raises(ValueError, match="do not lie"):
        O.Array(Memory(), "f32", (2, 4), strides=(-4, 1))
    with pytest.raises(ValueError, match="unknown dtype"):
        O.Array(Memory(), "f8", (4, 4))


def test_the_generator_is_the_array_languages():
    """Words of the mask's generator against ``rng.round10`` as a graph, on the
    interpreter: the same rounds, constants and key schedule."""
    import oracle
    from cudacaml_amd import dsl as D
    from cudacaml_amd import rng
    from cudacaml_amd.ir import I32, Graph

    seed, offset, row = 0x123456789ABCDEF, 0xFEDCBA9876543210, 77

    def word(i):
        c = lambda x: D.const(I32, int(np.uint32(x).astype(np.int32)))  # noqa: E731
        ctr = (lambda g: (g, c(row), c(offset & R.LOW), c(offset >> 32)))
        return D.map(lambda g: rng.round10(ctr(g), (c(seed & R.LOW), c(seed >> 32)))[i], D.iota((9,)))

    g = Graph.create("words", [("w%d" % i, word(i)) for i in range(4)])
    got = dict(oracle.Interp.run(oracle.Interp.compile(g), []))
    for group in range(9):
        want = R.philox((group, row, offset & R.LOW, offset >> 32), (seed & R.LOW, seed >> 32))
        assert [int(got["w%d" % i][group]) & R.LOW for i in range(4)] == want


def _difference(f, x, direction, eps=1e-5):
    return (f(x + eps * direction) - f(x - eps * direction)) / (2 * eps)


def test_reference_gradients_against_differences():
    """The references' hand-made gradients in 64 bits: a central difference of
    step 1e-5 is off by about 1e-10 of the value for functions of these sizes,
    and rounding by 1e-11; 1e-6 leaves room for their condition."""
    g = np.random.default_rng(3)
    x = dict(q=g.standard_normal((7, 2, 5)), k=g.standard_normal((7, 2, 5)) / 3, v=g.standard_normal((7, 4, 3)),
             g=-g.random((7, 4)), beta=g.random((7, 4)), state=g.standard_normal((4, 5, 3)))
    do, ds = g.standard_normal((7, 4, 3)), g.standard_normal((4, 5, 3))

    def loss(**kw):
        y = {**x, **kw}
        o, s = R.delta(y["q"], y["k"], y["v"], y["g"], y["beta"], 0.3, y["state"])
        return (o * do).sum() + (s * ds).sum()

    d = R.delta(x["q"], x["k"], x["v"], x["g"], x["beta"], 0.3, x["state"], do, ds)[2]
    for n in x:
        r = g.standard_normal(x[n].shape)
        want = _difference(lambda a: loss(**{n: a}), x[n], r)
        assert abs((d["d" + n] * r).sum() - want) < 1e-6 * max(1.0, abs(want)), n

    for post, pre, gate in (("rms", "layer", "silu"), ("layer", "rms", "sigmoid"), ("none", "none", "none")):
        y = dict(y=g.standard_normal((3, 9)), residual=g.standard_normal((3, 9)), channel_scale=g.standard_normal(9))
        if gate != "none":
            y["gate"] = g.standard_normal((3, 9))
        if post != "none":
            y.update(post_weight=g.standard_normal(9), post_bias=g.standard_normal(9))
        if pre != "none":
            y.update(pre_weight=g.standard_normal(9), pre_bias=g.standard_normal(9))
        dh, dn = g.standard_normal((3, 9)), g.standard_normal((3, 9))
        how = (post, pre, gate, 0.7, 1e-3, 0.3, 5, 6)

        def loss(**kw):
            out = R.norm_block({**y, **kw}, *how)
            return (out["h"] * dh).sum() + ((out["n"] * dn).sum() if pre != "none" else 0.0)

        d = R.norm_block({**y, "h": R.norm_block(y, *how)["h"], "dh": dh, "dn": dn}, *how, back=True)
        for n in y:
            r = g.standard_normal(y[n].shape)
            want = _difference(lambda a: loss(**{n: a}), y[n], r)
            assert abs((d[n] * r).sum() - want) < 1e-6 * max(1.0, abs(want)), (post, n)


def test_backward_of_no_sequences_is_no_error():
    """A batch of none has nothing saved, and its backward pass nothing to do.
    Where there are chunks, what the forward pass saved is still asked for."""
    L, sizes = _lib.lib(), [ctypes.c_size_t() for _ in range(3)]
    io = bytes(O.GatedDelta._backward_io.size)
    none = _lib.GatedDeltaDesc(0, 0, 100, 0, 2, 4, 16, 8, 1, 1.0)
    assert L.cchip_gated_delta_sizes(none, *sizes) == 0 and [s.value for s in sizes] == [0, 0, 0]
    assert _call(L.cchip_gated_delta_backward, none, io, None, 0, None)[0] == 0
    t = lambda h=8: (4096, 100 * 4 * h, 4 * h, h)  # noqa: E731
    some = _lib.GatedDeltaDesc(0, 2, 100, 0, 4, 4, 8, 8, 1, 1.0)
    words = [*t(), *t(), *t(), *t(1), *t(1), *[w for h in (8, 8, 8, 8, 1, 1) for w in t(h)], *(0,) * 6]
    rc, msg = _call(L.cchip_gated_delta_backward, some, O.GatedDelta._backward_io.pack(*words), None, 0, None)
    assert rc == 1 and "what the forward pass saved" in msg


def test_gated_delta_refuses_to_write_over_what_it_reads():
    """Other workgroups and later kernels read q, k, v, g, beta and the
    gradient of o after the first results are written."""
    x = _delta_arrays(t=100)
    op = O.GatedDelta("f32", 2, 100, 2, 4, 16, 8, states=False)
    op._device = -1
    names = ("q", "k", "v", "g", "beta")
    ins = [x[n] for n in names]

    def room(n):
        whole = torch.zeros(n + 16, dtype=torch.uint8)
        return whole[-whole.data_ptr() % 16:][:n]

    work, saved = room(op.workspace_bytes(backward=True)), room(op.saved_bytes())
    with pytest.raises(ValueError, match="o is written over v, which"):
        op.forward(*ins, x["v"], saved=saved)
    with pytest.raises(ValueError, match="o is written over v, which"):
        _one_token(op).forward(*(t[:, :1] for t in ins), x["v"][:, :1])

    def backward(workspace=work, **over):
        grads = {n: over.get(n, torch.zeros_like(x[n])) for n in names}
        op.backward(*ins, x["o"], saved, *grads.values(), workspace=workspace)

    for n in names:
        with pytest.raises(ValueError, match="d%s is written over %s, which" % (n, n)):
            backward(**{n: x[n]})
    with pytest.raises(ValueError, match="dv is written over the gradient of o"):
        backward(v=x["o"])
    z = torch.zeros_like(x["k"])
    with pytest.raises(ValueError, match="dq and dk are written to one place"):
        backward(q=z, k=z)
    big = room(max(op.workspace_bytes(backward=True), op.saved_bytes()))
    saved = big[:op.saved_bytes()]
    with pytest.raises(ValueError, match="the workspace is what"):
        backward(workspace=big)


def _one_token(op):
    one = O.GatedDelta("f32", 2, 1, 2, 4, 16, 8, states=False)
    one._device = op._device
    return one


def test_sizes_past_a_launch_are_refused():
    """What overflows no count on the way to its refusal."""
    for change in (dict(batch=1 << 30, value_heads=1 << 30, key_heads=1, tokens=0), dict(batch=1, tokens=0, value_heads=(1 << 31) - 1,
                                                                                     key_heads=1, value_dim=4096)):
        with pytest.raises(ValueError, match="launch"):
            O.GatedDelta(**{**dict(dtype="bf16", key_dim=64, value_dim=64), **change})
    rows = (1 << 32) - 1
    words = O.Dropout._io.pack(1, 0, 0, *(4096, 1 << 34) * 3)
    for cols in (1 << 34, (1 << 35) - 1):
        rc, msg = _call(_lib.lib().cchip_dropout_run, _lib.DropoutDesc(5, rows, cols, 0.5, 1.0), words, None)
        assert rc == 1 and ("more than 2^42 elements" in msg or "rows of out overlap" in msg), msg


# ---- workspaces --------------------------------------------------------------

class _Memory:
    """Buffers of host addresses, in the order they are made."""

    made = []

    def __init__(self, nbytes):
        self.ptr, self.nbytes, self.freed = 4096 * (len(self.made) + 1), nbytes, False
        self.made.append(self)

    def free(self):
        self.freed = True


@pytest.fixture
def memory(monkeypatch):
    monkeypatch.setattr(_Memory, "made", [])
    monkeypatch.setattr(O.Buffer, "alloc", staticmethod(_Memory))
    return _Memory.made


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_a_workspace_stays_where_a_graph_may_hold_it(memory, dtype):
    """A backward pass that needs more than a forward call leaves the forward
    call's workspace alone: a graph captured with it may be replayed yet."""
    op = O.GatedDelta(dtype, 1, 4096, 8, 32, 128, 128)
    assert op.workspace_bytes(backward=True) > op.workspace_bytes() > 0
    op.reserve(77)
    held = op._workspace(77)
    op.reserve(77, backward=True)
    assert op._workspace(77) == held and op._workspace(77, True) != held
    assert not any(m.freed for m in memory)
    assert [m.nbytes for m in memory] == [op.workspace_bytes(), op.workspace_bytes(backward=True)]
    op._workspace(78)
    assert len(memory) == 3  # another stream's is its own
    op.free()
    assert all(m.freed for m in memory)


def test_a_callers_workspace(memory):
    """The caller's memory is handed on, checked, and nothing is allocated."""
    op = O.GatedDelta("f32", 2, 100, 2, 4, 16, 8, states=False)
    op._device = -1
    n = op.workspace_bytes()
    w = torch.zeros(n + 16, dtype=torch.uint8)
    assert op._workspace(5, False, w) == (w.data_ptr(), n + 16) and not memory
    x = _delta_arrays(t=100)
    with pytest.raises(ValueError, match="workspace needs"):
        op.forward(*x.values(), workspace=w[:n - 16])
    with pytest.raises(ValueError, match="workspace needs"):
        op.forward(*x.values(), workspace=w[8:])
    with pytest.raises(ValueError, match="workspace has dtype"):
        op.forward(*x.values(), workspace=torch.zeros(n))
    block = O.NormBlock("f32", 4, 8)
    block._device = -1
    assert block.workspace_bytes() == 0 < block.workspace_bytes(backward=True)
    z = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="workspace needs"):
        block.backward(z, z.clone(), z.clone(), dn=z, h=z, grads=dict(pre_weight=torch.zeros(8)),
                       workspace=torch.zeros(4, dtype=torch.uint8))
    assert not memory
