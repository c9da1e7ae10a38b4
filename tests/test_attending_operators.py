"""Attention, the norm and rotation of its heads and the embedding without a
device: the ABI, what is refused, and the 64-bit references' gradients against
differences."""

import ctypes
import os
import re
import subprocess

import numpy as np
import pytest
import torch

import attending_reference as A
from cudacaml_amd import _lib
from cudacaml_amd import operators as O

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_structures_have_the_headers_sizes(tmp_path):
    """The header is strict C99, and what Python packs is what C reads."""
    names = ["cchip_attention", "cchip_attention_io", "cchip_head_norm", "cchip_head_norm_io", "cchip_embedding",
             "cchip_embedding_io"]
    at = ["cchip_attention_io, o", "cchip_attention_io, offsets", "cchip_head_norm_io, k_cache", "cchip_head_norm_io, positions",
          "cchip_embedding_io, dout", "cchip_embedding_io, accumulate"]
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "cchip_operators.h"\nint main(void) {\n'
                   + "".join('  printf("%%zu\\n", sizeof(%s));\n' % n for n in names)
                   + "".join('  printf("%%zu\\n", offsetof(%s));\n' % n for n in at) + "  return 0;\n}\n")
    exe = str(tmp_path / "sizes")
    subprocess.run(["gcc", "-std=c99", "-pedantic", "-Wall", "-Wextra", "-Werror", "-I" + os.path.join(ROOT, "include"),
                    "-o", exe, str(src)], check=True)
    got = [int(x) for x in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(_lib.AttentionDesc), O.Attention._forward_io.size, ctypes.sizeof(_lib.HeadNormDesc),
                   O.HeadNorm._io.size, ctypes.sizeof(_lib.EmbeddingDesc), O.Embedding._io.size,
                   3 * 32, 8 * 32, 5 * 32, 11 * 32, 5 * 8, 9 * 8]
    assert O.Attention._backward_io.size == O.Attention._forward_io.size


# ---- shapes that the handles refuse --------------------------------------------

ATTENTION = dict(dtype="bf16", batch=2, tokens=100, heads=4, kv_heads=2, head_dim=64)
BAD_ATTENTION = [
    (dict(dtype="f64"), "dtype"),
    (dict(kv_heads=3), "multiple"),
    (dict(kv_heads=0), "multiple"),
    (dict(heads=0), "multiple"),
    (dict(head_dim=0), "head_dim"),
    (dict(head_dim=129), "head_dim"),
    (dict(batch=-1), "negative"),
    (dict(tokens=1 << 31), "2\\^31"),
    (dict(keys=1 << 31), "2\\^31"),
    (dict(keys=0), "keys"),
    (dict(sequences=0), "sequences"),
    (dict(sequences=2), "batch of 1"),
    (dict(batch=1, sequences=2, keys=100), "packed"),
    (dict(scale=float("inf")), "finite"),
    (dict(scale=float("nan")), "finite"),
    (dict(batch=1 << 30, tokens=1 << 20), "launch"),
    (dict(batch=1 << 40), "launch"),
    (dict(batch=1, tokens=1 << 30, heads=1 << 20, kv_heads=1), "launch"),
]


@pytest.mark.parametrize("change,why", BAD_ATTENTION)
def test_attention_refuses_its_shapes(change, why):
    O.Attention(**ATTENTION)
    with pytest.raises(ValueError, match=why):
        O.Attention(**{**ATTENTION, **change})


HEADS = dict(dtype="bf16", batch=2, tokens=100, heads=4, kv_heads=2, head_dim=64)
BAD_HEADS = [
    (dict(dtype="i32"), "dtype"),
    (dict(weight_dtype="f16"), "weights"),
    (dict(heads=0), "heads"),
    (dict(kv_heads=0), "heads"),
    (dict(heads=1 << 21), "heads"),
    (dict(head_dim=0), "head_dim"),
    (dict(head_dim=513), "head_dim"),
    (dict(rotary=7), "rotary"),
    (dict(rotary=66), "rotary"),
    (dict(rotary=-2), "rotary"),
    (dict(norm="layer"), "norm"),
    (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"),
    (dict(keys=0), "keys"),
    (dict(keys=1 << 31), "2\\^31"),
    (dict(batch=1 << 16, tokens=1 << 15), "2\\^31"),
    (dict(tokens=-1), "negative"),
]


@pytest.mark.parametrize("change,why", BAD_HEADS)
def test_head_norm_refuses_its_shapes(change, why):
    O.HeadNorm(**HEADS)
    with pytest.raises(ValueError, match=why):
        O.HeadNorm(**{**HEADS, **change})


EMBEDDING = dict(dtype="bf16", tokens=100, vocab=50, width=64)
BAD_EMBEDDING = [
    (dict(dtype="u8"), "dtype"),
    (dict(weight_dtype="f16"), "dtype"),
    (dict(tokens=-1), "tokens"),
    (dict(tokens=(1 << 30) + 1), "tokens"),
    (dict(vocab=1 << 31), "vocab"),
    (dict(vocab=0), "vocab"),
    (dict(width=(1 << 20) + 1), "width"),
    (dict(width=0), "width"),
    (dict(scale=float("inf")), "scale"),
]


@pytest.mark.parametrize("change,why", BAD_EMBEDDING)
def test_embedding_refuses_its_shapes(change, why):
    O.Embedding(**EMBEDDING)
    with pytest.raises(ValueError, match=why):
        O.Embedding(**{**EMBEDDING, **change})


def test_what_is_kept_and_worked_in():
    one = O.Attention("bf16", 1, 640, 4, 2, 64)
    assert O.Attention("bf16", 2, 640, 4, 2, 64).saved_bytes() == 2 * one.saved_bytes() > 0
    # a cache has no backward pass; nothing to do needs nothing
    cache = O.Attention("bf16", 2, 1, 4, 2, 64, keys=4096)
    assert cache.saved_bytes() == 0 and cache.workspace_bytes(backward=True) == 0 < cache.workspace_bytes()
    for shape in [(0, 10), (10, 0)]:
        op = O.Attention("f32", *shape, 4, 2, 64)
        assert op.saved_bytes() == op.workspace_bytes() == op.workspace_bytes(backward=True) == 0
    assert O.HeadNorm("bf16", 2, 10, 4, 2, 64, norm="none").workspace_bytes(backward=True) == 0
    assert O.HeadNorm("bf16", 2, 10, 4, 2, 64).workspace_bytes(backward=True) > 0
    assert O.Embedding("bf16", 100, 50, 64).workspace_bytes(backward=True) == 0
    assert O.Embedding("bf16", 1000, 50, 64).workspace_bytes(backward=True) > 0


# ---- arrays and calls that the handles refuse ------------------------------------

def _attention_arrays(b=2, t=10, h=4, hk=2, d=16, n=None):
    z = lambda *s: torch.zeros(s)  # noqa: E731
    return dict(q=z(b, t, h, d), k=z(b, n or t, hk, d), v=z(b, n or t, hk, d), o=z(b, t, h, d))


@pytest.mark.parametrize("name,bad,why", [
    ("q", torch.zeros(2, 10, 4, 8), "shape"),
    ("k", torch.zeros(2, 10, 4, 16), "shape"),
    ("v", torch.zeros(2, 10, 2, 16, dtype=torch.float64), "dtype"),
    ("o", torch.zeros(2, 10, 4, 16, dtype=torch.float16), "dtype"),
    ("k", torch.zeros(2, 10, 16, 2).transpose(2, 3), "contiguous"),
    ("v", torch.zeros(2, 10, 2, 16), "device"),
    ("q", None, "q"),
])
def test_attention_refuses_arrays(name, bad, why):
    op = O.Attention("f32", 2, 10, 4, 2, 16)
    x = _attention_arrays()
    op._device = -1 if why != "device" else 0  # as if these were the device's
    x[name] = bad
    with pytest.raises((ValueError, TypeError), match=why):
        op.forward(*x.values())


def test_attention_refuses_calls():
    x = _attention_arrays()
    op = O.Attention("f32", 2, 10, 4, 2, 16)
    op._device = -1
    q, k, v, o = x.values()
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32)  # noqa: E731
    with pytest.raises(ValueError, match="saved"):
        op.backward(q, k, v, o, o, None, q, k, v)
    with pytest.raises(ValueError, match="offsets"):
        op.forward(*x.values(), offsets=i32(0, 5, 10))
    with pytest.raises(ValueError, match="lengths"):
        op.forward(*x.values(), lengths=i32(5, 10))
    with pytest.raises(ValueError, match="shape"):
        op.forward(*x.values(), saved=torch.zeros(16, dtype=torch.uint8))
    packed = O.Attention("f32", 1, 10, 4, 2, 16, sequences=3)
    packed._device = -1
    one = _attention_arrays(b=1)
    with pytest.raises(ValueError, match="offsets"):
        packed.forward(*one.values())
    with pytest.raises(ValueError, match="shape"):
        packed.forward(*one.values(), offsets=i32(0, 5, 10))
    with pytest.raises(ValueError, match="dtype"):
        packed.forward(*one.values(), offsets=torch.zeros(4, dtype=torch.int64))
    cache = O.Attention("f32", 2, 10, 4, 2, 16, keys=50)
    cache._device = -1
    with pytest.raises(ValueError, match="shape"):
        cache.forward(*x.values(), lengths=i32(5, 10))
    c = _attention_arrays(n=50)
    with pytest.raises(ValueError, match="lengths"):
        cache.forward(*c.values())
    with pytest.raises(ValueError, match="shape"):
        cache.forward(*c.values(), lengths=i32(5, 10, 3))
    with pytest.raises(ValueError, match="cache"):
        cache.backward(q, k, v, o, o, torch.zeros(0, dtype=torch.uint8), q, k, v)
    with pytest.raises(ValueError, match="saved"):
        cache.forward(*c.values(), lengths=i32(5, 10), saved=torch.zeros(16, dtype=torch.uint8))


def _heads_arrays(b=2, t=10, h=4, hk=2, d=16):
    z = lambda n: torch.zeros(b, t, n, d)  # noqa: E731
    return dict(q=z(h), k=z(hk), q_out=z(h), k_out=z(hk))


def test_head_norm_refuses_calls():
    op = O.HeadNorm("f32", 2, 10, 4, 2, 16)
    op._device = -1
    x = _heads_arrays()
    f = torch.zeros(8)
    for name, bad, why in [("q", torch.zeros(2, 10, 2, 16), "shape"), ("k_out", torch.zeros(2, 10, 2, 16, dtype=torch.float16), "dtype"),
                           ("q_out", torch.zeros(2, 10, 16, 4).transpose(2, 3), "contiguous")]:
        with pytest.raises(ValueError, match=why):
            op.forward(*{**x, name: bad}.values(), frequencies=f)
    with pytest.raises(ValueError, match="frequencies"):
        op.forward(*x.values())
    with pytest.raises(ValueError, match="shape"):
        op.forward(*x.values(), frequencies=torch.zeros(7))
    with pytest.raises(ValueError, match="shape"):
        op.forward(*x.values(), frequencies=f, positions=torch.zeros(10, dtype=torch.int32))
    with pytest.raises(ValueError, match="dtype"):
        op.forward(*x.values(), frequencies=f, positions=torch.zeros(2, 10, dtype=torch.int64))
    with pytest.raises(ValueError, match="q_weight"):
        op.forward(*x.values(), frequencies=f, q_weight=torch.ones(8))
    with pytest.raises(ValueError, match="cache"):
        op.forward(*x.values(), frequencies=f, v=x["k"])
    with pytest.raises(ValueError, match="unknown parameter"):
        op.backward(*x.values(), x["q"], x["k"], frequencies=f, grads=dict(weight=torch.zeros(16)))
    with pytest.raises(ValueError, match="written over"):
        op.forward(x["q"], x["k"], x["q_out"], x["q_out"][:, :, :2], frequencies=f)
    with pytest.raises(ValueError, match="written over k"):
        op.forward(x["q"], x["q_out"][:, :, :2], x["q_out"], x["k_out"], frequencies=f)
    with pytest.raises(ValueError, match="not head for head"):  # in place, but by other strides
        whole = torch.zeros(2, 20, 4, 16)
        op.forward(whole[:, ::2], x["k"], whole[:, :10], x["k_out"], frequencies=f)
    plain = O.HeadNorm("f32", 2, 10, 4, 2, 16, norm="none")
    plain._device = -1
    with pytest.raises(ValueError, match="norm that there is not"):
        plain.forward(*x.values(), frequencies=f, q_weight=torch.ones(16))
    cached = O.HeadNorm("f32", 2, 10, 4, 2, 16, keys=50)
    cached._device = -1
    c = torch.zeros(2, 50, 2, 16)
    with pytest.raises((ValueError, TypeError)):
        cached.forward(x["q"], x["k"], x["q_out"], frequencies=f, k_cache=c, v_cache=c.clone())
    with pytest.raises(ValueError, match="v_cache is written over k_cache"):
        cached.forward(x["q"], x["k"], x["q_out"], frequencies=f, v=x["k"].clone(), k_cache=c, v_cache=c)
    with pytest.raises(ValueError, match="shape"):
        cached.forward(x["q"], x["k"], x["q_out"], frequencies=f, v=x["k"], k_cache=c[:, 1:], v_cache=c)


def test_embedding_refuses_calls():
    op = O.Embedding("f32", 10, 50, 16)
    op._device = -1
    ids, w, out = torch.zeros(10, dtype=torch.int32), torch.zeros(50, 16), torch.zeros(10, 16)
    with pytest.raises(ValueError, match="no ids"):
        op.forward(None, w, out)
    with pytest.raises(ValueError, match="dtype"):
        op.forward(ids.long(), w, out)
    with pytest.raises(ValueError, match="shape"):
        op.forward(ids[1:], w, out)
    with pytest.raises(ValueError, match="weight"):
        op.forward(ids, w[1:], out)
    with pytest.raises(ValueError, match="no out"):
        op.forward(ids, w, None)
    with pytest.raises(ValueError, match="contiguous"):
        op.forward(ids, torch.zeros(16, 50).t(), out)
    with pytest.raises(ValueError, match="overlap"):
        op.forward(ids, w, out[:1].expand(10, 16))
    with pytest.raises(ValueError, match="written over"):
        op.forward(ids, w, w[:10])
    with pytest.raises(ValueError, match="written over"):
        op.backward(ids, w[:10], w)
    with pytest.raises(ValueError, match="no dout"):
        op.backward(ids, None, w)
    many = O.Embedding("f32", 1000, 50, 16)
    many._device = -1
    n = many.workspace_bytes(backward=True)
    for bad in (torch.zeros(n - 16, dtype=torch.uint8), torch.zeros(n + 16, dtype=torch.uint8)[8:]):
        with pytest.raises(ValueError, match="workspace needs"):
            many.backward(torch.zeros(1000, dtype=torch.int32), torch.zeros(1000, 16), w, workspace=bad)


# ---- the C entries ----------------------------------------------------------------

def _call(fn, *args):
    rc = fn(*args)
    return rc, _lib.lib().cchip_last_error().decode()


def test_attention_c_entries_refuse_before_any_device_work():
    L = _lib.lib()
    d = _lib.AttentionDesc(0, 2, 100, 0, 0, 4, 2, 8, 1.0)
    t = lambda p, h=4: (p << 20, 100 * 8 * h, 8 * h, 8)  # noqa: E731
    good = [*t(1), *t(2, 2), *t(3, 2), *t(4)]

    def forward(words, tail=(0, 0, 4098), ws=None, n=0, desc=d):
        # `saved` off its alignment: what is taken otherwise is refused for that
        return _call(L.cchip_attention_forward, desc, O.Attention._forward_io.pack(*words, *tail), ws, n, None)

    rc, msg = forward(good)
    assert rc == 1 and "saved is not aligned" in msg
    for at, value, why in [(0, 0, "no q"), (4, 0, "no k"), (12, 0, "no o"), (8, (3 << 20) + 2, "v is not aligned"),
                           (13, 0, "o overlap"), (14, 0, "o overlap"), (15, 4, "o overlap"), (6, 1 << 24, "tokens of k"),
                           (2, -32, "tokens of q"), (12, 2 << 20, "o is written over k"), (12, (1 << 20) + 16, "o is written over q")]:
        words = list(good)
        words[at] = value
        rc, msg = forward(words)
        assert rc == 1 and why in msg, (at, msg)
    for tail, why in [((4096, 0, 0), "offsets without"), ((0, 4096, 0), "lengths without")]:
        rc, msg = forward(good, tail)
        assert rc == 1 and why in msg
    packed = _lib.AttentionDesc(0, 1, 100, 3, 0, 4, 2, 8, 1.0)
    for tail, why in [((0, 0, 0), "need offsets"), ((4098, 0, 0), "offsets is not aligned"), ((4096, 4096, 0), "lengths without")]:
        rc, msg = forward(good, tail, desc=packed)
        assert rc == 1 and why in msg
    cache = _lib.AttentionDesc(0, 2, 1, 0, 4096, 4, 2, 8, 1.0)
    for tail, why in [((0, 0, 0), "needs lengths"), ((0, 4097, 0), "lengths is not aligned"), ((0, 4096, 4096), "no backward"),
                      ((0, 4096, 0), "workspace needs")]:
        rc, msg = forward([*t(1), 1 << 24, 1 << 16, 16, 8, 1 << 25, 1 << 16, 16, 8, *t(4)], tail, desc=cache)
        assert rc == 1 and why in msg, msg

    back = good + [*t(5), *t(6), *t(7, 2), *t(8, 2)]

    def backward(words, tail=(0, 0, 1 << 28), ws=None, n=0, desc=d):
        return _call(L.cchip_attention_backward, desc, O.Attention._backward_io.pack(*words, *tail), ws, n, None)

    rc, msg = backward(back)
    assert rc == 1 and re.search(r"workspace needs (\d+) bytes aligned to 16, has 0$", msg)
    need = int(re.search(r"needs (\d+)", msg).group(1))
    for ws, n in [(1 << 29, need - 1), ((1 << 29) + 8, need), (None, need)]:
        rc, msg = backward(back, ws=ws, n=n)
        assert rc == 1 and "workspace needs" in msg
    rc, msg = backward(back, ws=1 << 28, n=need)
    assert rc == 1 and "is what the forward pass saved" in msg
    rc, msg = backward(back, (0, 0, 0))
    assert rc == 1 and "needs what the forward pass saved" in msg
    for at, value, why in [(16, 0, "no the gradient of o"), (20, 0, "no dq"), (24, 8 << 20, "dk and dv are written to one place"),
                           (20, 4 << 20, "dq is written over o"), (28, 3 << 20, "dv is written over v"),
                           (24, 5 << 20, "dk is written over the gradient of o"), (26, 0, "dk overlap")]:
        words = list(back)
        words[at] = value
        rc, msg = backward(words)
        assert rc == 1 and why in msg, (at, msg)
    rc, msg = backward(back, desc=cache)
    assert rc == 1 and "no backward" in msg
    for fn in (L.cchip_attention_forward, L.cchip_attention_backward):
        rc, msg = _call(fn, None, None, None, 0, None)
        assert rc == 1 and "no descriptor" in msg
        rc, msg = _call(fn, d, None, None, 0, None)
        assert rc == 1 and "no tensors" in msg


def test_head_norm_and_embedding_c_entries_refuse():
    L = _lib.lib()
    d = _lib.HeadNormDesc(0, 0, 2, 100, 0, 4, 2, 8, 8, 0, 1, 1e-6)
    t = lambda p, h=4: (p << 20, 100 * 8 * h, 8 * h, 8)  # noqa: E731
    none = (0, 0, 0, 0)
    good = [*t(1), *t(2, 2), *none, *t(3), *t(4, 2), *none, *none, *none, *none, *none, *none, 0, 4096, 0, 0, 0, 0]

    def forward(words, desc=d):
        return _call(L.cchip_head_norm_forward, desc, O.HeadNorm._io.pack(*words), None)

    for at, value, why in [(0, 0, "no q"), (0, (1 << 20) + 2, "q is not aligned"), (2, -32, "tokens of q"), (12, 0, "no q_out"),
                           (16, 0, "no k_out"), (14, 0, "q_out overlap"), (12, 2 << 20, "q_out is written over k"),
                           (16, 3 << 20, "k_out is written over q_out"), (44, 4098, "positions is not"), (45, 0, "no frequencies"),
                           (45, 4098, "frequencies is not"), (46, 4098, "q_weight is not"), (49, 4098, "gradient of k_weight is not"),
                           (20, 4096, "without keys"), (8, 4096, "without keys")]:
        words = list(good)
        words[at] = value
        rc, msg = forward(words)
        assert rc == 1 and why in msg, (at, msg)
    back = [*t(1), *t(2, 2), *none, *none, *none, *none, *none, *t(3), *t(4, 2), *t(5), *t(6, 2), 0, 4096, 0, 0, 4096, 0]
    for at, value, why in [(28, 0, "gradient of q_out"), (36, 0, "no dq"), (36, 1 << 20, "dq is written over q"),
                           (40, 5 << 20, "dk is written over dq"), (37, 1, "dq overlap"), (0, 1 << 20, "workspace needs")]:
        words = list(back)
        words[at] = value
        rc, msg = _call(L.cchip_head_norm_backward, d, O.HeadNorm._io.pack(*words), None, 0, None)
        assert rc == 1 and why in msg, (at, msg)
    e = _lib.EmbeddingDesc(0, 0, 100, 50, 8, 1.0)
    words = [4096, 1 << 20, 8, 2 << 20, 8, 0, 0, 0, 0, 0]
    for at, value, why in [(0, 0, "no ids"), (0, 4098, "ids"), (1, 0, "weight"), (1, (1 << 20) + 1, "weight"), (3, 0, "out"),
                           (4, 7, "overlap"), (3, 1 << 20, "written over")]:
        bad = list(words)
        bad[at] = value
        rc, msg = _call(L.cchip_embedding_forward, e, O.Embedding._io.pack(*bad), None)
        assert rc == 1 and why in msg, (at, msg)
    for fn, more in ((L.cchip_head_norm_forward, ()), (L.cchip_head_norm_backward, (None, 0)), (L.cchip_embedding_forward, ()),
                     (L.cchip_embedding_backward, (None, 0))):
        rc, msg = _call(fn, None, None, *more, None)
        assert rc == 1 and "no descriptor" in msg
    for fn, desc in ((L.cchip_head_norm_forward, d), (L.cchip_embedding_forward, e)):
        rc, msg = _call(fn, desc, None, None)
        assert rc == 1 and "no tensors" in msg


# ---- the references ----------------------------------------------------------------

def _differences(f, x, got, name, step=1e-5):
    """Of a scalar function f at x against the gradient, in a direction."""
    way = np.random.default_rng(1).standard_normal(x.shape)
    slope = (f(x + step * way) - f(x - step * way)) / (2 * step)
    assert abs(slope - (got * way).sum()) <= 1e-8 * (1 + abs(slope)), name


@pytest.mark.parametrize("t,n,h,hk,d,scale", [(5, 5, 2, 1, 3, 0.7), (3, 7, 4, 2, 5, -0.4), (4, 2, 2, 2, 3, 1.0)])
def test_attention_reference(t, n, h, hk, d, scale):
    g = np.random.default_rng(0)
    q, do = g.standard_normal((2, t, h, d))
    k, v = g.standard_normal((2, n, hk, d))
    o, dq, dk, dv, *_ = A.attention(q, k, v, scale, do)
    for i, (x, got) in enumerate(((q, dq), (k, dk), (v, dv))):
        _differences(lambda y: (A.attention(*[y if j == i else z for j, z in enumerate((q, k, v))], scale) * do).sum(), x, got, i)
    if t > n:
        assert not o[:t - n].any() and not dq[:t - n].any()
    # a query that sees one key has its value
    first = max(t - n, 0)
    if t >= n:
        np.testing.assert_allclose(o[first], np.repeat(v[0], h // hk, axis=0), rtol=1e-14)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_head_norm_reference(interleaved, norm):
    g = np.random.default_rng(2)
    x, dy = g.standard_normal((2, 2, 3, 2, 7))
    w = g.standard_normal(7)
    angle = g.standard_normal((2, 3, 1, 2))
    f = lambda x, w: A.head_norm(x, w, angle, 4, interleaved, norm, 1e-3)  # noqa: E731
    dx, dw, _ = A.head_norm(x, w, angle, 4, interleaved, norm, 1e-3, dy)
    _differences(lambda y: (f(y, w) * dy).sum(), x, dx, "x")
    _differences(lambda y: (f(x, y) * dy).sum(), w, dw, "w")
    # a rotation keeps the lengths of pairs, and the rest
    y = f(x, w)
    xhat = x * w / (np.sqrt((x * x).mean(-1, keepdims=True) + 1e-3) if norm else 1.0)
    np.testing.assert_allclose((y ** 2).sum(-1), (xhat ** 2).sum(-1), rtol=1e-12)
    np.testing.assert_allclose(y[..., 4:], xhat[..., 4:], rtol=1e-12)


def test_embedding_reference():
    g = np.random.default_rng(3)
    ids = np.array([3, 0, 3, -1, 9, 3, 1])
    w, dout = g.standard_normal((5, 4)), g.standard_normal((7, 4))
    _differences(lambda y: (A.embed(ids, y, 1.5) * dout).sum(), w, A.embed_back(ids, dout, 5, 1.5)[0], "weight")
    assert not A.embed(ids, w, 1.5)[3:5].any()
