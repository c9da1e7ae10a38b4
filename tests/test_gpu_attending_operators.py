"""Attention, the norm and rotation of its heads and the embedding on the
device against the 64-bit references of attending_reference.py.

Bounds, from the formats alone; h is half a step relative to the value, 2^-8
of bf16, 2^-11 of f16 and 2^-24 of f32:
- attention, 16 bits: two operands or results are rounded on the way to each
  output (the weights p, or their gradients, and the output). A rounding is
  spread over half a step either way and at most h / sqrt(3) in the root mean
  square; two are sqrt(2/3) h: h in the 2-norm. Single elements of few terms
  may reach h for each.
- attention, f32: five chained sums of up to 128 products, each off by about
  sqrt(128) 2^-24 of its terms' norm: 4e-6, and 8e-6 for the gradients of k and
  v, which are sums over queries besides. Gradients of q and k are sums of
  differences that may cancel; what f32 is off of their terms is allowed too.
- all of attention: a score is an exponent, so what four roundings of it (its
  sum, its scale, the difference, its power of two) are off in f32, 2^-22 of
  the largest score, weights are off by, relative to themselves.
- head norm: one rounding of an f32 result, which a sum of at most 512
  squares in a tree, a root, a sine and a cosine and at most four products
  each put off by a few 2^-24: 2^-19 of the largest of a head's terms.
- embedding: one rounding, of a product; of the gradient, of a sum in f32,
  which each of its n terms may put off by 2^-24 of the sum of magnitudes.
"""

import numpy as np
import pytest
import torch

import attending_reference as A
from cudacaml_amd import backend_hip as H
from cudacaml_amd import operators as O
from cudacaml_amd.runtime import Buffer, Device, Stream

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BOUND = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 4e-6}


def f64(x):
    return x.detach().cpu().double().numpy()


def normal(dtype, *shape, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(TYPES[dtype])


def i32(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def nans(shape, dtype):
    return torch.full(shape, float("nan"), dtype=TYPES[dtype], device="cuda")


def same(a, b):
    """Bit for bit, NaN and all."""
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


# ---- attention -----------------------------------------------------------------

def attention_arrays(dtype, b, t, h, hk, d, seed=0, keys=None):
    n = keys or t
    x = dict(q=normal(dtype, b, t, h, d, seed=4 * seed), k=normal(dtype, b, n, hk, d, seed=4 * seed + 1),
             v=normal(dtype, b, n, hk, d, seed=4 * seed + 2))
    if not keys:
        x["do"] = normal(dtype, b, t, h, d, seed=4 * seed + 3)
    return x


def run_attention(x, dtype, cuts=None, scale=None, op=None, layout=lambda d: d, out=None, stream=None, **workspaces):
    b, t, h, d = x["q"].shape
    hk = x["k"].shape[2]
    op = op or O.Attention(dtype, b, t, h, hk, d, scale=scale, sequences=None if cuts is None else len(cuts) - 1)
    dev = layout({k: v.cuda() for k, v in x.items()})
    offsets = None if cuts is None else i32(*cuts)
    out = out or {n: nans(x[m].shape, dtype) for n, m in (("o", "q"), ("dq", "q"), ("dk", "k"), ("dv", "v"))}
    saved = torch.full((op.saved_bytes(),), 255, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    op.forward(dev["q"], dev["k"], dev["v"], out["o"], offsets=offsets, saved=saved, stream=stream,
               workspace=workspaces.get("forward"))
    op.backward(dev["q"], dev["k"], dev["v"], out["o"], dev["do"], saved, out["dq"], out["dk"], out["dv"], offsets=offsets,
                stream=stream, workspace=workspaces.get("backward"))
    torch.cuda.synchronize()
    return out


def check_attention(x, dtype, got, cuts=None, scale=None):
    b, t, h, d = x["q"].shape
    scale = d ** -0.5 if scale is None else scale
    a = {n: f64(v) for n, v in x.items()}
    pieces = [(i, 0, t) for i in range(b)] if cuts is None else [(0, lo, hi) for lo, hi in zip(cuts, cuts[1:])]
    want = {n: np.full(tuple(v.shape), np.nan) for n, v in got.items()}
    cancelled, largest = np.zeros(3), 0.0
    for i, lo, hi in pieces:
        part = [a[n][i, lo:hi] for n in ("q", "k", "v")]
        *r, c, top = A.attention(*part, scale, a["do"][i, lo:hi])
        cancelled += np.square(c)
        largest = max(largest, top)
        for n, v in zip(("o", "dq", "dk", "dv"), r):
            want[n][i, lo:hi] = v
    for n, c in zip(("o", "dq", "dk", "dv"), (0.0, *np.sqrt(cancelled))):
        g = f64(got[n])
        assert (np.isnan(g) == np.isnan(want[n])).all(), n  # tokens of no sequence are left as they were
        there = ~np.isnan(want[n])
        bound = 8e-6 if dtype == "f32" and n in ("dk", "dv") else BOUND[dtype]
        if there.sum() < 256:  # a root mean square says little: each rounding as far as it can be
            bound *= 2
        off = 2.0 ** -22 * largest
        A.close(g[there], want[n][there], n, bound + off, c * (1 + off / 4e-6))


SHAPES = [(1, 1, 1, 1, 1), (1, 1, 2, 1, 128), (2, 2, 1, 1, 33), (2, 5, 4, 2, 64), (1, 33, 2, 1, 128), (3, 64, 7, 1, 9), (1, 65, 5, 5, 16),
          (2, 300, 6, 2, 72), (1, 515, 3, 3, 105), (1, 700, 8, 2, 128), (1, 1100, 16, 1, 64), (1, 2100, 2, 1, 40)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", SHAPES)
def test_attention(device, dtype, shape):
    x = attention_arrays(dtype, *shape)
    check_attention(x, dtype, run_attention(x, dtype))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0])
def test_attention_scales(device, dtype, scale):
    """None, one that turns the order of scores round, and one that makes them
    so large that a row is nearly one key's."""
    x = attention_arrays(dtype, 1, 200, 4, 2, 24, seed=1)
    got = run_attention(x, dtype, scale=scale)
    check_attention(x, dtype, got, scale=scale)
    if scale == 0.0:
        assert not got["dq"].any() and not got["dk"].any()


CUTS = [[0, 0], [0, 300], [0, 1, 1, 130, 300], [0, 0, 0, 63, 64, 129, 129, 256, 299, 300], [7, 20, 20, 100, 291]]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("cuts", CUTS)
@pytest.mark.parametrize("heads", [(4, 2, 64), (3, 1, 100)])
def test_attention_packed(device, dtype, cuts, heads):
    x = attention_arrays(dtype, 1, 300, *heads, seed=2)
    check_attention(x, dtype, run_attention(x, dtype, cuts=cuts), cuts=cuts)


def test_attention_packed_long_and_many(device):
    """Eight waves a workgroup, some chunks of rows, and many short sequences."""
    for cuts in ([0, 5, 1500, 2600], list(range(0, 2601, 13))):
        x = attention_arrays("bf16", 1, 2600, 2, 1, 64, seed=3)
        check_attention(x, "bf16", run_attention(x, "bf16", cuts=cuts), cuts=cuts)


def test_attention_offsets_are_clamped(device):
    x = attention_arrays("bf16", 1, 120, 2, 1, 32, seed=4)
    a = run_attention(x, "bf16", cuts=[-9, 50, 1000])
    b = run_attention(x, "bf16", cuts=[0, 50, 120])
    for n in a:
        assert same(a[n], b[n]), n


def test_attention_offsets_that_decrease_stay_in_bounds(device):
    """Sequences that lie over one another have no result to speak of, but
    need no more of the workspace than others."""
    x = attention_arrays("bf16", 1, 1000, 2, 1, 32, seed=4)
    op = O.Attention("bf16", 1, 1000, 2, 1, 32, sequences=3)
    need = op.workspace_bytes(backward=True)
    guard = torch.full((need + (1 << 22),), 99, dtype=torch.uint8, device="cuda")
    for cuts in ([0, 1000, 0, 1000], [1000, 0, 1000, 0], [900, 500, 1000, 100]):
        run_attention(x, "bf16", cuts=cuts, op=op, backward=guard[:need])
    assert (guard[need:] == 99).all()
    a, b = run_attention(x, "bf16", cuts=[0, 10, 10, 1000], op=op), run_attention(x, "bf16", cuts=[0, 10, 10, 1000])
    for n in a:
        assert same(a[n], b[n]), n


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", [(0, 10, 2, 1, 8), (2, 0, 2, 1, 8)])
def test_attention_of_nothing(device, dtype, shape):
    x = attention_arrays(dtype, *shape)
    run_attention(x, dtype)


def _cached(dtype, tokens, heads, keys, lengths, seed=0, scale=None):
    h, hk, d = heads
    b = len(lengths)
    x = attention_arrays(dtype, b, tokens, h, hk, d, seed=seed, keys=keys)
    held = [min(max(n, 0), keys) for n in lengths]
    dev = {n: v.cuda() for n, v in x.items()}
    for i, n in enumerate(held):  # what is behind a length is not looked at
        dev["k"][i, n:] = float("nan")
        dev["v"][i, n:] = float("inf")
    o = nans(x["q"].shape, dtype)
    op = O.Attention(dtype, b, tokens, h, hk, d, keys=keys, scale=scale)
    op.forward(dev["q"], dev["k"], dev["v"], o, lengths=i32(*lengths))
    torch.cuda.synchronize()
    a = {n: f64(v) for n, v in x.items()}
    want = np.stack([A.attention(a["q"][i], a["k"][i, :n], a["v"][i, :n], d ** -0.5 if scale is None else scale)
                     for i, n in enumerate(held)])
    got = f64(o)
    for i, n in enumerate(held):
        assert not got[i, :max(0, tokens - n)].any()  # before the first key nothing is seen
    A.close(got, want, "o", BOUND[dtype] * (2 if want.size < 256 else 1))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("tokens,heads,keys,lengths", [
    (1, (1, 1, 1), 1, [1]), (1, (4, 4, 16), 50, [0, 3, 50, 1]), (1, (8, 2, 128), 200, [200, 1, 77]), (1, (8, 1, 64), 1000, [1000, 999]),
    (1, (6, 2, 105), 5000, [4999, 127, 129, 5000]), (1, (16, 1, 128), 3000, [3000]), (3, (8, 2, 128), 777, [777, 2, 300]),
    (1, (40, 1, 64), 300, [290, 256]), (2, (33, 1, 24), 600, [600, 1]), (5, (2, 2, 72), 130, [128, 64, 4]),
    (40, (8, 2, 128), 700, [700, 20, 41]), (150, (8, 4, 64), 2500, [2500, 151, 100]), (300, (2, 1, 100), 301, [300, 301, 0])])
def test_attention_over_a_cache(device, dtype, tokens, heads, keys, lengths):
    _cached(dtype, tokens, heads, keys, lengths, seed=5)


def test_attention_lengths_are_clamped(device):
    _cached("bf16", 1, (4, 1, 64), 300, [-5, 400, 1 << 30, -(1 << 31)], seed=6)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("tokens,keys", [(1, None), (40, 40), (700, None), (1, 2000)])
def test_attention_not_a_number_reaches_who_sees_it(device, dtype, tokens, keys):
    """In k or v, with the queries that do not see it as they were; rows of a
    cache and key heads that it is not in, too."""
    x = attention_arrays(dtype, 2, tokens, 4, 2, 48, seed=7, keys=keys)
    n = keys or tokens
    op = O.Attention(dtype, 2, tokens, 4, 2, 48, keys=keys)
    dev = {m: v.cuda() for m, v in x.items()}
    lengths = None if keys is None else i32(n, n)

    def run():
        o = nans(x["q"].shape, dtype)
        op.forward(dev["q"], dev["k"], dev["v"], o, lengths=lengths)
        torch.cuda.synchronize()
        return o

    want = run()
    at = n * 2 // 3
    for m in ("k", "v"):
        for bad in (float("nan"), float("inf"), float("-inf")):
            keep = dev[m][1, at, 1, 5].item()
            dev[m][1, at, 1, 5] = bad
            got = run()
            first = max(0, at - (n - tokens))  # the first query that sees it
            assert same(got[0], want[0]) and same(got[1, :, :2], want[1, :, :2])
            assert same(got[1, :first], want[1, :first])
            seen = got[1, first:, 2:]
            if bad != bad:
                assert torch.isnan(seen if m == "k" else seen[..., 5]).all()
            if m == "v":
                assert not torch.isfinite(seen[..., 5]).any() and torch.isfinite(seen[..., :5]).all()
            dev[m][1, at, 1, 5] = keep


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("tokens,keys", [(90, None), (300, None), (1, 90), (1, 1500)])
def test_attention_keys_of_minus_infinity(device, dtype, tokens, keys):
    """Keys that every score with is -infinity weigh nothing, and queries that
    see none but those have zeros; the lowest finite scores are scores."""
    x = attention_arrays(dtype, 1, tokens, 2, 1, 32, seed=8, keys=keys)
    x["q"] = x["q"].abs() + 0.5
    n = keys or tokens
    out = n // 3
    x["k"][:, :out] = float("-inf")
    op = O.Attention(dtype, 1, tokens, 2, 1, 32, keys=keys)
    dev = {m: v.cuda() for m, v in x.items()}
    o = nans(x["q"].shape, dtype)
    op.forward(dev["q"], dev["k"], dev["v"], o, lengths=None if keys is None else i32(n))
    got = f64(o)
    a = {m: f64(v) for m, v in x.items()}
    first = 0 if keys else out
    assert not got[0, :first].any()
    want = A.attention(a["q"][0, first:], a["k"][0, out:], a["v"][0, out:], 32 ** -0.5)
    A.close(got[0, first:], want, "o", BOUND[dtype] * (2 if want.size < 256 else 1))
    op.forward(dev["q"], torch.full_like(dev["k"], float("-inf")), dev["v"], o, lengths=None if keys is None else i32(n))
    torch.cuda.synchronize()
    assert not o.any()


@pytest.mark.parametrize("dtype", list(TYPES))
def test_attention_far_scores(device, dtype):
    """Scores of some thousands that rise and fall along the keys, so that the
    largest seen changes by more than any exponential can hold."""
    x = attention_arrays(dtype, 1, 400, 2, 1, 16, seed=9)
    x["q"][..., 0] = 60.0
    x["k"][0, :, 0, 0] = torch.linspace(-7, 7, 400).cos().to(TYPES[dtype]) * 64
    got = run_attention(x, dtype)
    check_attention(x, dtype, got)


@pytest.mark.parametrize("scale", [1e-4, 3e4])
def test_attention_gradients_of_small_and_large_values(device, scale):
    """f16 has neither: tiles with powers of two of their own."""
    x = attention_arrays("bf16", 1, 150, 4, 2, 64, seed=10)
    for n in ("v", "do"):
        x[n] = x[n] * scale
    check_attention(x, "bf16", run_attention(x, "bf16"))


def _fused(dev):
    """q, k and v side by side, as one projection leaves them."""
    b, t = dev["q"].shape[:2]
    whole = torch.cat([dev[n].reshape(b, t, -1) for n in ("q", "k", "v")], dim=-1)
    out, at = dict(dev), 0
    for n in ("q", "k", "v"):
        size = dev[n].shape[2] * dev[n].shape[3]
        out[n] = whole[..., at:at + size].view(dev[n].shape)
        at += size
    return out


def _heads_first(dev):
    return {n: x.transpose(1, 2).contiguous().transpose(1, 2) for n, x in dev.items()}


def _off_by_one(dev):
    def put(x):
        b, t, h, d = x.shape
        y = torch.empty(b, t, h * d + 3, dtype=x.dtype, device="cuda")[..., 1:1 + h * d].view(x.shape)
        return y.copy_(x)

    return {n: put(x) for n, x in dev.items()}


def _far_apart(tokens):
    """Tokens or rows of the batch so far apart that they pass 2^32 elements."""
    def put(x):
        b, t, h, d = x.shape
        step = (1 << 23) if tokens else h * d
        row = t * step if tokens else (1 << 32) + 8
        whole = torch.empty((b - 1) * row + (t - 1) * step + h * d, dtype=x.dtype, device="cuda")
        return whole.as_strided((b, t, h, d), (row, step, d, 1)).copy_(x)

    return lambda dev: {n: put(x) if n in ("k", "do") else x for n, x in dev.items()}


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("layout", [_fused, _heads_first, _off_by_one])
@pytest.mark.parametrize("shape", [(2, 70, 4, 2, 64), (2, 300, 3, 1, 40), (2, 33, 2, 2, 13)])
def test_attention_strides(device, dtype, layout, shape):
    x = attention_arrays(dtype, *shape, seed=11)
    a, b = run_attention(x, dtype), run_attention(x, dtype, layout=layout)
    for n in a:
        assert same(a[n], b[n]), n


@pytest.mark.parametrize("dtype", list(TYPES))
def test_attention_inputs_read_again(device, dtype):
    """Keys of one row and head for all of them, values of one token."""
    x = attention_arrays(dtype, 2, 150, 4, 2, 64, seed=30)
    x["k"] = x["k"][:1, :, :1].expand_as(x["k"]).contiguous()
    x["v"] = x["v"][:, :1].expand_as(x["v"]).contiguous()
    again = lambda d: {**d, "k": d["k"][:1, :, :1].expand(d["k"].shape), "v": d["v"][:, :1].expand(d["v"].shape)}  # noqa: E731
    a, b = run_attention(x, dtype), run_attention(x, dtype, layout=again)
    for n in a:
        assert same(a[n], b[n]), n


@pytest.mark.parametrize("dtype", list(TYPES))
def test_attention_rows_do_not_depend_on_one_another(device, dtype):
    """A sequence alone, among others and behind one that is much longer: its
    rows lie with others in a tile or alone, with the same results."""
    x = attention_arrays(dtype, 1, 700, 6, 2, 64, seed=31)
    a = run_attention(x, dtype, cuts=[0, 450, 530, 700])
    parts = {n: v[:, 450:530].contiguous() for n, v in x.items()}
    b = run_attention(parts, dtype, cuts=[0, 80])
    for n in ("o", "dq"):
        assert same(a[n][:, 450:530], b[n]), n
    q = x["q"].clone()
    q[:, ::2] *= 30  # every other query's scores rise far more
    c = run_attention({**x, "q": q}, dtype, cuts=[0, 450, 530, 700])
    assert same(a["o"][:, 1::2], c["o"][:, 1::2])


@pytest.mark.parametrize("shape,tokens", [((2, 300, 2, 1, 64), False), ((1, 600, 2, 1, 64), True)])
def test_attention_tensors_past_32_bits(device, shape, tokens):
    x = attention_arrays("bf16", *shape, seed=12)
    a, b = run_attention(x, "bf16"), run_attention(x, "bf16", layout=_far_apart(tokens))
    for n in a:
        assert same(a[n], b[n]), n


@pytest.mark.parametrize("tokens", [1, 200])
def test_attention_cache_past_32_bits(device, tokens):
    """A long cache whose heads lie one behind the other."""
    x = attention_arrays("f16", 1, tokens, 4, 2, 64, seed=13, keys=1500)
    dev = {n: v.cuda() for n, v in x.items()}
    far = {}
    for n in ("k", "v"):
        whole = torch.empty((1 << 32) + 1500 * 64, dtype=torch.float16, device="cuda")
        far[n] = whole.as_strided(dev[n].shape, (1, 64, 1 << 32, 1)).copy_(dev[n])
    op = O.Attention("f16", 1, tokens, 4, 2, 64, keys=1500)
    out = []
    for kv in (dev, far):
        out.append(nans(x["q"].shape, "f16"))
        op.forward(dev["q"], kv["k"], kv["v"], out[-1], lengths=i32(1400))
    torch.cuda.synchronize()
    assert same(*out) and torch.isfinite(out[0]).all()


@pytest.mark.parametrize("dtype", list(TYPES))
def test_attention_writes_only_its_outputs(device, dtype):
    """Into tensors with something between tokens and heads, from workspaces
    that end where they say."""
    shape = (2, 150, 4, 2, 40)
    x = attention_arrays(dtype, *shape, seed=14)
    op = O.Attention(dtype, *shape)
    wholes, out = {}, {}
    for n, m in (("o", "q"), ("dq", "q"), ("dk", "k"), ("dv", "v")):
        b, t, h, d = x[m].shape
        wholes[n] = torch.full((b, t + 1, h + 1, d + 3), 7.0, dtype=TYPES[dtype], device="cuda")
        out[n] = wholes[n][:, :t, :h, :d]
    need = op.workspace_bytes(backward=True)
    guard = torch.full((need + 4096,), 99, dtype=torch.uint8, device="cuda")
    run_attention(x, dtype, op=op, out=out, backward=guard[:need])
    plain = run_attention(x, dtype)
    assert (guard[need:] == 99).all()
    for n in out:
        assert same(out[n], plain[n]), n
        out[n].fill_(7.0)
        assert (wholes[n] == 7.0).all(), n


def test_attention_differences(device):
    """The gradient against differences of the forward pass: as far apart as the
    reference's own, and what 4e-6 of o does to them."""
    shape, step = (1, 70, 4, 2, 24), 0.02
    x = attention_arrays("f32", *shape, seed=15)
    got = run_attention(x, "f32")
    do = f64(x["do"])
    g = torch.Generator().manual_seed(16)
    for n in ("q", "k", "v"):
        way = torch.randn(x[n].shape, generator=g)
        ends = [run_attention({**x, n: x[n] + s * way}, "f32")["o"] for s in (step, -step)]
        slope = sum(s * (f64(o) * do).sum() for s, o in zip((1, -1), ends)) / (2 * step)
        a = [{**{m: f64(v) for m, v in x.items()}, n: f64(x[n] + s * way)} for s in (step, -step)]
        exact = [A.attention(y["q"][0], y["k"][0], y["v"][0], 24 ** -0.5) for y in a]
        apart = ((exact[0] - exact[1]) * do[0]).sum() / (2 * step)
        analytic = (f64(got["d" + n]) * f64(way)).sum()
        a0 = {m: f64(v) for m, v in x.items()}
        true = (dict(zip(("q", "k", "v"), A.attention(a0["q"][0], a0["k"][0], a0["v"][0], 24 ** -0.5, do[0])[1:4]))[n] * f64(way)[0]).sum()
        allowed = abs(apart - true) + 4e-6 * np.linalg.norm(f64(got["o"])) * np.linalg.norm(do) / step
        assert abs(slope - analytic) <= allowed + 8e-6 * np.linalg.norm(f64(got["d" + n])) * np.linalg.norm(f64(way)), n


def test_attention_is_deterministic(device):
    """Jobs come from queues and keys from splits, in any order; sums do not."""
    x = attention_arrays("bf16", 1, 4500, 8, 1, 64, seed=17)
    a = run_attention(x, "bf16")
    for _ in range(2):
        b = run_attention(x, "bf16")
        for n in a:
            assert same(a[n], b[n]), n
    x = attention_arrays("bf16", 2, 1, 8, 2, 128, seed=18, keys=3000)
    op = O.Attention("bf16", 2, 1, 8, 2, 128, keys=3000)
    assert op.workspace_bytes() > 0
    dev, out = {n: v.cuda() for n, v in x.items()}, []
    for _ in range(3):
        out.append(nans(x["q"].shape, "bf16"))
        op.forward(dev["q"], dev["k"], dev["v"], out[-1], lengths=i32(3000, 2000))
    torch.cuda.synchronize()
    assert same(out[0], out[1]) and same(out[0], out[2])


def test_attention_long_rows(device):
    """Against plain products in f32 on the device, which are off by as much
    as theirs: a chunk of rows, chunks of keys and many tiles."""
    b, t, h, hk, d = 1, 6000, 4, 1, 128
    x = attention_arrays("bf16", b, t, h, hk, d, seed=19)
    got = run_attention(x, "bf16")
    q, k, v, do = (x[n][0].cuda().float() for n in ("q", "k", "v", "do"))
    seen = torch.ones(t, t, dtype=torch.bool, device="cuda").tril()
    dk, dv = torch.zeros(t, d, device="cuda"), torch.zeros(t, d, device="cuda")
    for i in range(h):
        s = (q[:, i] @ k[:, 0].t() * d ** -0.5).masked_fill(~seen, float("-inf"))
        p = torch.softmax(s, -1)
        o = p @ v[:, 0]
        A.close(f64(got["o"][0, :, i]), f64(o), "o", BOUND["bf16"])
        dp = do[:, i] @ v[:, 0].t()
        ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * d ** -0.5
        A.close(f64(got["dq"][0, :, i]), f64(ds @ k[:, 0]), "dq", BOUND["bf16"])
        dk += ds.t() @ q[:, i]
        dv += p.t() @ do[:, i]
    A.close(f64(got["dk"][0, :, 0]), f64(dk), "dk", BOUND["bf16"])
    A.close(f64(got["dv"][0, :, 0]), f64(dv), "dv", BOUND["bf16"])


def test_attention_on_another_stream(device):
    x = attention_arrays("bf16", 2, 200, 4, 2, 64, seed=20)
    op = O.Attention("bf16", 2, 200, 4, 2, 64)
    want = run_attention(x, "bf16", op=op)
    for stream in (torch.cuda.Stream(), Stream.create(), torch.cuda.Stream().cuda_stream):
        got = run_attention(x, "bf16", op=op, stream=stream)
        for n in want:
            assert same(got[n], want[n]), n


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_in_a_graph(device, dtype):
    """Captured once and replayed on new inputs, with eager calls of the same
    handle between, and a second graph that shares its workspaces."""
    shape = (2, 130, 4, 2, 64)
    op = O.Attention(dtype, *shape)
    one, two = (attention_arrays(dtype, *shape, seed=s) for s in (21, 22))
    want = [run_attention(x, dtype) for x in (one, two)]
    dev = {n: v.cuda() for n, v in one.items()}
    stream = torch.cuda.Stream()
    op.reserve(stream, backward=True)
    graphs = []
    for _ in range(2):
        out = {n: nans(v.shape, dtype) for n, v in want[0].items()}
        saved = torch.empty(op.saved_bytes(), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            op.forward(dev["q"], dev["k"], dev["v"], out["o"], saved=saved, stream=stream)
            op.backward(dev["q"], dev["k"], dev["v"], out["o"], dev["do"], saved, out["dq"], out["dk"], out["dv"], stream=stream)
        graphs.append((graph, out, saved))
    for i in (0, 1, 0, 1):
        for n, v in (one, two)[i].items():
            dev[n].copy_(v)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            for graph, out, _ in graphs:
                graph.replay()
        torch.cuda.synchronize()
        for _, out, _ in graphs:
            for n in out:
                assert same(out[n], want[i][n]), (i, n)
                out[n].fill_(float("nan"))
        got = run_attention(two, dtype, op=op, stream=stream)
        for n in got:
            assert same(got[n], want[1][n]), n


def test_attention_in_a_graph_with_the_callers_workspace(device):
    """A step over a cache that grows between replays: lengths are the device's."""
    b, keys = 2, 2000
    x = attention_arrays("f16", b, 1, 8, 2, 64, seed=23, keys=keys)
    dev = {n: v.cuda() for n, v in x.items()}
    op = O.Attention("f16", b, 1, 8, 2, 64, keys=keys)
    work = torch.empty(op.workspace_bytes(), dtype=torch.uint8, device="cuda")
    assert work.numel() > 0
    lengths, o = i32(0, 0), nans(x["q"].shape, "f16")
    stream = torch.cuda.Stream()
    live = Buffer.live_count()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        op.forward(dev["q"], dev["k"], dev["v"], o, lengths=lengths, workspace=work, stream=stream)
    assert Buffer.live_count() == live
    op.free()
    for held in ((0, 1), (700, 2000), (3, 1999), (2000, 0)):
        lengths.copy_(torch.tensor(held))
        o.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        want = nans(x["q"].shape, "f16")
        O.Attention("f16", b, 1, 8, 2, 64, keys=keys).forward(dev["q"], dev["k"], dev["v"], want, lengths=i32(*held))
        torch.cuda.synchronize()
        assert same(o, want), held


# ---- norm and rotation of heads --------------------------------------------------

def run_heads(dtype, b, t, h, hk, d, rotary=None, interleaved=False, norm="rms", weight="f32", weights=True, positions=None,
              seed=0, layout=lambda x: x, in_place=False, stream=None):
    rotary = d // 2 * 2 if rotary is None else rotary
    eps = 1e-3
    op = O.HeadNorm(dtype, b, t, h, hk, d, norm=norm, rotary=rotary, interleaved=interleaved, eps=eps, weight_dtype=weight)
    x = {n: normal(dtype, b, t, c, d, seed=4 * seed + i) * (1 + i) for i, (n, c) in enumerate((("q", h), ("k", hk), ("dq", h), ("dk", hk)))}
    freq = torch.exp(-torch.arange(rotary // 2) * 0.4).float()
    w = {n: (1.0 + 0.3 * normal("f32", d, seed=4 * seed + 9 + i)).to(TYPES[weight]) for i, n in enumerate(("q_weight", "k_weight"))}
    w = w if weights and norm != "none" else {}
    dev = {n: layout(v.cuda()) for n, v in x.items()}
    given = dict(frequencies=freq.cuda(), positions=None if positions is None else positions.cuda(), stream=stream,
                 **{n: v.cuda() for n, v in w.items()})
    out = {n: layout(nans(v.shape, dtype)) for n, v in x.items()}
    grads = {n: nans((d,), weight) for n in (("q_weight", "k_weight") if norm != "none" else ())}
    torch.cuda.synchronize()
    if in_place:
        for n in ("q", "k"):
            out[n].copy_(dev[n])
        torch.cuda.synchronize()
        op.forward(out["q"], out["k"], out["q"], out["k"], **given)
        for n in ("dq", "dk"):
            out[n].copy_(dev[n])
        torch.cuda.synchronize()
        op.backward(dev["q"], dev["k"], out["dq"], out["dk"], out["dq"], out["dk"], grads=grads, **given)
    else:
        op.forward(dev["q"], dev["k"], out["q"], out["k"], **given)
        op.backward(dev["q"], dev["k"], dev["dq"], dev["dk"], out["dq"], out["dk"], grads=grads, **given)
    torch.cuda.synchronize()
    at = np.broadcast_to(np.arange(t), (b, t)) if positions is None else positions.numpy()
    angle = at[:, :, None, None].astype(np.float64) * f64(freq)
    for n in ("q", "k"):
        a, g = f64(x[n]), f64(x["d" + n])
        ww = f64(w[n + "_weight"]) if w else None
        how = (rotary, interleaved, norm == "rms", eps)
        want = A.head_norm(a, ww, angle, *how)
        plain = A.head_norm(a, ww, angle * 0, *how)
        A.near(f64(out[n]), want, n, A.HALF[dtype], 2.0 ** -19 * np.abs(plain).max(-1, keepdims=True))
        dx, dw, terms = A.head_norm(a, ww, angle, *how, dy=g)
        inv = 1.0 / np.sqrt((a * a).mean(-1, keepdims=True) + eps) if norm == "rms" else 1.0
        big = np.abs(g).max(-1, keepdims=True) * (1.0 if ww is None else np.abs(ww).max()) * inv
        # the part along x is at most its largest element by the mean's, which is at most big
        A.near(f64(out["d" + n]), dx, "d" + n, A.HALF[dtype], 2.0 ** -19 * big * (1 + np.abs(a * inv).max(-1, keepdims=True)))
        if norm == "rms":
            A.near(f64(grads[n + "_weight"]), dw, n + "_weight", A.HALF[weight], 2.0 ** -18 * terms)
    return out, grads


HEAD_CASES = [
    ((1, 1, 1, 1, 1), dict(rotary=0)),
    ((1, 1, 1, 1, 2), dict()),
    ((2, 5, 4, 2, 64), dict()),
    ((2, 5, 4, 2, 64), dict(interleaved=True)),
    ((2, 33, 3, 1, 128), dict(rotary=64)),
    ((2, 33, 3, 1, 128), dict(rotary=64, interleaved=True)),
    ((1, 70, 7, 5, 37), dict(rotary=20)),
    ((1, 70, 7, 5, 37), dict(rotary=14, interleaved=True)),
    ((1, 9, 2, 3, 320), dict(rotary=318)),
    ((1, 9, 2, 2, 512), dict()),
    ((1, 9, 2, 2, 511), dict(rotary=2, interleaved=True)),
    ((3, 11, 16, 2, 96), dict(norm="none")),
    ((3, 11, 16, 2, 96), dict(norm="none", rotary=0)),
    ((3, 11, 5, 2, 80), dict(weights=False)),
    ((1, 2100, 3, 2, 64), dict()),
    ((2, 1500, 5, 1, 24), dict(rotary=10, interleaved=True)),
]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape,how", HEAD_CASES)
def test_head_norm(device, dtype, shape, how):
    run_heads(dtype, *shape, **how)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_head_norm_weights_of_its_type(device, dtype):
    run_heads(dtype, 2, 50, 4, 2, 64, weight=dtype, seed=1)


@pytest.mark.parametrize("interleaved", [False, True])
def test_head_norm_far_positions(device, interleaved):
    """Of millions, and below zero: the angle has no rounding but the sine's."""
    p = torch.tensor([[0, 1 << 24, (1 << 31) - 1, -5], [999999, 7, 7, -(1 << 31)]], dtype=torch.int32)
    run_heads("f32", 2, 4, 3, 2, 64, interleaved=interleaved, positions=p, seed=2)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("how", [dict(), dict(interleaved=True, rotary=32)])
def test_head_norm_in_place(device, dtype, how):
    a, ga = run_heads(dtype, 2, 40, 4, 2, 72, seed=3, **how)
    b, gb = run_heads(dtype, 2, 40, 4, 2, 72, seed=3, in_place=True, **how)
    for x, y in ((a, b), (ga, gb)):
        for n in x:
            assert same(x[n], y[n]), n


def _guarded(x):
    b, t, h, d = x.shape
    return torch.empty(b, t, h + 1, d + 3, dtype=x.dtype, device="cuda")[:, :, :h, 1:1 + d].copy_(x)


def _head_major(x):
    return x.transpose(1, 2).contiguous().transpose(1, 2)


def _far_rows(x):
    b, t, h, d = x.shape
    whole = torch.empty((1 << 32) + t * h * d, dtype=x.dtype, device="cuda")
    return whole.as_strided((b, t, h, d), (1 << 32, h * d, d, 1)).copy_(x)


@pytest.mark.parametrize("layout", [_guarded, _head_major, _far_rows])
def test_head_norm_strides(device, layout):
    a, ga = run_heads("bf16", 2, 21, 3, 2, 64, seed=4)
    b, gb = run_heads("bf16", 2, 21, 3, 2, 64, seed=4, layout=layout)
    for x, y in ((a, b), (ga, gb)):
        for n in x:
            assert same(x[n], y[n]), n


def test_head_norm_one_gradient_and_none(device):
    """Of one weight only, and the same gradients of q and k without any."""
    op = O.HeadNorm("bf16", 2, 30, 4, 2, 64)
    x = [normal("bf16", 2, 30, c, 64, seed=5 + i).cuda() for i, c in enumerate((4, 2, 4, 2))]
    freq, w = torch.rand(32, device="cuda"), torch.rand(64, device="cuda")
    live = Buffer.live_count()
    got = []
    for names in ((), ("k_weight",), ("q_weight", "k_weight")):
        out, grads = [nans(y.shape, "bf16") for y in x[:2]], {n: nans((64,), "f32") for n in names}
        op.backward(*x, *out, frequencies=freq, q_weight=w, k_weight=w, grads=grads)
        torch.cuda.synchronize()
        assert Buffer.live_count() == live + (len(names) > 0)  # no workspace without a sum
        got.append((out, grads))
    for out, _ in got[1:]:
        assert same(out[0], got[0][0][0]) and same(out[1], got[0][0][1])
    assert same(got[1][1]["k_weight"], got[2][1]["k_weight"])
    op.free()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", [(0, 5, 2, 1, 16), (3, 0, 2, 1, 16)])
def test_head_norm_of_nothing(device, dtype, shape):
    """Gradients of the weights are zeros then."""
    op = O.HeadNorm(dtype, *shape)
    x = [torch.empty(shape[:2] + (c, 16), dtype=TYPES[dtype], device="cuda") for c in (2, 1)]
    grads = {n: nans((16,), "f32") for n in ("q_weight", "k_weight")}
    freq = torch.rand(8, device="cuda")
    op.forward(*x, *x, frequencies=freq)
    op.backward(*x, *x, *x, frequencies=freq, grads=grads)
    torch.cuda.synchronize()
    assert not any(g.any() for g in grads.values())


def test_head_norm_zeros_and_not_a_number(device):
    """A head of zeros stays one with a finite gradient; one that is not a
    number stays by itself."""
    op = O.HeadNorm("f32", 1, 6, 3, 1, 32)
    x = [normal("f32", 1, 6, c, 32, seed=6 + i).cuda() for i, c in enumerate((3, 1, 3, 1))]
    freq = torch.rand(16, device="cuda")

    def run():
        out = [nans(x[i % 2].shape, "f32") for i in range(4)]
        op.forward(*x[:2], *out[:2], frequencies=freq)
        op.backward(*x, *out[2:], frequencies=freq)
        torch.cuda.synchronize()
        return out

    want = run()
    x[0][0, 2, 1] = 0.0
    x[0][0, 4, 0, 3] = float("nan")
    got = run()
    assert not got[0][0, 2, 1].any() and torch.isfinite(got[2][0, 2, 1]).all()
    for i in (0, 2):
        assert torch.isnan(got[i][0, 4, 0]).all()
        for y in (got[i], want[i]):
            y[0, 2, 1] = y[0, 4, 0] = 0.0
        assert same(got[i], want[i]), i
    assert same(got[1], want[1])


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape,rotary", [((3, 1, 4, 2, 64), 64), ((2, 20, 4, 2, 40), 16), ((1, 2100, 2, 1, 16), 16)])
def test_head_norm_into_a_cache(device, dtype, shape, rotary):
    """k and v at the tokens' positions, nothing elsewhere, and nothing for
    positions outside it."""
    b, t, h, hk, d = shape
    keys = 2 * t + 5
    op = O.HeadNorm(dtype, b, t, h, hk, d, rotary=rotary, keys=keys)
    plain = O.HeadNorm(dtype, b, t, h, hk, d, rotary=rotary)
    q, k, v = (normal(dtype, b, t, c, d, seed=7 + i).cuda() for i, c in enumerate((h, hk, hk)))
    freq, w = torch.rand(rotary // 2, device="cuda"), torch.rand(d, device="cuda")
    order = torch.stack([torch.randperm(keys, generator=torch.Generator().manual_seed(i))[:t] for i in range(b)]).int()
    order[0, 0] = -1
    order[-1, -1] = keys if b > 1 or t > 1 else order[-1, -1]
    positions = order.cuda()
    want = [nans(y.shape, dtype) for y in (q, k)]
    plain.forward(q, k, *want, frequencies=freq, positions=positions, q_weight=w, k_weight=w)
    for with_k in (True, False):
        q_out, k_out = (nans(y.shape, dtype) for y in (q, k))
        caches = [torch.full((b, keys, hk, d), 5.0, dtype=TYPES[dtype], device="cuda") for _ in range(2)]
        op.forward(q, k, q_out, k_out if with_k else None, frequencies=freq, positions=positions, q_weight=w, k_weight=w, v=v,
                   k_cache=caches[0], v_cache=caches[1])
        torch.cuda.synchronize()
        assert same(q_out, want[0]) and (not with_k or same(k_out, want[1]))
        for cache, rows in zip(caches, (want[1], v)):
            full = torch.full((b, keys, hk, d), 5.0, dtype=TYPES[dtype], device="cuda")
            for i in range(b):
                inside = [(j, p) for j, p in enumerate(order[i].tolist()) if 0 <= p < keys]
                if inside:
                    full[i, [p for _, p in inside]] = rows[i, [j for j, _ in inside]]
            assert same(cache, full)


def test_head_norm_in_a_graph_and_on_streams(device):
    a, ga = run_heads("bf16", 2, 40, 4, 2, 64, seed=8)
    b, gb = run_heads("bf16", 2, 40, 4, 2, 64, seed=8, stream=torch.cuda.Stream())
    for x, y in ((a, b), (ga, gb)):
        for n in x:
            assert same(x[n], y[n]), n
    op = O.HeadNorm("bf16", 2, 40, 4, 2, 64)
    x = [normal("bf16", 2, 40, c, 64, seed=9 + i).cuda() for i, c in enumerate((4, 2, 4, 2))]
    y = [normal("bf16", 2, 40, c, 64, seed=19 + i).cuda() for i, c in enumerate((4, 2, 4, 2))]
    freq, w = torch.rand(32, device="cuda"), torch.rand(64, device="cuda")

    def run(v, out, grads, stream=None):
        op.forward(*v[:2], *out[:2], frequencies=freq, q_weight=w, k_weight=w, stream=stream)
        op.backward(*v, *out[2:], frequencies=freq, q_weight=w, k_weight=w, grads=grads, stream=stream)

    def fresh():
        return [nans(v.shape, "bf16") for v in x], {n: nans((64,), "f32") for n in ("q_weight", "k_weight")}

    want = []
    for v in (x, y):
        want.append(fresh())
        run(v, *want[-1])
    stream = torch.cuda.Stream()
    op.reserve(stream)
    held, out = [v.clone() for v in x], fresh()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        run(held, *out, stream=stream)
    for i in (0, 1, 0):
        for a, b in zip(held, (x, y)[i]):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(same(a, b) for a, b in zip(out[0], want[i][0]))
        assert all(same(out[1][n], want[i][1][n]) for n in out[1])
        run(y, *fresh())


# ---- embedding -------------------------------------------------------------------

def run_embedding(dtype, ids, vocab, width, weight=None, scale=1.0, accumulate=False, seed=0, gap=0):
    weight = weight or dtype
    tokens = len(ids)
    op = O.Embedding(dtype, tokens, vocab, width, scale=scale, weight_dtype=weight)

    def rows(x):
        whole = torch.full((x.shape[0], x.shape[1] + gap), 7.0, dtype=x.dtype, device="cuda")
        whole[:, :x.shape[1]].copy_(x)
        return whole, whole[:, :x.shape[1]]

    w, dout, before = (normal(k, n, width, seed=3 * seed + i) for i, (k, n) in enumerate(((weight, vocab), (dtype, tokens), (weight, vocab))))
    table, out, dw = rows(w)[1], rows(torch.full((tokens, width), float("nan"), dtype=TYPES[dtype])), rows(before)
    d_ids = torch.from_numpy(ids.astype(np.int32)).cuda()
    need = op.workspace_bytes(backward=True)
    guard = torch.full((need + 256,), 99, dtype=torch.uint8, device="cuda")
    op.forward(d_ids, table, out[1])
    op.backward(d_ids, rows(dout)[1], dw[1], accumulate=accumulate, workspace=guard[:need])
    torch.cuda.synchronize()
    assert (guard[need:] == 99).all() and (out[0][:, width:] == 7.0).all() and (dw[0][:, width:] == 7.0).all()
    s = float(np.float32(scale))
    A.near(f64(out[1]), A.embed(ids, f64(w), s), "out", A.HALF[dtype], 2.0 ** -24 * np.abs(A.embed(ids, f64(w), s)))
    want, terms = A.embed_back(ids, f64(dout), vocab, s)
    inside = ids[(ids >= 0) & (ids < vocab)]
    most = np.bincount(inside).max() if len(inside) else 0
    slack = (most + 3) * 2.0 ** -24 * terms
    if accumulate:
        there = np.isin(np.arange(vocab), inside)[:, None]
        want, slack = want + f64(before), slack + 2.0 ** -24 * (np.abs(f64(before)) + np.abs(want)) * there
        untouched = ~there[:, 0]
        assert (f64(dw[1])[untouched] == f64(before)[untouched]).all()
    A.near(f64(dw[1]), want, "dweight", A.HALF[weight], slack)
    return out[1], dw[1]


def ids_of(tokens, vocab, seed=0, skew=True):
    """As words come: some of them often."""
    g = np.random.default_rng(seed)
    x = g.random(tokens)
    return np.minimum((vocab * (x ** 4 if skew else x)).astype(np.int64), vocab - 1)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("tokens,vocab,width", [(1, 1, 1), (2, 7, 9), (300, 40, 64), (511, 2000, 33), (512, 5, 8), (513, 5, 8), (600, 1000, 100),
                                                (2049, 300, 65), (5000, 70000, 24), (16384, 900, 16), (16385, 900, 16), (20000, 300000, 8)])
def test_embedding(device, dtype, tokens, vocab, width):
    run_embedding(dtype, ids_of(tokens, vocab, seed=tokens), vocab, width, seed=1)


@pytest.mark.parametrize("tokens", [50, 700, 20000])
@pytest.mark.parametrize("weight,dtype", [("f32", "bf16"), ("f16", "f16"), ("f32", "f32")])
def test_embedding_accumulates_into_gaps(device, tokens, weight, dtype):
    """Scaled, rows apart, added to what is there; words of none stay."""
    run_embedding(dtype, ids_of(tokens, 1000, seed=2), 1000, 41, weight=weight, scale=-2.5, accumulate=True, seed=2, gap=5)
    run_embedding(dtype, ids_of(tokens, 1000, seed=2), 1000, 41, weight=weight, scale=6.5, seed=2, gap=3)


@pytest.mark.parametrize("tokens", [40, 3000, 30000])
def test_embedding_words_there_are_not(device, tokens):
    g = np.random.default_rng(3)
    ids = g.integers(-3, 13, tokens)
    ids[:4] = [-(1 << 31), (1 << 31) - 1, 10, -1]
    run_embedding("bf16", ids, 10, 20, seed=3)
    run_embedding("bf16", np.full(tokens, -1), 10, 20, seed=3)


@pytest.mark.parametrize("tokens,width", [(100, 8), (100, 2100), (2000, 8), (2000, 2100), (17000, 8)])
def test_embedding_runs_over_many_pieces(device, tokens, width):
    """One word for all tokens, and long runs that end and begin anywhere."""
    run_embedding("f32", np.full(tokens, 3), 5, width, seed=4)
    if width == 8:
        ids = np.sort(np.random.default_rng(4).integers(0, 20, tokens))
        run_embedding("f32", ids, 20, width, seed=4)
        run_embedding("f32", np.repeat(np.arange(tokens // 32 + 1), 32)[:tokens], tokens // 32 + 1, width, seed=4)


def test_embedding_is_deterministic(device):
    ids = ids_of(20000, 500, seed=5)
    a = run_embedding("f32", ids, 500, 64, seed=5)
    b = run_embedding("f32", ids, 500, 64, seed=5)
    assert same(a[0], b[0]) and same(a[1], b[1])


def test_embedding_of_nothing(device):
    op = O.Embedding("bf16", 0, 5, 8)
    dw = nans((5, 8), "bf16")
    ids, rows = torch.empty(0, dtype=torch.int32, device="cuda"), torch.empty(0, 8, dtype=torch.bfloat16, device="cuda")
    op.forward(ids, dw, rows)
    op.backward(ids, rows, dw, accumulate=True)
    torch.cuda.synchronize()
    assert torch.isnan(dw).all()
    op.backward(ids, rows, dw)
    torch.cuda.synchronize()
    assert not dw.any()


def test_embedding_tables_past_32_bits(device):
    """The last words of a table of 2^33 elements."""
    vocab, width = (1 << 20) + 3, 8192
    table = torch.empty(vocab, width, dtype=torch.float16, device="cuda")
    ids = np.array([vocab - 1, 5, vocab - 2, vocab - 1])
    rows = normal("f16", 3, width, seed=6).cuda()
    for i, w in enumerate((vocab - 1, 5, vocab - 2)):
        table[w] = rows[i]
    out = nans((4, width), "f16")
    d_ids = torch.from_numpy(ids.astype(np.int32)).cuda()
    op = O.Embedding("f16", 4, vocab, width)
    op.forward(d_ids, table, out)
    torch.cuda.synchronize()
    assert same(out, rows[[0, 1, 2, 0]])
    op.backward(d_ids, out, table)
    torch.cuda.synchronize()
    assert same(table[vocab - 2], rows[2]) and same(table[5], rows[1]) and same(table[vocab - 1], rows[0] * 2)
    assert not table[6:1000].any() and not table[vocab - 1000:vocab - 2].any()


@pytest.mark.parametrize("tokens", [200, 3000, 20000])
def test_embedding_in_a_graph(device, tokens):
    op = O.Embedding("bf16", tokens, 300, 40)
    runs = [(torch.from_numpy(ids_of(tokens, 300, seed=s).astype(np.int32)).cuda(), normal("bf16", tokens, 40, seed=s).cuda()) for s in (7, 8)]
    want = []
    for ids, dout in runs:
        want.append(nans((300, 40), "bf16"))
        op.backward(ids, dout, want[-1])
    ids, dout, dw = runs[0][0].clone(), runs[0][1].clone(), nans((300, 40), "bf16")
    stream = torch.cuda.Stream()
    op.reserve(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        op.backward(ids, dout, dw, stream=stream)
    for i in (0, 1, 0, 1):
        ids.copy_(runs[i][0])
        dout.copy_(runs[i][1])
        graph.replay()
        torch.cuda.synchronize()
        assert same(dw, want[i])
        dw.fill_(float("nan"))
        op.backward(*runs[1], nans((300, 40), "bf16"))


# ---- together --------------------------------------------------------------------

@pytest.mark.parametrize("dtype", list(TYPES))
def test_a_layer_forward_and_back(device, dtype):
    """Words to the table's gradient through all three operators, each against
    the 64-bit formula of what the one before it left."""
    b, t, h, hk, d, vocab = 2, 90, 4, 2, 32, 50
    g = np.random.default_rng(9)
    ids = torch.from_numpy(g.integers(0, vocab, b * t).astype(np.int32)).cuda()
    width = (h + 2 * hk) * d
    table, w = normal(dtype, vocab, width, seed=24).cuda(), (1 + 0.1 * normal("f32", 2, d, seed=25)).cuda()
    freq, do = torch.rand(d // 2, device="cuda"), normal(dtype, b, t, h, d, seed=26).cuda()
    embed, heads, attend = (O.Embedding(dtype, b * t, vocab, width), O.HeadNorm(dtype, b, t, h, hk, d), O.Attention(dtype, b, t, h, hk, d))
    x = nans((b * t, width), dtype)
    embed.forward(ids, table, x)
    split = lambda y: (y.view(b, t, h + 2 * hk, d)[:, :, :h], y.view(b, t, h + 2 * hk, d)[:, :, h:h + hk],  # noqa: E731
                       y.view(b, t, h + 2 * hk, d)[:, :, h + hk:])
    q, k, v = split(x)
    qr, kr, o = nans(q.shape, dtype), nans(k.shape, dtype), nans(q.shape, dtype)
    how = dict(frequencies=freq, q_weight=w[0], k_weight=w[1])
    heads.forward(q, k, qr, kr, **how)
    saved = torch.empty(attend.saved_bytes(), dtype=torch.uint8, device="cuda")
    attend.forward(qr, kr, v, o, saved=saved)
    dx, grads = nans(x.shape, dtype), {n: nans((d,), "f32") for n in ("q_weight", "k_weight")}
    dq, dk, dv = split(dx)
    attend.backward(qr, kr, v, o, do, saved, dq, dk, dv)
    torch.cuda.synchronize()
    dqr, dkr = dq.clone(), dk.clone()
    heads.backward(q, k, dq, dk, dq, dk, grads=grads, **how)  # in place
    dtable = nans(table.shape, dtype)
    embed.backward(ids, dx, dtable)
    torch.cuda.synchronize()
    n_ids = ids.cpu().numpy()
    A.near(f64(x), A.embed(n_ids, f64(table), 1.0), "x", A.HALF[dtype], 0.0)
    angle = np.arange(t)[None, :, None, None] * f64(freq)
    for y, r, dr, got, ww, dw in ((q, qr, dqr, dq, w[0], grads["q_weight"]), (k, kr, dkr, dk, w[1], grads["k_weight"])):
        want = A.head_norm(f64(y), f64(ww), angle, d, False, True, 1e-6)
        A.near(f64(r), want, "heads", A.HALF[dtype], 2.0 ** -19 * np.abs(want).max(-1, keepdims=True) * 1.5)
        dx_, dw_, terms = A.head_norm(f64(y), f64(ww), angle, d, False, True, 1e-6, dy=f64(dr))
        A.near(f64(dw), dw_, "weight", 2.0 ** -24, 2.0 ** -18 * terms)
        A.close(f64(got), dx_, "heads back", BOUND[dtype])
    parts = [A.attention(f64(qr)[i], f64(kr)[i], f64(v)[i], d ** -0.5, f64(do)[i]) for i in range(b)]
    for i, (n, got) in enumerate((("o", o), ("dq", dqr), ("dk", dkr), ("dv", dv))):
        c = 0.0 if i == 0 else np.sqrt(sum(p[4][i - 1] ** 2 for p in parts))
        off = 2.0 ** -22 * max(p[5] for p in parts)
        A.close(f64(got), np.stack([p[i] for p in parts]), n, (8e-6 if dtype == "f32" else BOUND[dtype]) + off, c * (1 + off / 4e-6))
    want, terms = A.embed_back(n_ids, f64(dx), vocab, 1.0)
    A.near(f64(dtable), want, "table", A.HALF[dtype], 32 * 2.0 ** -24 * terms)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_a_layer_token_by_token(device, dtype):
    """A prompt in two chunks into a cache and then a captured step replayed for
    each token, lengths and positions counted on the device, against the
    whole sequence in one call."""
    b, t, h, hk, d, keys = 2, 60, 8, 2, 64, 80
    qkv = normal(dtype, b, t, h + 2 * hk, d, seed=27).cuda()
    freq = torch.rand(d // 2, device="cuda")
    q, k, v = qkv[:, :, :h], qkv[:, :, h:h + hk], qkv[:, :, h + hk:]
    qr, kr, whole = nans(q.shape, dtype), nans(k.shape, dtype), nans(q.shape, dtype)
    O.HeadNorm(dtype, b, t, h, hk, d).forward(q, k, qr, kr, frequencies=freq)
    O.Attention(dtype, b, t, h, hk, d).forward(qr, kr, v, whole)
    kc, vc = nans((b, keys, hk, d), dtype), nans((b, keys, hk, d), dtype)
    got = nans(q.shape, dtype)
    for lo, hi in ((0, 33), (33, 50)):
        n = hi - lo
        at = torch.arange(lo, hi, dtype=torch.int32, device="cuda").repeat(b, 1)
        turned = nans((b, n, h, d), dtype)
        O.HeadNorm(dtype, b, n, h, hk, d, keys=keys).forward(q[:, lo:hi], k[:, lo:hi], turned, frequencies=freq, positions=at,
                                                             v=v[:, lo:hi], k_cache=kc, v_cache=vc)
        O.Attention(dtype, b, n, h, hk, d, keys=keys).forward(turned, kc, vc, got[:, lo:hi], lengths=i32(hi, hi))
        torch.cuda.synchronize()
    heads, attend = O.HeadNorm(dtype, b, 1, h, hk, d, keys=keys), O.Attention(dtype, b, 1, h, hk, d, keys=keys)
    one, turned, o = qkv[:, :1].clone(), nans((b, 1, h, d), dtype), nans((b, 1, h, d), dtype)
    position, lengths = torch.full((b, 1), 50, dtype=torch.int32, device="cuda"), i32(51, 51)
    stream = torch.cuda.Stream()
    attend.reserve(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        heads.forward(one[:, :, :h], one[:, :, h:h + hk], turned, frequencies=freq, positions=position, v=one[:, :, h + hk:],
                      k_cache=kc, v_cache=vc, stream=stream)
        attend.forward(turned, kc, vc, o, lengths=lengths, stream=stream)
        position.add_(1)
        lengths.add_(1)
    for i in range(50, t):
        one.copy_(qkv[:, i:i + 1])
        graph.replay()
        got[:, i:i + 1] = o
        torch.cuda.synchronize()
    assert same(kc[:, :t], kr) and same(vc[:, :t], v) and torch.isnan(kc[:, t:]).all()
    A.close(f64(got), f64(whole), "o", 2 * BOUND[dtype])  # each is BOUND off the formula


def test_attending_on_residents(device):
    """The framework's own buffers, no other library's tensors."""
    x = attention_arrays("f32", 1, 70, 2, 1, 16, seed=28)
    live = Buffer.live_count()
    res = {n: H.upload(np.ascontiguousarray(x[n].numpy())) for n in ("q", "k", "v")}
    freq = H.upload(np.linspace(1, 0.1, 8).astype(np.float32))
    heads, attend = O.HeadNorm("f32", 1, 70, 2, 1, 16, norm="none"), O.Attention("f32", 1, 70, 2, 1, 16)
    qr, kr, o = (O.Array.empty("f32", tuple(x[n].shape)) for n in ("q", "k", "q"))
    heads.forward(res["q"], res["k"], qr, kr, frequencies=freq)
    attend.forward(qr, kr, res["v"], o)
    Device.synchronize()
    got = np.empty((1, 70, 2, 16), np.float32)
    o.buf.download(got)
    angle = np.arange(70)[None, :, None, None] * np.linspace(1, 0.1, 8).astype(np.float32).astype(np.float64)
    a = {n: f64(v) for n, v in x.items()}
    turned = [A.head_norm(a[n], None, angle, 16, False, False, 0.0)[0] for n in ("q", "k")]
    A.close(got[0], A.attention(*turned, a["v"][0], 0.25), "o", 2 * BOUND["f32"])
    for r in list(res.values()) + [freq]:
        H.free_resident(r)
    for r in (qr, kr, o):
        r.free()
    heads.free()
    attend.free()
    assert Buffer.live_count() == live


# ---- the example -------------------------------------------------------------------

def _example_loss(z, w, ids, target, frequencies):
    """The example's layer in 64 bits."""
    rms = lambda x: x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6)  # noqa: E731
    split = lambda x, h: x.reshape(z.batch, z.tokens, h, z.head_dim)  # noqa: E731
    x = z.width ** 0.5 * w["words"][ids]
    n = rms(x) * w["first"]
    angle = np.arange(z.tokens)[None, :, None, None] * frequencies
    q, k = (A.head_norm(split(n @ w[a], h), w[b], angle, z.head_dim, False, True, 1e-6)
            for a, b, h in (("wq", "qn", z.heads), ("wk", "kn", z.kv_heads)))
    v = split(n @ w["wv"], z.kv_heads)
    o = np.stack([A.attention(q[i], k[i], v[i], z.head_dim ** -0.5) for i in range(z.batch)])
    y = o.reshape(len(ids), -1) @ w["wo"]
    m = rms(x + rms(y) * w["post"]) * w["pre"]
    return ((m @ w["we"] - target) ** 2).mean()


def test_the_example_runs_and_its_gradients(device):
    """Gradients of all weights against differences of the layer in 64 bits,
    whose own error is their step's square: with half the step a quarter, and
    so a third of what halving changes. What f32 is off by, in a chain of some
    twenty sums: 1e-5 of the gradient's norm."""
    from cudacaml_amd.examples import attention_layer as E

    z = E.Sizes()
    live = Buffer.live_count()
    layer = E.Layer(z)
    ids, target = E.recall_task(z, 1)
    for _ in range(3):
        assert np.isfinite(layer.step(ids, target))
    loss, grads = layer.gradients(ids, target)
    w = {n: v.astype(np.float64) for n, v in layer.weights.items()}
    f = lambda w: _example_loss(z, w, ids, target.astype(np.float64), layer.frequencies.astype(np.float64))  # noqa: E731
    assert abs(loss - f(w)) <= 1e-5 * abs(loss)
    assert set(grads) == set(w)
    g = np.random.default_rng(2)
    for n in grads:
        way = g.standard_normal(w[n].shape)
        slopes = [(f({**w, n: w[n] + h * way}) - f({**w, n: w[n] - h * way})) / (2 * h) for h in (1e-4, 5e-5)]
        off = abs((grads[n] * way).sum() - slopes[1])
        allowed = abs(slopes[0] - slopes[1]) + 1e-9 + 1e-5 * np.linalg.norm(grads[n]) * np.linalg.norm(way)
        assert off <= allowed, (n, off, allowed)
    a, b = layer.predict(ids), layer.evaluate(ids)
    assert np.abs(a - b).max() <= 1e-5 * np.abs(b).max()
    layer.release()
    del layer
    import gc

    gc.collect()
    assert Buffer.live_count() <= live
