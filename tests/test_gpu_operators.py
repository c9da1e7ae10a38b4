"""The layer operators on the device against the 64-bit references of
operator_reference.py.

Bounds, in the 2-norm over an output, from the formats alone:
- f32 results: a result passes through at most five chained sums of up to 128
  products; f32 sums of n terms are off by about sqrt(n) 2^-24 of their terms'
  norm, 7e-7 each, and 3.4e-6 together: 4e-6. The gradient of g sums 64 of
  such results once more: 8e-6.
- bf16 results are rounded to at most 2^-9 of themselves, and in the gated
  delta rule come through one operand that is rounded to as much: 2 x 2^-9.
  f16 results likewise: 2 x 2^-12, operands being kept to 16 bits or more. No
  f16 is nearer to a value below 2^-14 than half its step of 2^-24 there.
- results that a single element could dominate are also held element by
  element, to 16 times the bound of the larger of the value and the root mean
  square: what a rounding of one operand can do to a sum of few terms.
"""

import numpy as np
import pytest
import torch

import operator_reference as R
from cudacaml_amd import backend_hip as H
from cudacaml_amd import operators as O
from cudacaml_amd.runtime import Buffer, Device, Stream

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BOUND = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 4e-6}


def close(got, want, name, bound=None):
    bound = bound or BOUND[got.dtype]
    a, b = got.detach().double().cpu().numpy(), np.asarray(want, dtype=np.float64)
    assert a.shape == b.shape, name
    if not b.size:
        return
    assert np.isfinite(a).all(), name
    norm = np.linalg.norm(b)
    if norm == 0.0:
        assert not a.any(), name
        return
    rms = norm / np.sqrt(b.size)
    step = 2.0 ** -25 if got.dtype == torch.float16 else 0.0  # what the nearest f16 to a tiny value may be off
    miss = np.maximum(np.abs(a - b) - step, 0.0)
    off = np.linalg.norm(miss) / norm
    assert off <= bound, "%s is %.3g off, %.3g allowed" % (name, off, bound)
    most = (miss / np.maximum(np.abs(b), rms)).max()
    assert most <= 16 * bound, "%s has an element %.3g off, %.3g allowed" % (name, most, 16 * bound)


def arrays(dtype, batch, tokens, hk, hv, dk, dv, seed=0, states=0, back=False):
    """What a layer feeds the rule: unit keys and queries, decays and rates in
    0 .. 1, already rounded to the type."""
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    x = dict(q=torch.nn.functional.normalize(n(batch, tokens, hk, dk), dim=-1),
             k=torch.nn.functional.normalize(n(batch, tokens, hk, dk), dim=-1), v=n(batch, tokens, hv, dv),
             g=-torch.nn.functional.softplus(n(batch, tokens, hv) - 1.0), beta=torch.sigmoid(n(batch, tokens, hv)))
    if back:
        x["do"] = n(batch, tokens, hv, dv)
    x = {k: v.to(TYPES[dtype]) for k, v in x.items()}
    if states:
        x["state"] = n(states, hv, dk, dv) * 0.3
        if back:
            x["dstate_out"] = n(states, hv, dk, dv) * 0.3
    return x


def run_delta(x, dtype, cuts=None, back=False, layout=None, stream=None, handle=None, save=None):
    """Every output of the operator for CPU arrays x, as device tensors."""
    b, t, hk, dk = x["q"].shape
    hv, dv = x["v"].shape[2:]
    states = "state" in x
    op = handle or O.GatedDelta(dtype, b, t, hk, hv, dk, dv, sequences=None if cuts is None else len(cuts) - 1,
                                states=states)
    dev = {k: v.cuda() for k, v in x.items()}
    if layout:
        dev = layout(dev)
    e = torch.empty_like
    offsets = None if cuts is None else torch.tensor(cuts, dtype=torch.int32, device="cuda")
    out = {"o": torch.full((b, t, hv, dv), float("nan"), dtype=TYPES[dtype], device="cuda")}
    if states:
        out["state"] = torch.full_like(dev["state"], float("nan"))
    saved = None
    if back or save:
        saved = torch.full((op.saved_bytes(),), 255, dtype=torch.uint8, device="cuda")
    ins = [dev[n] for n in ("q", "k", "v", "g", "beta")]
    op.forward(*ins, out["o"], state=dev.get("state"), state_out=out.get("state"), offsets=offsets, saved=saved,
               stream=stream)
    if back:
        for n in ("q", "k", "v", "g", "beta"):
            out["d" + n] = torch.full(x[n].shape, float("nan"), dtype=TYPES[dtype], device="cuda")
        if states:
            out["dstate"] = e(out["state"])
        op.backward(*ins, dev["do"], saved, *(out["d" + n] for n in ("q", "k", "v", "g", "beta")),
                    dstate_out=dev.get("dstate_out"), dstate=out.get("dstate"), offsets=offsets, stream=stream)
    torch.cuda.synchronize()
    return out


def check_delta(x, dtype, cuts=None, back=False, **kw):
    got = run_delta(x, dtype, cuts, back, **kw)
    want = R.delta_batch({n: v.double().numpy() for n, v in x.items()}, cuts, x["q"].shape[3] ** -0.5,
                         x["state"].double().numpy() if "state" in x else None, back)
    for n, v in got.items():
        close(v, want[n], n, 8e-6 if n == "dg" and v.dtype == torch.float32 else None)
    return got


SHAPES = [  # batch, tokens, key heads, value heads, key_dim, value_dim
    (1, 1, 1, 1, 1, 1), (3, 1, 2, 4, 128, 128), (2, 2, 1, 2, 64, 64), (2, 8, 2, 2, 72, 100), (2, 9, 1, 1, 128, 64), (2, 16, 1, 2, 64, 96), (3, 17, 1, 1, 100, 40),
    (1, 63, 1, 2, 64, 32), (1, 64, 2, 2, 128, 128), (2, 65, 1, 4, 17, 250), (1, 130, 3, 3, 40, 33), (2, 200, 2, 4, 128, 96),
]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", SHAPES)
def test_gated_delta_forward(device, dtype, shape):
    check_delta(arrays(dtype, *shape, states=shape[0]), dtype)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", SHAPES)
def test_gated_delta_backward(device, dtype, shape):
    check_delta(arrays(dtype, *shape, seed=1, states=shape[0], back=True), dtype, back=True)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_gated_delta_without_states(device, dtype):
    check_delta(arrays(dtype, 2, 150, 2, 4, 128, 128, seed=2, back=True), dtype, back=True)
    check_delta(arrays(dtype, 2, 5, 2, 4, 64, 128, seed=2), dtype)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("cuts", [[0, 0], [0, 0, 1, 1, 64, 129, 129, 300], [0, 300], [0, 63, 64, 65, 192, 256, 299, 300]])
def test_gated_delta_packed(device, dtype, cuts):
    """Empty sequences, single tokens, ends inside and at chunks' ends; an
    empty one's last state is its first."""
    x = arrays(dtype, 1, max(cuts[-1], 1), 2, 4, 64, 72, seed=3, states=len(cuts) - 1, back=True)
    if cuts[-1] == 0:
        x = {k: v[:, :0] if v.dim() < 5 and "state" not in k else v for k, v in x.items()}
    got = check_delta(x, dtype, cuts, back=True)
    for i, (a, b) in enumerate(zip(cuts, cuts[1:])):
        if a == b:
            assert torch.equal(got["state"][i].cpu(), x["state"][i])
            assert torch.equal(got["dstate"][i].cpu(), x["dstate_out"][i])


def test_gated_delta_offsets_are_clamped(device):
    """Offsets below 0 or past the tokens count as those."""
    x = arrays("bf16", 1, 150, 1, 2, 32, 32, seed=17, states=3, back=True)
    a, b = run_delta(x, "bf16", [-7, 70, 150, 2000000000], back=True), run_delta(x, "bf16", [0, 70, 150, 150], back=True)
    for n in a:
        assert torch.equal(a[n], b[n]), n


def test_gated_delta_no_tokens(device):
    x = arrays("bf16", 2, 0, 1, 2, 32, 32, states=2)
    got = run_delta(x, "bf16")
    assert torch.equal(got["state"].cpu(), x["state"])


def test_gated_delta_state_in_place_and_one_token_at_a_time(device):
    """A prompt, then tokens one by one on the same state: as one sequence."""
    x = arrays("f32", 2, 100, 2, 4, 64, 64, seed=4, states=2)
    want = R.delta_batch({n: v.double().numpy() for n, v in x.items()}, None, 64 ** -0.5, x["state"].double().numpy(), False)
    dev = {k: v.cuda() for k, v in x.items()}
    state, o = dev["state"].clone(), torch.empty_like(dev["v"])
    part = lambda a, b: [dev[n][:, a:b] for n in ("q", "k", "v", "g", "beta")]  # noqa: E731
    O.GatedDelta("f32", 2, 70, 2, 4, 64, 64).forward(*part(0, 70), o[:, :70], state=state, state_out=state)
    one = O.GatedDelta("f32", 2, 1, 2, 4, 64, 64)
    for t in range(70, 97):
        one.forward(*part(t, t + 1), o[:, t:t + 1], state=state, state_out=state)
    O.GatedDelta("f32", 2, 3, 2, 4, 64, 64).forward(*part(97, 100), o[:, 97:], state=state, state_out=state)
    close(o, want["o"], "o")
    close(state, want["state"], "state")


def _from_one_projection(dev):
    """q, k and v as slices of one tensor, an odd number of elements apart."""
    b, t, hk, dk = dev["q"].shape
    hv, dv = dev["v"].shape[2:]
    whole = torch.full((b, t, 2 * hk * dk + hv * dv + 3), float("nan"), dtype=dev["q"].dtype, device="cuda")
    at = 1
    for n, h, d in (("q", hk, dk), ("k", hk, dk), ("v", hv, dv)):
        part = whole[:, :, at:at + h * d].unflatten(2, (h, d))
        part.copy_(dev[n])
        dev[n] = part
        at += h * d
    return dev


def _heads_first(dev):
    """Everything stored [batch, heads, tokens, ...]."""
    return {k: v.transpose(1, 2).contiguous().transpose(1, 2) if "state" not in k else v for k, v in dev.items()}


@pytest.mark.parametrize("layout", [_from_one_projection, _heads_first])
@pytest.mark.parametrize("shape", [(2, 70, 2, 4, 64, 96), (2, 70, 1, 2, 20, 12), (3, 3, 2, 2, 20, 12)])
def test_gated_delta_strides(device, layout, shape):
    """Views of any stride and alignment give what contiguous tensors give."""
    x = arrays("bf16", *shape, seed=5, states=shape[0], back=True)
    a = run_delta(x, "bf16", back=True)
    b = run_delta(x, "bf16", back=True, layout=layout)
    for n in a:
        assert torch.equal(a[n], b[n]), n


def _far_apart(tokens):
    """v, o's gradient and dv with tokens or rows of the batch so far apart
    that their last elements lie past 2^32 bytes (and 2^31 elements)."""
    def far(t):
        b, n, h, d = t.shape
        step = (1 << 23) if tokens else h * d
        row = n * step if tokens else (1 << 31) + 8
        whole = torch.empty((b - 1) * row + (n - 1) * step + h * d, dtype=t.dtype, device="cuda")
        part = whole.as_strided((b, n, h, d), (row, step, d, 1))
        part.copy_(t)
        return part

    return lambda dev: {k: far(v) if k in ("v", "do") else v for k, v in dev.items()}


@pytest.mark.parametrize("shape,tokens", [((2, 3, 1, 2, 32, 32), False), ((2, 300, 1, 2, 32, 32), False),
                                          ((2, 300, 1, 2, 32, 32), True)])
def test_gated_delta_tensors_past_32_bits(device, shape, tokens):
    x = arrays("bf16", *shape, seed=15, states=shape[0], back=True)
    a = run_delta(x, "bf16", back=shape[1] > 3)
    b = run_delta(x, "bf16", back=shape[1] > 3, layout=_far_apart(tokens))
    for n in a:
        assert torch.equal(a[n], b[n]), n


def test_gated_delta_writes_only_its_outputs(device):
    """Strided outputs: what lies between their elements keeps its value."""
    x = {k: v.cuda() for k, v in arrays("bf16", 2, 70, 2, 4, 40, 24, seed=6).items()}
    op = O.GatedDelta("bf16", 2, 70, 2, 4, 40, 24, states=False)
    wide = torch.full((2, 70, 4, 29), 7.0, dtype=torch.bfloat16, device="cuda")
    op.forward(*x.values(), wide[..., 2:26])
    plain = torch.empty(2, 70, 4, 24, dtype=torch.bfloat16, device="cuda")
    op.forward(*x.values(), plain)
    torch.cuda.synchronize()
    assert torch.equal(wide[..., 2:26], plain)
    assert bool((wide[..., :2] == 7).all()) and bool((wide[..., 26:] == 7).all())


@pytest.mark.parametrize("dtype", list(TYPES))
def test_gated_delta_extreme_gates(device, dtype):
    """Decays to nothing (g of -inf and of the type's lowest value forget the
    state), no decay, rates of 0 (a token that writes nothing still has a
    gradient of its rate) and of 1."""
    x = arrays(dtype, 2, 140, 1, 2, 64, 64, seed=7, states=2, back=True)
    x["g"][0, 10] = -float("inf")
    x["g"][0, 70:73] = torch.finfo(TYPES[dtype]).min
    x["g"][1, 20:90] = 0.0
    x["beta"][0, 30:40] = 0.0
    x["beta"][1, 64:100] = 1.0
    x["beta"][1, 127] = 0.0
    check_delta(x, dtype, back=True)


def test_gated_delta_equal_keys(device):
    """Keys that are all the same and rates of 1: the triangular systems are
    as far from the identity as they get."""
    x = arrays("f32", 1, 130, 1, 1, 32, 32, seed=8, states=1, back=True)
    x["k"] = x["k"][:, :1].expand_as(x["k"]).clone()
    x["beta"].fill_(1.0)
    x["g"].fill_(-1e-3)
    check_delta(x, "f32", back=True)


def test_gated_delta_large_values(device):
    """Values far from 1, as bf16 holds them: nothing inside has less range."""
    x = arrays("bf16", 1, 100, 1, 2, 64, 64, seed=9, back=True)
    x["v"] = (x["v"].float() * 1e20).bfloat16()
    x["do"] = (x["do"].float() * 1e-18).bfloat16()
    check_delta(x, "bf16", back=True)


def test_gated_delta_nan_stays_in_its_sequence(device):
    """A NaN reaches its own sequence and value heads and no chunk before its
    own in the forward pass."""
    cuts = [0, 100, 200, 300]
    x = arrays("bf16", 1, 300, 1, 2, 64, 64, seed=10, states=3, back=True)
    clean = run_delta(x, "bf16", cuts, back=True)
    x["v"][0, 170, 1, 3] = float("nan")
    got = run_delta(x, "bf16", cuts, back=True)
    same = torch.ones(300, dtype=torch.bool)
    same[100:200] = False
    for n in ("o", "dq", "dk", "dv", "dg", "dbeta"):
        assert torch.equal(got[n][:, same], clean[n][:, same]), n
    assert torch.equal(got["o"][:, 100:164], clean["o"][:, 100:164])
    assert torch.equal(got["o"][:, :, 0], clean["o"][:, :, 0])
    assert got["o"][0, 170, 1].isnan().any()
    assert torch.equal(got["state"][[0, 2]], clean["state"][[0, 2]])


def test_gated_delta_is_deterministic_and_handles_keep_nothing(device):
    """The same call twice gives the same bits, other calls between or not."""
    x = arrays("bf16", 2, 300, 2, 8, 128, 64, seed=11, back=True)
    y = arrays("bf16", 2, 300, 2, 8, 128, 64, seed=12, back=True)
    op = O.GatedDelta("bf16", 2, 300, 2, 8, 128, 64, states=False)
    a = run_delta(x, "bf16", back=True, handle=op)
    run_delta(y, "bf16", back=True, handle=op)
    b = run_delta(x, "bf16", back=True, handle=op)
    for n in a:
        assert torch.equal(a[n], b[n]), n


def test_gated_delta_differences(device):
    """The kernels' own forward pass against their gradient: a central
    difference of step h is off by h^2 times third derivatives (1e-4 for unit
    directions and h = 1e-2), and the f32 forward pass's rounding of about
    4e-6 of a sum of 2e4 terms' norm over 2 h adds as much: 2e-2 of the norm
    of gradient times direction."""
    x = arrays("f32", 1, 150, 1, 2, 32, 32, seed=13, states=1, back=True)
    got = run_delta(x, "f32", back=True)
    w = {n: v.double() for n, v in x.items()}

    def loss(name, value):
        out = run_delta({**x, name: value.float()}, "f32")
        return float((out["o"].double().cpu() * w["do"]).sum() + (out["state"].double().cpu() * w["dstate_out"]).sum())

    g = torch.Generator().manual_seed(1)
    for n, at in (("q", "dq"), ("k", "dk"), ("v", "dv"), ("g", "dg"), ("beta", "dbeta"), ("state", "dstate")):
        d = torch.randn(x[n].shape, generator=g, dtype=torch.float64)
        d /= d.norm()
        h = 1e-2
        want = (loss(n, w[n] + h * d) - loss(n, w[n] - h * d)) / (2 * h)
        grad = got[at].double().cpu()
        assert abs(float((grad * d).sum()) - want) <= 2e-2 * max(1.0, float(grad.norm())), n


def test_gated_delta_on_another_stream(device):
    """Work on a stream of its own, its workspace with it, next to other work
    on the default stream with the same handle."""
    x = arrays("bf16", 2, 200, 2, 4, 64, 64, seed=14, states=2, back=True)
    op = O.GatedDelta("bf16", 2, 200, 2, 4, 64, 64)
    want = run_delta(x, "bf16", back=True, handle=op)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for stream in (side, Stream.create(), side.cuda_stream):
        got = run_delta(x, "bf16", back=True, handle=op, stream=stream)
        for n in want:
            assert torch.equal(got[n], want[n]), n


def test_gated_delta_in_a_graph(device):
    """Captured once and replayed on new inputs, with eager calls between."""
    shape = (2, 130, 1, 2, 64, 64)
    op = O.GatedDelta("bf16", *shape, states=False)
    one, two = (arrays("bf16", *shape, seed=s, back=True) for s in (15, 16))
    want = [run_delta(x, "bf16", back=True) for x in (one, two)]
    dev = {k: v.cuda() for k, v in one.items()}
    names = ("q", "k", "v", "g", "beta")
    out = {"o": torch.empty_like(dev["v"]), **{"d" + n: torch.empty_like(dev[n]) for n in names}}
    saved = torch.empty(op.saved_bytes(), dtype=torch.uint8, device="cuda")
    stream = torch.cuda.Stream()
    op.reserve(stream, backward=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        op.forward(*(dev[n] for n in names), out["o"], saved=saved, stream=stream)
        op.backward(*(dev[n] for n in names), dev["do"], saved, *(out["d" + n] for n in names), stream=stream)
    for i in (0, 1, 0, 1):
        for n, v in (one, two)[i].items():
            dev[n].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        for n in out:
            assert torch.equal(out[n], want[i][n]), (i, n)
        run_delta(two, "bf16", back=True)


def test_operators_on_residents(device):
    """The framework's own buffers, no other library's tensors."""
    x = arrays("f32", 1, 70, 1, 1, 16, 16, seed=17)
    live = Buffer.live_count()
    res = {k: H.upload(np.ascontiguousarray(v.numpy())) for k, v in x.items()}
    o = O.Array.empty("f32", (1, 70, 1, 16))
    op = O.GatedDelta("f32", 1, 70, 1, 1, 16, 16, states=False)
    op.forward(*res.values(), o)
    Device.synchronize()
    got = np.empty((1, 70, 1, 16), np.float32)
    o.buf.download(got)
    want = R.delta_batch({n: v.double().numpy() for n, v in x.items()}, None, 0.25, None, False)
    close(torch.from_numpy(got), want["o"], "o")
    for r in res.values():
        H.free_resident(r)
    o.free()
    op.free()
    assert Buffer.live_count() == live


# ---- norm block --------------------------------------------------------------

def norm_arrays(dtype, weight, rows, width, norm, pre, gate, residual=True, bias=True, channel=True, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    x = dict(y=n(rows, width), dh=n(rows, width))
    if gate != "none":
        x["gate"] = n(rows, width)
    if residual:
        x["residual"] = 2 * n(rows, width)
    if pre != "none":
        x.update(dn=n(rows, width), h=2 * n(rows, width) + 0.5)
    x = {k: v.to(TYPES[dtype]) for k, v in x.items()}
    w = {}
    if norm != "none":
        w["post_weight"] = 1 + 0.1 * n(width)
        if bias:
            w["post_bias"] = 0.1 * n(width)
    if pre != "none":
        w["pre_weight"] = 1 + 0.1 * n(width)
        if bias:
            w["pre_bias"] = 0.1 * n(width)
    if channel:
        w["channel_scale"] = 1 + 0.1 * n(width)
    return x, {k: v.to(TYPES[weight]) for k, v in w.items()}


def check_norm(dtype, weight, rows, width, norm, pre, gate, p=0.2, view=lambda t: t, change=None, **kw):
    x, w = norm_arrays(dtype, weight, rows, width, norm, pre, gate, **kw)
    if change:
        change(x, w)
    seed, offset = 0x1234567890ABCDEF, 1 << 33
    op = O.NormBlock(dtype, rows, width, norm=norm, pre=pre, gate=gate, dropout=p, scale=0.7, eps=1e-5, weight_dtype=weight)
    dev, wd = {k: view(v.cuda()) for k, v in x.items()}, {k: v.cuda() for k, v in w.items()}
    wide = {k: v.double().numpy() for k, v in {**x, **w}.items()}
    how = (norm, pre, gate, 0.7, 1e-5, p, seed, offset)
    empty = lambda: view(torch.full((rows, width), float("nan"), dtype=TYPES[dtype], device="cuda"))  # noqa: E731
    got = {"h": empty()}
    if pre != "none":
        got["n"] = empty()
    op.forward(dev["y"], got["h"], got.get("n"), gate=dev.get("gate"), residual=dev.get("residual"), seed=seed,
               offset=offset, **wd)
    torch.cuda.synchronize()
    for n, want in R.norm_block(wide, *how).items():
        close(got[n], want, n)
    out = {"y": empty()}
    if "gate" in x:
        out["gate"] = empty()
    if "residual" in x:
        out["residual"] = empty()
    grads = {n: torch.full_like(v, float("nan")) for n, v in wd.items()}
    op.backward(dev["y"], dev["dh"], out["y"], dn=dev.get("dn"), h=dev.get("h"), gate=dev.get("gate"),
                dgate=out.get("gate"), dresidual=out.get("residual"), grads=grads, seed=seed, offset=offset, **wd)
    torch.cuda.synchronize()
    want = R.norm_block(wide, *how, back=True)
    for n, v in {**out, **grads}.items():
        close(v, want[n], n)


NORMS = [  # rows, width, norm, pre, gate
    (1, 1, "rms", "rms", "none"), (5, 3, "layer", "layer", "sigmoid"), (33, 16, "rms", "none", "silu"),
    (70, 128, "rms", "rms", "silu"), (9, 129, "layer", "rms", "none"), (6, 512, "none", "layer", "silu"),
    (5, 513, "rms", "rms", "sigmoid"), (3, 2048, "layer", "layer", "silu"), (4, 2049, "rms", "rms", "none"),
    (3, 4096, "rms", "rms", "silu"), (2, 5000, "layer", "rms", "none"), (2, 8192, "rms", "layer", "sigmoid"),
    (2, 10001, "rms", "rms", "silu"), (1, 16384, "layer", "layer", "none"), (1, 20000, "rms", "rms", "silu"),
    (1, 32768, "layer", "layer", "silu"), (17, 40, "none", "none", "silu"),
]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("case", NORMS)
def test_norm_block(device, dtype, case):
    check_norm(dtype, "f32", *case)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("kw", [dict(), dict(bias=False), dict(channel=False), dict(residual=False, p=0.0),
                                dict(bias=False, channel=False, p=1.0)])
def test_norm_block_parameters(device, dtype, kw):
    """Parameters in the type of the rows, and each of them left out."""
    check_norm(dtype, dtype, 37, 200, "layer", "rms", "silu", seed=1, **kw)
    check_norm(dtype, dtype, 37, 1000, "rms", "layer", "none", seed=2, **kw)


def test_norm_block_many_rows(device):
    """More rows than workgroups: the parameters' gradients are sums over
    workgroups, and two runs give the same bits."""
    check_norm("f32", "f32", 5003, 24, "rms", "rms", "silu", seed=3)
    x, w = norm_arrays("bf16", "f32", 6007, 640, "rms", "rms", "none", seed=4)
    op = O.NormBlock("bf16", 6007, 640, dropout=0.1)
    dev, wd = {k: v.cuda() for k, v in x.items()}, {k: v.cuda() for k, v in w.items()}
    runs = []
    for _ in range(2):
        grads = {n: torch.empty_like(v) for n, v in wd.items()}
        op.backward(dev["y"], dev["dh"], torch.empty_like(dev["y"]), dn=dev["dn"], h=dev["h"], grads=grads, seed=5, **wd)
        torch.cuda.synchronize()
        runs.append(grads)
    for n in wd:
        assert torch.equal(runs[0][n], runs[1][n]), n


def test_norm_block_strided_rows(device):
    """Rows an odd number of elements apart, at odd addresses."""
    def view(t):
        wide = torch.full((t.shape[0], t.shape[1] + 5), float("nan"), dtype=t.dtype, device="cuda")
        part = wide[:, 3:3 + t.shape[1]]
        part.copy_(t)
        return part

    check_norm("bf16", "f32", 11, 136, "rms", "layer", "silu", view=view, seed=6)
    check_norm("f32", "f32", 11, 77, "layer", "rms", "none", view=view, seed=7)


def test_rows_past_32_bits(device):
    """Rows 2^30 + 9 elements apart: the last of them past 2^32 bytes."""
    def view(t):
        whole = torch.empty((t.shape[0] - 1) * ((1 << 30) + 9) + t.shape[1], dtype=t.dtype, device="cuda")
        part = whole.as_strided(tuple(t.shape), ((1 << 30) + 9, 1))
        part.copy_(t)
        return part

    check_norm("bf16", "f32", 4, 136, "rms", "layer", "silu", view=view, seed=6)
    x = torch.randn(4, 100, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    far, out = view(x.cuda()), view(torch.zeros(4, 100, dtype=torch.bfloat16, device="cuda"))
    O.Dropout("bf16", 4, 100, 0.3).forward(far, out, seed=5, offset=6)
    torch.cuda.synchronize()
    close(out, R.drop(x.double().numpy(), 0.3, 5, 6), "out")


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("how", [("rms", "rms", "none"), ("layer", "layer", "silu"), ("layer", "none", "sigmoid")])
def test_norm_block_many_wide_rows(device, dtype, how):
    """Over 8192 columns the parameters' gradients are summed apart."""
    check_norm(dtype, "f32", 70, 8200, *how, seed=16)


def test_norm_block_rows_of_zeros_and_constants(device):
    """A row of zeros has eps to divide by; a layer norm centres a constant
    row to nothing."""
    def change(x, w):
        x["y"][1] = 0.0
        x["y"][2] = 5.0
        x["h"][1] = 0.0

    check_norm("f32", "f32", 4, 64, "layer", "rms", "none", change=change, seed=8)


def test_norm_block_in_place(device):
    """h over the residual and n over y, as an inference loop keeps them."""
    x, w = norm_arrays("bf16", "f32", 20, 300, "rms", "rms", "none", seed=9)
    op = O.NormBlock("bf16", 20, 300)
    dev, wd = {k: v.cuda() for k, v in x.items()}, {k: v.cuda() for k, v in w.items()}
    h, n = torch.empty_like(dev["y"]), torch.empty_like(dev["y"])
    op.forward(dev["y"], h, n, residual=dev["residual"], **wd)
    y, r = dev["y"].clone(), dev["residual"].clone()
    op.forward(y, r, y, residual=r, **wd)
    torch.cuda.synchronize()
    assert torch.equal(r, h) and torch.equal(y, n)


def test_norm_block_differences(device):
    """As for the gated delta rule: a step of 1e-2 along unit directions; sums
    of 1000 results of size 1 are off by 1e-7 x 30 / 2e-2 = 2e-4 and third
    derivatives by 1e-4: 1e-2 of the norms."""
    x, w = norm_arrays("f32", "f32", 12, 80, "layer", "rms", "silu", seed=10)
    op = O.NormBlock("f32", 12, 80, norm="layer", pre="rms", gate="silu", dropout=0.3, scale=0.7, eps=1e-5)
    inputs = {k: x[k] for k in ("y", "gate", "residual")}

    def forward(a):
        d = {k: v.float().cuda() for k, v in a.items()}
        h, n = torch.empty(12, 80, device="cuda"), torch.empty(12, 80, device="cuda")
        op.forward(d["y"], h, n, gate=d["gate"], residual=d["residual"], seed=3, **{k: d[k] for k in w})
        torch.cuda.synchronize()
        return h, n

    h, _ = forward({**inputs, **w})
    dev, wd = {k: v.cuda() for k, v in x.items()}, {k: v.cuda() for k, v in w.items()}
    out = {k: torch.empty(12, 80, device="cuda") for k in inputs}
    grads = {k: torch.empty_like(v) for k, v in wd.items()}
    op.backward(dev["y"], dev["dh"], out["y"], dn=dev["dn"], h=h, gate=dev["gate"], dgate=out["gate"],
                dresidual=out["residual"], grads=grads, seed=3, **wd)
    torch.cuda.synchronize()
    g = torch.Generator().manual_seed(2)
    for n, grad in {**out, **grads}.items():
        base = {k: v.double() for k, v in {**inputs, **w}.items()}
        d = torch.randn(base[n].shape, generator=g, dtype=torch.float64)
        d /= d.norm()
        step = 1e-2

        def loss(sign):
            a, b = forward({**base, n: base[n] + sign * step * d})
            return float((a.double().cpu() * x["dh"].double()).sum() + (b.double().cpu() * x["dn"].double()).sum())

        want = (loss(1) - loss(-1)) / (2 * step)
        grad = grad.double().cpu()
        assert abs(float((grad * d).sum()) - want) <= 1e-2 * max(1.0, float(grad.norm())), n


def test_norm_block_no_rows(device):
    """No rows: parameters' gradients are zero, nothing else is written."""
    op = O.NormBlock("f32", 0, 16)
    z = torch.empty(0, 16, device="cuda")
    grads = {n: torch.full((16,), float("nan"), device="cuda") for n in ("post_weight", "pre_weight")}
    op.forward(z, z, z)
    op.backward(z, z, z, dn=z, h=z, grads=grads)
    torch.cuda.synchronize()
    assert not grads["post_weight"].any() and not grads["pre_weight"].any()


# ---- dropout -----------------------------------------------------------------

@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (2, 8), (5, 21), (33, 64), (4, 1001), (700, 3)])
@pytest.mark.parametrize("p", [0.0, 0.3, 1.0])
def test_dropout(device, dtype, shape, p):
    """The reference's mask exactly, forward and backward, with a residual."""
    g = torch.Generator().manual_seed(4)
    x, r = (torch.randn(shape, generator=g).to(TYPES[dtype]) for _ in range(2))
    seed, offset = 0xFFFFFFFF00000001, 0x1FFFFFFFF
    op = O.Dropout(dtype, *shape, p, scale=0.5)
    xd, rd, out, dx = x.cuda(), r.cuda(), torch.empty(shape, dtype=TYPES[dtype], device="cuda"), None
    op.forward(xd, out, seed=seed, offset=offset, residual=rd)
    keep, up = R.kept(*shape, p, seed, offset)
    want = r.double().numpy() + 0.5 * R.drop(x.double().numpy(), p, seed, offset)
    torch.cuda.synchronize()
    close(out, want, "out")
    dx = torch.empty_like(out)
    op.backward(xd, dx, seed=seed, offset=offset)
    torch.cuda.synchronize()
    assert np.array_equal(dx.double().cpu().numpy() != 0, keep & (x.double().numpy() != 0))
    close(dx, 0.5 * R.drop(x.double().numpy(), p, seed, offset), "dx")


def test_dropout_drops_what_is_not_a_number(device):
    """A dropped infinity or NaN is zero; a kept one stays."""
    x = torch.full((4, 64), float("inf"), device="cuda")
    x[1::2] = float("nan")
    out = torch.empty_like(x)
    O.Dropout("f32", 4, 64, 0.5).forward(x, out, seed=9)
    keep, _ = R.kept(4, 64, 0.5, 9, 0)
    torch.cuda.synchronize()
    got = out.cpu().numpy()
    assert (got[~keep] == 0).all() and not np.isfinite(got[keep]).any()


def test_dropout_rate_seeds_and_offsets(device):
    """About p of many values are dropped (5 sigma), and other seeds and
    offsets drop others: two masks agree where independent ones would."""
    n, p = 1 << 20, 0.3
    x = torch.ones(1024, 1024, device="cuda")
    masks = []
    for seed, offset in ((1, 0), (2, 0), (1, 1)):
        out = torch.empty_like(x)
        O.Dropout("f32", 1024, 1024, p).forward(x, out, seed=seed, offset=offset)
        masks.append(out != 0)
    torch.cuda.synchronize()
    for m in masks:
        assert abs(float(m.double().mean()) - (1 - p)) < 5 * (p * (1 - p) / n) ** 0.5
    agree = p * p + (1 - p) * (1 - p)
    for m in masks[1:]:
        assert abs(float((m == masks[0]).double().mean()) - agree) < 5 * (agree * (1 - agree) / n) ** 0.5


def test_dropout_step_on_the_device(device):
    """A captured call draws anew on each replay through its step word, and as
    an eager call with that offset; strides do not change a mask; in place."""
    x = torch.randn(50, 70, device="cuda")
    step = torch.zeros((), dtype=torch.int64, device="cuda")
    out = torch.empty_like(x)
    op = O.Dropout("f32", 50, 70, 0.4)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        op.forward(x, out, seed=3, offset=10, step=step, stream=stream)
        step.add_(1)
    for i in range(4):
        graph.replay()
        torch.cuda.synchronize()
        wide = torch.zeros(50, 75, device="cuda")
        wide[:, 2:72] = x
        op.forward(wide[:, 2:72], wide[:, 2:72], seed=3, offset=10 + i)
        torch.cuda.synchronize()
        assert torch.equal(wide[:, 2:72], out), i
        assert not wide[:, :2].any() and not wide[:, 72:].any()


def test_the_example_learns_and_serves(device):
    """A recurrent layer trained on graphs and operators: its loss falls, and
    token by token it gives what whole sequences give."""
    from cudacaml_amd.examples import delta_layer as E

    z = E.Sizes()
    live = Buffer.live_count()
    layer = E.Layer(z)
    x, target = E.recall_task(z, 1)
    losses = [layer.step(x, target, seed=i) for i in range(12)]
    assert losses[-1] < 0.75 * losses[0], losses
    a, b = layer.predict(x), layer.evaluate(x)
    assert np.abs(a - b).max() <= 1e-4 * np.abs(b).max()
    layer.release()
    del layer
    import gc

    gc.collect()
    assert Buffer.live_count() <= live


# ---- workspaces of captured calls --------------------------------------------

def test_a_graph_keeps_its_workspace(device):
    """A captured forward pass with eager backward passes of the same handle on
    the same stream between its replays, which need a larger workspace."""
    shape = (2, 130, 1, 2, 64, 64)
    op = O.GatedDelta("bf16", *shape, states=False)
    one, two = (arrays("bf16", *shape, seed=s, back=True) for s in (31, 32))
    want = [run_delta(x, "bf16", back=True) for x in (one, two)]
    dev = {k: v.cuda() for k, v in one.items()}
    names = ("q", "k", "v", "g", "beta")
    o = torch.empty_like(dev["v"])
    stream = torch.cuda.Stream()
    op.reserve(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        op.forward(*(dev[n] for n in names), o, stream=stream)
    for i in (0, 1, 0, 1):
        for n, v in (one, two)[i].items():
            dev[n].copy_(v)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want[i]["o"]), i
        with torch.cuda.stream(stream):
            got = run_delta(two, "bf16", back=True, handle=op, stream=stream)
            run_delta(two, "bf16", handle=op, stream=stream)
        for n in got:
            assert torch.equal(got[n], want[1][n]), n


def test_a_graph_with_the_callers_workspace(device):
    """Such a graph outlives its handle and may run on any stream, with calls
    on the capture stream next to it."""
    shape = (2, 130, 1, 2, 64, 64)
    op = O.GatedDelta("f32", *shape, states=False)
    x = arrays("f32", *shape, seed=33)
    want = run_delta(x, "f32")["o"]
    dev = {k: v.cuda() for k, v in x.items()}
    o = torch.empty_like(want)
    work = torch.empty(op.workspace_bytes(), dtype=torch.uint8, device="cuda")
    stream, other = torch.cuda.Stream(), torch.cuda.Stream()
    live = Buffer.live_count()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        op.forward(*dev.values(), o, workspace=work, stream=stream)
    assert Buffer.live_count() == live
    op.free()
    del op
    for _ in range(3):
        o.fill_(float("nan"))
        torch.cuda.synchronize()
        with torch.cuda.stream(other):
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want)
        with torch.cuda.stream(stream):
            assert torch.equal(run_delta(x, "f32", stream=stream)["o"], want)


# ---- nothing to go back through ----------------------------------------------

@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", [(2, 0, 1, 2, 32, 32), (3, 0, 2, 2, 100, 40)])
def test_gated_delta_backward_of_no_tokens(device, dtype, shape):
    """Rows without tokens: the last states' gradient is that of the first."""
    x = arrays(dtype, *shape, states=shape[0], back=True)
    got = run_delta(x, dtype, back=True)
    assert torch.equal(got["dstate"].cpu(), x["dstate_out"]) and torch.equal(got["state"].cpu(), x["state"])
    got = run_delta({n: v for n, v in x.items() if n != "dstate_out"}, dtype, back=True)
    assert not got["dstate"].any()


# ---- the triangular systems --------------------------------------------------

@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("dims", [(64, 32), (128, 64), (40, 20)])
def test_gated_delta_inverses_reach_across_a_chunk(device, dtype, dims):
    """Equal keys, rates of 0.05 and hardly a decay: (I + A)^-1 falls by 5% a
    token, so that every block of it, the one 48 tokens off the diagonal too,
    is in the results."""
    x = arrays(dtype, 2, 130, 1, 2, *dims, seed=34, states=2, back=True)
    x["k"] = x["k"][:, :1].expand_as(x["k"]).clone()
    x["beta"].fill_(0.05)
    x["g"].fill_(-1e-3)
    check_delta(x, dtype, back=True)


# ---- products of f16 inputs --------------------------------------------------

@pytest.mark.parametrize("dims,back", [((64, 64), False), ((128, 32), False), ((128, 32), True), ((20, 12), False),
                                       ((20, 12), True)])
def test_gated_delta_f16_products_are_whole(device, dims, back):
    """Keys and queries whose every element has the same last bits: of k . k,
    the product of what eight bits leave of each is 1.5e-5 and always of one
    sign. A state that misses it is 0.7e-5 to 3e-5 off, where an f32 state's
    bound is 4e-6. (No gradients where k . k is 1: with a rate of 1 a token then
    takes back all that came before it along k, and they are differences that
    hold no digit of their terms.)"""
    x = arrays("f16", 1, 130, 1, 2, *dims, seed=35, states=1, back=back)
    for n in ("q", "k"):
        x[n].fill_(2.0 ** round(-0.5 * np.log2(dims[0])) * (1.0 + 4.0 / 1024.0))
    x["beta"].fill_(1.0)
    x["g"].fill_(-0.05)
    check_delta(x, "f16", back=back)


# ---- more workgroups than a launch has along one axis ------------------------

def test_dropout_of_more_rows_than_a_launch_has_work_items(device):
    """2^32 - 1 rows of one column, in place: rows at the ends and around each
    2^30th against the generator, and about p of all of them dropped."""
    rows, p, seed, offset = (1 << 32) - 1, 0.25, 0x123456789, 7
    x = torch.ones(rows, 1, dtype=torch.bfloat16, device="cuda")
    O.Dropout("bf16", rows, 1, p).forward(x, x, seed=seed, offset=offset)
    torch.cuda.synchronize()
    for at in (0, (1 << 30) - 50, (1 << 31) - 50, 3 * (1 << 30) - 50, rows - 100):
        got = x[at:at + 100, 0].float().cpu().numpy()
        low = [R.philox((0, r, offset, 0), (seed & R.LOW, seed >> 32))[0] & 0xFFFF for r in range(at, at + 100)]
        want = np.where(np.array(low) >= 16384, float(torch.tensor(4 / 3).bfloat16()), 0.0)
        assert np.array_equal(got, want), at
    kept = sum(int((x[at:at + (1 << 28)] != 0).sum()) for at in range(0, rows, 1 << 28))
    assert abs(kept / rows - 0.75) < 5 * (0.1875 / rows) ** 0.5
    del x
    torch.cuda.empty_cache()


def test_dropout_of_the_longest_rows(device):
    """2^35 - 3 columns, in place: 2^32 groups of eight, the last one short."""
    cols, seed = (1 << 35) - 3, 99
    x = torch.ones(1, cols, dtype=torch.float16, device="cuda")
    O.Dropout("f16", 1, cols, 0.5).forward(x, x, seed=seed)
    torch.cuda.synchronize()
    for group in (0, (1 << 30) + 1, 1 << 31, (1 << 32) - 1):
        got = x[0, 8 * group:8 * group + 8].float().cpu().numpy()
        words = R.philox((group, 0, 0, 0), (seed, 0))
        halves = [h for w in words for h in (w & 0xFFFF, w >> 16)][:len(got)]
        assert np.array_equal(got, [2.0 * (h >= 32768) for h in halves]), group
    assert len(got) == 5
    del x
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", list(TYPES))
def test_gated_delta_more_heads_than_a_launch_has_workgroups(device, dtype):
    """One token of 2^24 + 32 states of one element."""
    b, h = (1 << 19) + 1, 32
    g = torch.Generator(device="cuda").manual_seed(3)
    r = lambda *s: torch.randn(s, generator=g, device="cuda").to(TYPES[dtype])  # noqa: E731
    q, k, v, a, beta = r(b, 1, 1, 1), r(b, 1, 1, 1), r(b, 1, h, 1), -r(b, 1, h).abs(), r(b, 1, h).sigmoid()
    state = torch.randn(b, h, 1, 1, generator=g, device="cuda")
    o, end = torch.empty_like(v), torch.empty_like(state)
    O.GatedDelta(dtype, b, 1, 1, h, 1, 1, scale=0.5).forward(q, k, v, a, beta, o, state=state, state_out=end)
    torch.cuda.synchronize()
    s = a.double().exp()[:, 0] * state.double()[..., 0, 0]
    s = s + k.double()[:, 0, :, 0] * beta.double()[:, 0] * (v.double()[:, 0, :, 0] - s * k.double()[:, 0, :, 0])
    close(end[..., 0, 0], s.cpu().numpy(), "state")
    close(o[:, 0, :, 0], (0.5 * s * q.double()[:, 0, :, 0]).cpu().numpy(), "o")


def test_gated_delta_more_column_blocks_than_a_launch_has_workgroups(device):
    """4096 sequences, all but a few empty, of 32 heads of 4096 columns."""
    n, hv, dv, tokens = 4096, 32, 4096, 70
    x = {k: v.cuda() for k, v in arrays("bf16", 1, tokens, 1, hv, 16, dv, seed=36).items()}
    cuts = [0, 3] + [3] * (n // 2) + [20] * (n // 2 - 2) + [tokens]
    out = []
    for c in (cuts, [0, 3, 20, tokens]):
        o = torch.full_like(x["v"], float("nan"))
        op = O.GatedDelta("bf16", 1, tokens, 1, hv, 16, dv, sequences=len(c) - 1, states=False)
        op.forward(*x.values(), o, offsets=torch.tensor(c, dtype=torch.int32, device="cuda"))
        torch.cuda.synchronize()
        op.free()
        out.append(o)
    assert torch.equal(out[0], out[1])


# ---- 32 value columns a workgroup, wide heads --------------------------------

MANY = [  # more than 128 blocks of 32 value columns, so that a workgroup takes 32 (whole heads, pieces, single elements)
    (3, 100, 8, 24, 128, 64), (5, 70, 4, 32, 64, 32), (4, 66, 4, 12, 128, 100), (5, 70, 4, 32, 100, 40), (3, 130, 2, 16, 61, 90),
    (5, 70, 8, 32, 5, 7), (5, 65, 16, 32, 3, 3), (1, 70, 1, 5, 24, 4096),
]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("states", [False, True])
@pytest.mark.parametrize("shape", MANY)
def test_gated_delta_many_blocks(device, dtype, shape, states):
    """Forward with and without what a backward pass needs, and backward."""
    assert shape[0] * shape[3] * -(-shape[5] // 32) > 128
    x = arrays(dtype, *shape, seed=41, states=shape[0] if states else 0, back=True)
    check_delta(x, dtype, back=True)
    check_delta({n: v for n, v in x.items() if n not in ("do", "dstate_out")}, dtype)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_gated_delta_many_packed_sequences(device, dtype):
    cuts = [0, 1, 1, 65, 66, 130, 258, 259, 300, 300, 320]
    check_delta(arrays(dtype, 1, 320, 4, 16, 48, 40, seed=42, states=len(cuts) - 1, back=True), dtype, cuts, back=True)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", [(1, 130, 1, 1, 16, 1001), (1, 70, 1, 2, 128, 512), (2, 1, 1, 1, 20, 1500)])
def test_gated_delta_wide_values(device, dtype, shape):
    """Few heads of many columns: 16 columns a workgroup, and single tokens."""
    check_delta(arrays(dtype, *shape, seed=43, states=shape[0], back=True), dtype, back=True)
    check_delta(arrays(dtype, *shape, seed=43, states=shape[0]), dtype)


# ---- where gradients are written ---------------------------------------------

def _between_guards(like):
    """A place for a result at an odd element, its heads a few elements apart,
    and the whole that it lies in, of sevens."""
    b, t, h = like.shape[:3]
    if like.dim() == 3:
        whole = torch.full((b, t, 2 * h + 3), 7.0, dtype=like.dtype, device="cuda")
        return whole[..., 1:2 * h + 1:2], whole
    whole = torch.full((b, t, h, like.shape[3] + 5), 7.0, dtype=like.dtype, device="cuda")
    return whole[..., 3:3 + like.shape[3]], whole


def _heads_first_place(like):
    whole = torch.full(tuple(like.shape[i] for i in (0, 2, 1)) + tuple(like.shape[3:]), 7.0, dtype=like.dtype, device="cuda")
    return whole.transpose(1, 2), whole


def run_delta_into(x, dtype, place):
    """``run_delta`` of the backward pass with its results placed; also how
    many elements of each whole are none of its result and not seven."""
    b, t, hk, dk = x["q"].shape
    hv, dv = x["v"].shape[2:]
    op = O.GatedDelta(dtype, b, t, hk, hv, dk, dv, states=False)
    dev = {k: v.cuda() for k, v in x.items()}
    names = ("q", "k", "v", "g", "beta")
    ins = [dev[n] for n in names]
    out, whole = {}, {}
    for n in ("o",) + tuple("d" + n for n in names):
        out[n], whole[n] = place(dev["v" if n == "o" else n[1:]])
    saved = torch.full((op.saved_bytes(),), 255, dtype=torch.uint8, device="cuda")
    op.forward(*ins, out["o"], saved=saved)
    op.backward(*ins, dev["do"], saved, *(out["d" + n] for n in names))
    torch.cuda.synchronize()
    touched = {}
    for n in out:
        got = out[n].clone()
        out[n].fill_(7.0)
        touched[n] = int((whole[n] != 7.0).sum())
        out[n] = got
    return out, touched


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("place", [_between_guards, _heads_first_place])
@pytest.mark.parametrize("shape", [(2, 70, 2, 4, 64, 96), (2, 130, 1, 2, 100, 40), (2, 70, 1, 2, 5, 3), (1, 65, 1, 1, 33, 17),
                                   (3, 70, 8, 48, 64, 32), (3, 70, 8, 48, 40, 27), (3, 67, 8, 48, 5, 7)])
def test_gated_delta_writes_gradients_where_they_belong(device, dtype, place, shape):
    """Results of any stride and alignment are those of contiguous ones, and
    what lies between their elements keeps its value."""
    x = arrays(dtype, *shape, seed=44, back=True)
    want = run_delta(x, dtype, back=True)
    got, touched = run_delta_into(x, dtype, place)
    for n in want:
        assert torch.equal(got[n], want[n]), n
        assert touched[n] == 0, n


def test_gated_delta_results_past_32_bits(device):
    """o, dq, dk and dv with tokens 2^23 elements apart: the last ones lie past
    2^32 bytes and 2^31 elements."""
    x = arrays("bf16", 2, 300, 1, 2, 32, 32, seed=45, back=True)
    want = run_delta(x, "bf16", back=True)

    def place(like):
        b, n, h = like.shape[:3]
        if like.dim() == 3:
            t = torch.empty_like(like)
            return t, torch.full((1,), 7.0)
        whole = torch.empty((b * n - 1) * (1 << 23) + h * like.shape[3], dtype=like.dtype, device="cuda")
        return whole.as_strided(tuple(like.shape), (n << 23, 1 << 23, like.shape[3], 1)), torch.full((1,), 7.0)

    got, _ = run_delta_into(x, "bf16", place)
    for n in want:
        assert torch.equal(got[n], want[n]), n
    del got
    torch.cuda.empty_cache()


# ---- what a norm block's dropout drops ---------------------------------------

@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("width", [40, 1000, 5000, 9001])
@pytest.mark.parametrize("how", [("rms", "rms", "silu"), ("layer", "none", "sigmoid"), ("none", "rms", "silu")])
def test_norm_block_drops_what_is_not_a_number(device, dtype, width, how):
    """Gates that are infinite or NaN where they are dropped (and values of y,
    where no norm reads them): results and gradients are those of any other
    gate there, and theirs are zero."""
    rows, p, seed, offset = 6, 0.4, 0x1234567890ABCDEF, 1 << 33
    x, w = norm_arrays(dtype, "f32", rows, width, *how, seed=46)
    drop = torch.from_numpy(~R.kept(rows, width, p, seed, offset)[0])
    clean = {k: v.clone() for k, v in x.items()}
    bad = torch.tensor([float("inf"), -float("inf"), float("nan")]).to(TYPES[dtype]).repeat(rows * width)[:rows * width].view(rows, width)
    for n in ("gate",) + (("y",) if how[0] == "none" else ()):
        x[n] = torch.where(drop, bad, x[n])
        clean[n] = torch.where(drop, torch.zeros_like(x[n]), x[n])
    op = O.NormBlock(dtype, rows, width, norm=how[0], pre=how[1], gate=how[2], dropout=p, scale=0.7, eps=1e-5)
    dev, wd = {k: v.cuda() for k, v in x.items()}, {k: v.cuda() for k, v in w.items()}
    wide = {k: v.double().numpy() for k, v in {**clean, **w}.items()}
    got = {n: torch.empty_like(dev["y"]) for n in (("h", "n") if how[1] != "none" else ("h",))}
    op.forward(dev["y"], got["h"], got.get("n"), gate=dev["gate"], residual=dev["residual"], seed=seed, offset=offset, **wd)
    out = {n: torch.empty_like(dev["y"]) for n in ("y", "gate", "residual")}
    grads = {n: torch.empty_like(v) for n, v in wd.items()}
    op.backward(dev["y"], dev["dh"], out["y"], dn=dev.get("dn"), h=dev.get("h"), gate=dev["gate"], dgate=out["gate"],
                dresidual=out["residual"], grads=grads, seed=seed, offset=offset, **wd)
    torch.cuda.synchronize()
    want = R.norm_block(wide, *how, 0.7, 1e-5, p, seed, offset)
    for n, v in got.items():
        close(v, want[n], n)
    want = R.norm_block(wide, *how, 0.7, 1e-5, p, seed, offset, back=True)
    for n, v in {**out, **grads}.items():
        close(v, want[n], n)
    assert not out["gate"].cpu()[drop].any()
    if how[0] == "none":
        assert not out["y"].cpu()[drop].any()


# ---- results over inputs -----------------------------------------------------

@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("width", [100, 3000, 9001])
def test_norm_block_over_any_of_its_inputs(device, dtype, width):
    """h and n each over y, the gate or the residual, row for row."""
    x, w = norm_arrays(dtype, "f32", 9, width, "layer", "rms", "silu", seed=47)
    op = O.NormBlock(dtype, 9, width, norm="layer", pre="rms", gate="silu", dropout=0.2)
    dev, wd = {k: v.cuda() for k, v in x.items()}, {k: v.cuda() for k, v in w.items()}
    h, n = torch.empty_like(dev["y"]), torch.empty_like(dev["y"])
    op.forward(dev["y"], h, n, gate=dev["gate"], residual=dev["residual"], seed=2, **wd)
    names = ("y", "gate", "residual")
    for a in names:
        for b in names:
            if a != b:
                t = {k: dev[k].clone() for k in names}
                op.forward(t["y"], t[a], t[b], gate=t["gate"], residual=t["residual"], seed=2, **wd)
                torch.cuda.synchronize()
                assert torch.equal(t[a], h) and torch.equal(t[b], n), (a, b)


# ---- 16-bit results to their own rounding ------------------------------------

# Half a unit of the last place, and what f32 sums (4e-6) or products of 16-bit
# planes (three of 2^-17) add before it.
ROUNDING = {"bf16": 2.0 ** -9, "f16": 2.0 ** -12}


@pytest.mark.parametrize("dtype", list(ROUNDING))
@pytest.mark.parametrize("case", [(50, 128, "rms", "none", "silu"), (40, 700, "layer", "rms", "sigmoid"), (30, 4096, "rms", "rms", "none"),
                                  (12, 9000, "layer", "layer", "silu")])
def test_norm_block_rounds_its_results_once(device, dtype, case):
    x, w = norm_arrays(dtype, "f32", *case, seed=48)
    how = (*case[2:], 0.7, 1e-5, 0.2, 11, 12)
    op = O.NormBlock(dtype, *case[:2], norm=case[2], pre=case[3], gate=case[4], dropout=0.2, scale=0.7, eps=1e-5)
    dev, wd = {k: v.cuda() for k, v in x.items()}, {k: v.cuda() for k, v in w.items()}
    wide = {k: v.double().numpy() for k, v in {**x, **w}.items()}
    got = {n: torch.empty_like(dev["y"]) for n in (("h", "n") if case[3] != "none" else ("h",))}
    op.forward(dev["y"], got["h"], got.get("n"), gate=dev.get("gate"), residual=dev["residual"], seed=11, offset=12, **wd)
    out = {n: torch.empty_like(dev["y"]) for n in ("y", "residual") + (("gate",) if "gate" in x else ())}
    op.backward(dev["y"], dev["dh"], out["y"], dn=dev.get("dn"), h=dev.get("h"), gate=dev.get("gate"), dgate=out.get("gate"),
                dresidual=out["residual"], seed=11, offset=12, **wd)
    torch.cuda.synchronize()
    for want, results in ((R.norm_block(wide, *how), got), (R.norm_block(wide, *how, back=True), out)):
        for n, v in results.items():
            close(v, want[n], n, ROUNDING[dtype] + 4e-6)


@pytest.mark.parametrize("dtype", list(ROUNDING))
@pytest.mark.parametrize("shape", [(2, 200, 2, 4, 128, 96), (3, 100, 8, 24, 128, 64), (2, 130, 1, 2, 100, 40), (3, 5, 2, 4, 64, 64)])
@pytest.mark.parametrize("states", [False, True])
def test_gated_delta_rounds_o_and_dv_once(device, dtype, shape, states):
    x = arrays(dtype, *shape, seed=49, states=shape[0] if states else 0, back=True)
    got = run_delta(x, dtype, back=True)
    want = R.delta_batch({n: v.double().numpy() for n, v in x.items()}, None, shape[4] ** -0.5,
                         x["state"].double().numpy() if states else None, True)
    for n in ("o", "dv", "dbeta"):
        close(got[n], want[n], n, ROUNDING[dtype] + 3 * 2.0 ** -17)
    got = run_delta({n: v for n, v in x.items() if n not in ("do", "dstate_out")}, dtype)
    close(got["o"], want["o"], "o", ROUNDING[dtype] + 3 * 2.0 ** -17)


# ---- gradients of 16-bit heads to their own rounding -------------------------

# What a bf16 or f16 gradient of q and k adds to its rounding: S, dS, U and Y in
# 11 bits and M and B in 16, a few roundings of 2^-12 in 2^-9 or of as much in
# 2^-12 (where S and dS are f32): 2^-9 (1 + 1/8), and twice 2^-12.
GRADIENT = {"bf16": 2.0 ** -9 * 1.125, "f16": 2.0 ** -11}


@pytest.mark.parametrize("dtype", list(GRADIENT))
@pytest.mark.parametrize("alike", [0.0, 1.0, 4.0])
@pytest.mark.parametrize("shape", [(2, 200, 2, 4, 128, 96), (3, 100, 8, 24, 128, 64), (2, 130, 1, 2, 64, 40)])
def test_gated_delta_gradients_of_keys_that_are_alike(device, dtype, alike, shape):
    """Keys and queries around one direction: differences of the parts that
    make dq and dk are smaller than the parts, and what those lose shows."""
    x = arrays(dtype, *shape, seed=51, back=True)
    g = torch.Generator().manual_seed(52)
    mean = alike * torch.randn(1, 1, shape[2], shape[4], generator=g)
    for n in ("q", "k"):
        x[n] = torch.nn.functional.normalize(torch.randn(x[n].shape, generator=g) + mean, dim=-1).to(TYPES[dtype])
    got = run_delta(x, dtype, back=True)
    want = R.delta_batch({n: v.double().numpy() for n, v in x.items()}, None, shape[4] ** -0.5, None, True)
    for n in ("dq", "dk"):
        close(got[n], want[n], n, GRADIENT[dtype])


@pytest.mark.parametrize("up", [1e33, 1e-33])
def test_gated_delta_values_as_far_from_one_as_bf16_has_them(device, up):
    """v far up and the gradient of o as far down, and the other way round:
    the gradients of q, k, g and beta, products of the two, are about 1."""
    x = arrays("bf16", 2, 130, 1, 2, 64, 64, seed=53, back=True)
    x["v"] = (x["v"].float() * up).bfloat16()
    x["do"] = (x["do"].float() / up).bfloat16()
    check_delta(x, "bf16", back=True)


@pytest.mark.parametrize("shape", [(2, 130, 1, 2, 64, 96), (3, 100, 8, 24, 128, 96)])
def test_gated_delta_columns_of_different_size(device, shape):
    """Value columns 2^20 apart whose gradients of o are as far apart the other
    way: every column has its share of dq, dk, dg and dbeta."""
    x = arrays("bf16", *shape, seed=54, back=True)
    size = torch.ones(shape[5])
    size[:32], size[32:48] = 2.0 ** 10, 2.0 ** -10
    x["v"] = (x["v"].float() * size).bfloat16()
    x["do"] = (x["do"].float() / size).bfloat16()
    got = run_delta(x, "bf16", back=True)
    want = R.delta_batch({n: v.double().numpy() for n, v in x.items()}, None, shape[4] ** -0.5, None, True)
    for n in ("dq", "dk", "dg", "dbeta"):
        close(got[n], want[n], n)
    for lo, hi in ((0, 32), (32, 48), (48, 96)):
        for n in ("o", "dv"):
            close(got[n][..., lo:hi], want[n][..., lo:hi], "%s %d" % (n, lo))
