"""Attention, the norm and rotation of its heads and the embedding where a
formula is still defined but little is left of it: no eps, infinities, the
largest values, counts of tokens that few calls have. Tolerances are those of
test_gpu_attending_operators.py."""

import numpy as np
import pytest
import torch

import attending_reference as A
from cudacaml_amd import operators as O
from test_gpu_attending_operators import (BOUND, TYPES, attention_arrays, check_attention, f64, ids_of, nans, normal, run_attention,
                                          run_embedding, same)

pytestmark = pytest.mark.gpu


# ---- norm and rotation of heads --------------------------------------------------

@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("h,hk,d,rotary,tokens", [(3, 1, 64, 64, 7), (2, 4, 128, 128, 7), (5, 3, 40, 16, 7), (9, 2, 64, 64, 2100)])
def test_head_norm_without_eps(device, dtype, h, hk, d, rotary, tokens):
    """Heads that do not fill a wave: what is beyond the last one adds nothing
    to the gradients of the weights, with an eps of zero either."""
    op = O.HeadNorm(dtype, 1, tokens, h, hk, d, rotary=rotary, eps=0.0)
    x = {n: normal(dtype, 1, tokens, c, d, seed=40 + i) for i, (n, c) in enumerate((("q", h), ("k", hk), ("dq", h), ("dk", hk)))}
    freq = torch.exp(-torch.arange(rotary // 2) * 0.4).float()
    w = {n: 1.0 + 0.3 * normal("f32", d, seed=44 + i) for i, n in enumerate(("q_weight", "k_weight"))}
    dev = {n: v.cuda() for n, v in x.items()}
    given = dict(frequencies=freq.cuda(), **{n: v.cuda() for n, v in w.items()})
    out, grads = {n: nans(v.shape, dtype) for n, v in x.items()}, {n: nans((d,), "f32") for n in w}
    op.forward(dev["q"], dev["k"], out["q"], out["k"], **given)
    op.backward(dev["q"], dev["k"], dev["dq"], dev["dk"], out["dq"], out["dk"], grads=grads, **given)
    torch.cuda.synchronize()
    angle = np.arange(tokens)[None, :, None, None] * f64(freq)
    for n in ("q", "k"):
        a, g, ww = f64(x[n]), f64(x["d" + n]), f64(w[n + "_weight"])
        how = (rotary, False, True, 0.0)
        plain = A.head_norm(a, ww, angle * 0, *how)
        A.near(f64(out[n]), A.head_norm(a, ww, angle, *how), n, A.HALF[dtype], 2.0 ** -19 * np.abs(plain).max(-1, keepdims=True))
        dx, dw, terms = A.head_norm(a, ww, angle, *how, dy=g)
        inv = 1.0 / np.sqrt((a * a).mean(-1, keepdims=True))
        big = np.abs(g).max(-1, keepdims=True) * np.abs(ww).max() * inv
        A.near(f64(out["d" + n]), dx, "d" + n, A.HALF[dtype], 2.0 ** -19 * big * (1 + np.abs(a * inv).max(-1, keepdims=True)))
        A.near(f64(grads[n + "_weight"]), dw, n + "_weight", A.HALF["f32"], 2.0 ** -18 * terms)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("d,rotary", [(40, 0), (64, 16), (37, 20), (64, 64)])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_head_norm_elements_that_are_not_rotated_stand_alone(device, dtype, d, rotary, bad):
    """Without a norm they are copied: what is not finite in one changes no
    other, forward or back, and in a rotated one its pair alone."""
    op = O.HeadNorm(dtype, 1, 5, 3, 2, d, rotary=rotary, norm="none")
    x = [normal(dtype, 1, 5, c, d, seed=50 + i).cuda() for i, c in enumerate((3, 2, 3, 2))]
    freq = torch.linspace(1.0, 0.1, rotary // 2, device="cuda")

    def run():
        out = [nans(v.shape, dtype) for v in x]
        op.forward(*x[:2], *out[:2], frequencies=freq)
        op.backward(*x, *out[2:], frequencies=freq)
        torch.cuda.synchronize()
        return out

    want = run()
    for at in {0, rotary // 2, max(rotary - 1, 0), rotary % d, d - 1}:
        mates = {at} if at >= rotary else {at, (at + rotary // 2) % rotary}
        keep = [v[0, 3, 1, at].item() for v in x]
        for v in x:
            v[0, 3, 1, at] = bad
        for got, before in zip(run(), want):
            for i in mates:
                assert not torch.isfinite(got[0, 3, 1, i]), (at, i)
                got[0, 3, 1, i] = before[0, 3, 1, i]
            assert same(got, before), at
        for v, k in zip(x, keep):
            v[0, 3, 1, at] = k


# ---- attention -------------------------------------------------------------------

def _apart(x, odd):
    """The array, or a copy whose heads begin off all 16-byte places."""
    if not odd:
        return x
    b, t, h, d = x.shape
    return torch.empty(b, t, h * d + 3, dtype=x.dtype, device="cuda")[..., 1:1 + h * d].view(x.shape).copy_(x)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("d,odd", [(41, False), (64, True), (128, True), (72, True), (64, False)])
@pytest.mark.parametrize("tokens,keys", [(300, None), (200, 330)])
def test_attention_values_not_finite_wherever_they_stand(device, dtype, d, odd, tokens, keys):
    """In the first tile of keys and later ones, alone and with others, in heads
    that are copied to their tile and in those that pass through registers,
    with eight waves a workgroup: who sees one has it in its column, all else is
    as it was."""
    n = keys or tokens
    q, k, v = (normal(dtype, 1, t, c, d, seed=60 + i).cuda() for i, (t, c) in enumerate(((tokens, 4), (n, 2), (n, 2))))
    k, v = _apart(k, odd), _apart(v, odd)
    op = O.Attention(dtype, 1, tokens, 4, 2, d, keys=keys)
    lengths = None if keys is None else torch.tensor([n], dtype=torch.int32, device="cuda")

    def run():
        o = nans(q.shape, dtype)
        op.forward(q, k, v, o, lengths=lengths)
        torch.cuda.synchronize()
        return o

    want = run()
    assert torch.isfinite(want).all()
    for bad in (float("inf"), float("-inf"), float("nan")):
        for places in ([0], [3], [31, 32], [63], [64], [5, 127], [2, 130, 200], [n - 1], [n - 70, n - 3]):
            keep = v.clone()
            for i, at in enumerate(places):
                v[0, at, 1, (7 + 5 * i) % d] = bad
            got = run()
            assert same(got[0, :, :2], want[0, :, :2]), places
            changed = torch.zeros(tokens, d, dtype=torch.bool, device="cuda")
            for i, at in enumerate(places):
                changed[max(0, at - (n - tokens)):, (7 + 5 * i) % d] = True
            changed = changed[:, None].expand(tokens, 2, d)
            assert not torch.isfinite(got[0, :, 2:][changed]).any(), places
            assert same(got[0, :, 2:][~changed], want[0, :, 2:][~changed]), places
            v.copy_(keep)


@pytest.mark.parametrize("d,odd", [(41, False), (128, False), (64, True)])
@pytest.mark.parametrize("tokens,keys", [(300, None), (40, 700), (1, 700)])
def test_attention_infinities_of_f32_are_infinities(device, d, odd, tokens, keys):
    """A query that sees one has it, of whatever tile the key is; of both signs,
    or NaN, it has NaN."""
    n = keys or tokens
    inf, nan = float("inf"), float("nan")
    q, k, v = (normal("f32", 1, t, c, d, seed=70 + i).cuda() for i, (t, c) in enumerate(((tokens, 2), (n, 1), (n, 1))))
    k, v = _apart(k, odd), _apart(v, odd)
    op = O.Attention("f32", 1, tokens, 2, 1, d, keys=keys)
    lengths = None if keys is None else torch.tensor([n], dtype=torch.int32, device="cuda")
    out = [nans(q.shape, "f32") for _ in range(2)]
    op.forward(q, k, v, out[0], lengths=lengths)
    want = out[0].clone()
    for places in ([(3, inf)], [(0, -inf)], [(100, nan)], [(40, inf), (45, -inf)], [(10, inf), (n - 2, inf)], [(n - 1, -inf)], [(9, inf), (n - 3, nan)]):
        keep = v.clone()
        column = want[0, :, :, 7].clone()
        for at, x in places:
            v[0, at, 0, 7] = x
            column[max(0, at - (n - tokens)):] += x
        op.forward(q, k, v, out[1], lengths=lengths)
        torch.cuda.synchronize()
        assert torch.equal(torch.nan_to_num(out[1][0, :, :, 7], nan=7.0), torch.nan_to_num(column, nan=7.0)), places
        rest = torch.arange(d, device="cuda") != 7
        assert same(out[1][..., rest], want[..., rest]), places
        v.copy_(keep)


@pytest.mark.parametrize("tokens,d", [(20, 64), (150, 41), (150, 128)])
def test_attention_largest_f32_values(device, tokens, d):
    """Next to what f32 holds, which no 16 bits hold, where their sums stay
    below it: one to a column, which the others' do not take beyond the largest
    f32, 3.4028e38. Forward and back; scores are zeros, so no term is larger
    than 1."""
    x = attention_arrays("f32", 1, tokens, 2, 1, d, seed=8)
    x["q"].zero_()
    x["do"] *= 2.0 ** -20
    x["v"][0, 2, 0, 3], x["v"][0, tokens - 7, 0, 5], x["v"][0, 5, 0, 6] = 3.402e38, -3.402e38, 3.395e38
    check_attention(x, "f32", run_attention(x, "f32"))


@pytest.mark.parametrize("tokens,keys", [(150, None), (1, 300), (70, 700)])
@pytest.mark.parametrize("power", [-104, 80])
def test_attention_small_and_large_f32_values(device, tokens, keys, power):
    """As exact as others: three planes hold all bits of values from 2^-110 on."""
    x = attention_arrays("f32", 1, tokens, 2, 1, 64, seed=33, keys=keys)
    x["v"] *= 2.0 ** power
    o = nans(x["q"].shape, "f32")
    op = O.Attention("f32", 1, tokens, 2, 1, 64, keys=keys)
    op.forward(*(x[n].cuda() for n in ("q", "k", "v")), o, lengths=None if keys is None else torch.tensor([keys], dtype=torch.int32, device="cuda"))
    a = {n: f64(v)[0] for n, v in x.items()}
    A.close(f64(o)[0], A.attention(a["q"], a["k"], a["v"], 64 ** -0.5), "o", BOUND["f32"] * (2 if a["q"].size < 256 else 1))


@pytest.mark.parametrize("dtype,large,small", [("bf16", 1.0, 2.0 ** -24), ("f16", 2.0 ** 8, 2.0 ** -8)])
def test_attention_gradients_of_rows_far_smaller_than_their_neighbours(device, dtype, large, small):
    """Every other token's gradient of o: a tile's elements are whole down to
    2^-28 of its largest, which those here are but for few, and those to
    2^-38; so its queries' gradients are as exact as the others'."""
    x = attention_arrays(dtype, 1, 200, 4, 2, 64, seed=32)
    x["do"][:, ::2] *= large
    x["do"][:, 1::2] *= small
    got = f64(run_attention(x, dtype)["dq"])[0]
    a = {n: f64(v)[0] for n, v in x.items()}
    want = A.attention(a["q"], a["k"], a["v"], 64 ** -0.5, a["do"])[1]
    tiny = 2.0 ** -25 if dtype == "f16" else 0.0  # half of f16's least step
    for rows in (slice(0, None, 2), slice(1, None, 2)):
        off = np.linalg.norm(got[rows] - want[rows])
        assert off <= BOUND[dtype] * np.linalg.norm(want[rows]) + tiny * want[rows].size ** 0.5


# ---- embedding -------------------------------------------------------------------

@pytest.mark.parametrize("tokens,vocab,width", [(192 * 2048, 5000, 3), (192 * 2048 + 1, 5000, 3), (257 * 2048 + 9, 600000, 8), ((1 << 20) + 2047, 70, 1)])
def test_embedding_of_many_tokens(device, tokens, vocab, width):
    """On both sides of where blocks' places are made by groups of blocks, the
    last group and block whole and not, in one to three passes."""
    ids = ids_of(tokens, vocab, seed=tokens)
    ids[::1000] = -1
    run_embedding("f32", ids, vocab, width, seed=7)
    run_embedding("bf16", ids, vocab, width, seed=8, accumulate=True, weight="f32")


def test_embedding_of_a_hundred_million_tokens(device):
    """Groups of more than 64 blocks. Rows of whole numbers, whose sums f32
    holds, so that the order of a sum does not count."""
    tokens, vocab = (1 << 27) + 3 * 2048 + 77, 3000
    g = torch.Generator(device="cuda").manual_seed(9)
    ids = torch.randint(-2, vocab, (tokens,), generator=g, dtype=torch.int32, device="cuda")
    dout = torch.randint(-8, 9, (tokens, 1), generator=g, device="cuda", dtype=torch.int32)
    want = torch.zeros(vocab + 2, dtype=torch.int64, device="cuda").index_add_(0, (ids + 2).long(), dout[:, 0].long())[2:]
    dout, dw = dout.to(torch.bfloat16), nans((vocab, 1), "f32")
    op = O.Embedding("bf16", tokens, vocab, 1, weight_dtype="f32")
    op.backward(ids, dout, dw)
    torch.cuda.synchronize()
    assert torch.equal(dw[:, 0].long(), want)
    op.free()
