"""Attention, the norm and rotation of its heads, and the embedding in 64 bits,
written from their formulas, and how results are held against them."""

import numpy as np

HALF = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}  # half a step, relative to the value


def attention(q, k, v, scale, do=None):
    """One sequence: q [t, h, d], k and v [n, hk, d], the queries the last t of
    the n tokens. o; with do also dq, dk, dv, for each of the three the norm of
    the sums of magnitudes that its terms cancel from, and the largest score."""
    t, h, d = q.shape
    n, hk = k.shape[:2]
    of = np.arange(h) // (h // hk)
    o = np.zeros((t, h, d))
    back = do is not None
    dq, dk, dv = np.zeros((t, h, d)), np.zeros((n, hk, d)), np.zeros((n, hk, d))
    aq, ak = np.zeros((t, h, d)), np.zeros((n, hk, d))
    largest = 0.0
    seen = np.arange(n)[None, :] <= np.arange(t)[:, None] + (n - t)
    for i in range(h):
        kk, vv = k[:, of[i]], v[:, of[i]]
        with np.errstate(invalid="ignore"):
            s = np.where(seen, scale * (q[:, i] @ kk.T), -np.inf)
            top = s.max(axis=1, keepdims=True, initial=-np.inf)
            e = np.exp(s - np.where(np.isinf(top), 0.0, top))
            total = e.sum(axis=1, keepdims=True)
            p = np.divide(e, total, out=np.zeros_like(e), where=total > 0)
            o[:, i] = p @ vv
        if not back:
            continue
        largest = max(largest, np.abs(s[seen]).max(initial=0.0))
        dp = do[:, i] @ vv.T
        mean = (p * dp).sum(axis=1, keepdims=True)
        ds = scale * p * (dp - mean)
        dq[:, i] = ds @ kk
        dk[:, of[i]] += ds.T @ q[:, i]
        dv[:, of[i]] += p.T @ do[:, i]
        # dp is a sum over the head, and the mean one over dp: both in f32
        terms = np.abs(scale) * p * (np.abs(do[:, i]) @ np.abs(vv.T))
        terms = terms + p * terms.sum(axis=1, keepdims=True)
        aq[:, i] = terms @ np.abs(kk)
        ak[:, of[i]] += terms.T @ np.abs(q[:, i])
    if not back:
        return o
    return o, dq, dk, dv, (np.linalg.norm(aq), np.linalg.norm(ak), 0.0), largest


def turn(x, angle, rotary, interleaved):
    """Pairs of the first `rotary` elements of x [..., head, dim] by angle
    [..., 1, rotary / 2]."""
    y = x.copy()
    a, b = (np.s_[..., 0:rotary:2], np.s_[..., 1:rotary:2]) if interleaved else (
        np.s_[..., :rotary // 2], np.s_[..., rotary // 2:rotary])
    y[a] = x[a] * np.cos(angle) - x[b] * np.sin(angle)
    y[b] = x[b] * np.cos(angle) + x[a] * np.sin(angle)
    return y


def head_norm(x, weight, angle, rotary, interleaved, norm, eps, dy=None):
    """x [b, t, h, d]; y, or with dy dx and the gradient of the weight and the
    sum of its terms' magnitudes."""
    w = np.ones(x.shape[-1]) if weight is None else weight
    inv = 1.0 / np.sqrt((x * x).mean(axis=-1, keepdims=True) + eps) if norm else np.ones(x.shape[:-1] + (1,))
    xhat = x * inv
    if dy is None:
        return turn(xhat * w, angle, rotary, interleaved)
    dn = turn(dy, -angle, rotary, interleaved)
    g = dn * w
    dx = inv * (g - xhat * (g * xhat).mean(axis=-1, keepdims=True)) if norm else g
    parts = dn * xhat
    return dx, parts.sum(axis=(0, 1, 2)), np.abs(parts).sum(axis=(0, 1, 2))


def embed(ids, weight, scale):
    there = (ids >= 0) & (ids < len(weight))
    return scale * np.where(there[:, None], weight[np.where(there, ids, 0)], 0.0) if len(weight) else np.zeros((len(ids), weight.shape[1]))


def embed_back(ids, dout, vocab, scale):
    """The table's gradient, and the sums of its terms' magnitudes."""
    there = (ids >= 0) & (ids < vocab)
    g, a = np.zeros((vocab, dout.shape[1])), np.zeros((vocab, dout.shape[1]))
    np.add.at(g, ids[there], scale * dout[there])
    np.add.at(a, ids[there], np.abs(scale * dout[there]))
    return g, a


def close(got, want, name, bound, cancelled=0.0):
    """In the 2-norm over all of it within `bound` of want, and what f32 sums of
    terms of norm `cancelled` may be off; and each element within 16 bounds of
    its value or the root mean square, which is what a rounding of one operand
    can do to a sum of few terms."""
    a, b = np.asarray(got, dtype=np.float64), np.asarray(want, dtype=np.float64)
    assert a.shape == b.shape, name
    if not b.size:
        return
    assert np.isfinite(a).all(), "%s is not finite" % name
    allowed = bound * np.linalg.norm(b) + 4e-6 * cancelled
    off = np.linalg.norm(a - b)
    assert off <= allowed, "%s is %.3g off, %.3g allowed, of %.3g" % (name, off, allowed, np.linalg.norm(b))
    each = 16 * (bound * np.maximum(np.abs(b), np.linalg.norm(b) / np.sqrt(b.size)) + 4e-6 * cancelled / np.sqrt(b.size))
    assert (np.abs(a - b) <= each).all(), "%s has an element %.3g of what is allowed" % (name, (np.abs(a - b) / each).max())


def near(got, want, name, half, slack):
    """Each element of a result that is rounded once, from f32 values that are
    `slack` off at the most."""
    a, b = np.asarray(got, dtype=np.float64), np.asarray(want, dtype=np.float64)
    assert a.shape == b.shape, name
    if not b.size:
        return
    assert np.isfinite(a).all(), "%s is not finite" % name
    tiny = 2.0 ** -25 if half == HALF["f16"] else 0.0  # half of f16's least step
    most = half * (np.abs(b) + slack) + slack + tiny
    with np.errstate(invalid="ignore", divide="ignore"):
        ratio = np.where(np.abs(a - b) > 0, np.abs(a - b) / most, 0.0).max()
    assert ratio <= 1.0, "%s is off by %.3g of what is allowed" % (name, ratio)
