"""Plain 64-bit forms of the layer operators, from their definitions: one
token, one row and one counter at a time, gradients derived by hand from the
same definitions (and checked against differences in test_operators.py)."""

import numpy as np

M0, M1, W0, W1, LOW = 0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85, 0xFFFFFFFF


def philox(counter, key):
    c, k = list(counter), list(key)
    for r in range(10):
        a, b = M0 * c[0], M1 * c[2]
        c = [(b >> 32) ^ c[1] ^ k[0], b & LOW, (a >> 32) ^ c[3] ^ k[1], a & LOW]
        k = [(k[0] + W0) & LOW, (k[1] + W1) & LOW]
    return c


def kept(rows, cols, p, seed, offset):
    """The kept columns of each row, and the scale of a kept value."""
    bar = int(np.rint(p * 65536.0))
    keep = np.zeros((rows, cols), bool)
    for r in range(rows):
        for g in range((cols + 7) // 8):
            words = philox((g, r, offset & LOW, offset >> 32), (seed & LOW, seed >> 32))
            halves = [h for w in words for h in (w & 0xFFFF, w >> 16)]
            for j in range(min(8, cols - 8 * g)):
                keep[r, 8 * g + j] = halves[j] >= bar
    return keep, (0.0 if bar >= 65536 else 65536.0 / (65536 - bar))


def drop(x, p, seed, offset):
    keep, up = kept(x.shape[0], x.shape[1], p, seed, offset)
    out = np.zeros(x.shape)
    out[keep] = x[keep] * up
    return out


# ---- gated delta rule --------------------------------------------------------

def delta(q, k, v, g, beta, scale, state, do=None, dstate_out=None):
    """One sequence: q, k [tokens, key heads, dk], v [tokens, value heads, dv],
    g and beta [tokens, value heads], state [value heads, dk, dv]. Gives o and
    the last state, and with ``do`` the gradients of q, k, v, g, beta, state."""
    tokens, heads = g.shape
    group = heads // q.shape[1]
    kr, qr = np.repeat(k, group, 1), np.repeat(q, group, 1)
    o, states, s = np.zeros(v.shape), [], state.astype(np.float64)
    alpha = np.exp(g.astype(np.float64))
    for t in range(tokens):
        states.append(s)
        s = alpha[t][:, None, None] * s
        u = beta[t][:, None] * (v[t] - np.einsum("hkv,hk->hv", s, kr[t]))
        s = s + kr[t][:, :, None] * u[:, None, :]
        o[t] = scale * np.einsum("hkv,hk->hv", s, qr[t])
    if do is None:
        return o, s
    e = np.zeros(s.shape) if dstate_out is None else dstate_out.astype(np.float64)
    dq, dk = np.zeros(qr.shape), np.zeros(kr.shape)
    dv, dg, db = np.zeros(v.shape), np.zeros(g.shape), np.zeros(g.shape)
    for t in reversed(range(tokens)):
        before, a, kt = states[t], alpha[t][:, None, None], kr[t]
        seen = a * before
        left = v[t] - np.einsum("hkv,hk->hv", seen, kt)
        u = beta[t][:, None] * left
        now = seen + kt[:, :, None] * u[:, None, :]
        dq[t] = scale * np.einsum("hkv,hv->hk", now, do[t])
        e = e + scale * qr[t][:, :, None] * do[t][:, None, :]
        du = np.einsum("hkv,hk->hv", e, kt)
        dleft = beta[t][:, None] * du
        dk[t] = np.einsum("hkv,hv->hk", e, u) - np.einsum("hkv,hv->hk", seen, dleft)
        db[t] = (du * left).sum(-1)
        dv[t] = dleft
        dseen = e - kt[:, :, None] * dleft[:, None, :]
        dg[t] = (dseen * seen).sum((-1, -2))
        e = a * dseen
    group_sum = lambda x: x.reshape(tokens, q.shape[1], group, x.shape[-1]).sum(2)  # noqa: E731
    return o, s, dict(dq=group_sum(dq), dk=group_sum(dk), dv=dv, dg=dg, dbeta=db, dstate=e)


def delta_batch(x, cuts, scale, state, back):
    """``delta`` over the rows of a batch or, with ``cuts``, its packed
    sequences; x is a dict of arrays [batch, tokens, ...]."""
    names = ("q", "k", "v", "g", "beta")
    parts = [(i, 0, x["q"].shape[1]) for i in range(x["q"].shape[0])] if cuts is None else \
            [(0, a, b) for a, b in zip(cuts, cuts[1:])]
    out = {"o": np.zeros(x["v"].shape)}
    heads, dk, dv = x["v"].shape[2], x["q"].shape[3], x["v"].shape[3]
    out["state"] = np.zeros((len(parts), heads, dk, dv))
    if back:
        out["dstate"] = np.zeros(out["state"].shape)
        out.update({"d" + n: np.zeros(x[n].shape) for n in names})
    for i, (row, lo, hi) in enumerate(parts):
        s0 = np.zeros((heads, dk, dv)) if state is None else state[i]
        args = [x[n][row, lo:hi].astype(np.float64) for n in names]
        if back:
            o, s, d = delta(*args, scale, s0, x["do"][row, lo:hi].astype(np.float64),
                            x["dstate_out"][i] if "dstate_out" in x else None)
            for n in names:
                out["d" + n][row, lo:hi] = d["d" + n]
            out["dstate"][i] = d["dstate"]
        else:
            o, s = delta(*args, scale, s0)
        out["o"][row, lo:hi], out["state"][i] = o, s
    return out


# ---- norm block --------------------------------------------------------------

def _norm(x, kind, eps):
    if kind == "none":
        return x, None
    if kind == "layer":
        x = x - x.mean(-1, keepdims=True)
    inv = 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    return x * inv, inv


def _norm_back(d, xhat, inv, kind):
    if kind == "none":
        return d
    mean = d.mean(-1, keepdims=True) if kind == "layer" else 0.0
    return (d - mean - xhat * (d * xhat).mean(-1, keepdims=True)) * inv


def norm_block(x, post, pre, gate, scale, eps, p, seed, offset, back=False):
    """x: y, gate, residual, post_weight, post_bias, channel_scale, pre_weight,
    pre_bias as they are given. Forward: h and n. Backward, from y, gate, h,
    dh, dn: the gradients of everything given."""
    one = {n: x.get(n, v) for n, v in (("post_weight", 1.0), ("post_bias", 0.0), ("channel_scale", 1.0),
                                       ("pre_weight", 1.0), ("pre_bias", 0.0))}
    y = x["y"].astype(np.float64)
    yhat, yinv = _norm(y, post, eps)
    a = yhat * one["post_weight"] + one["post_bias"]
    act, slope = np.ones(y.shape), np.zeros(y.shape)
    if gate != "none":
        z = x["gate"].astype(np.float64)
        sig = 1.0 / (1.0 + np.exp(-z))
        act = z * sig if gate == "silu" else sig
        slope = sig * (1.0 + z * (1.0 - sig)) if gate == "silu" else sig * (1.0 - sig)
    t = scale * one["channel_scale"]
    if not back:
        h = x.get("residual", 0.0) + t * drop(a * act, p, seed, offset)
        out = {"h": h}
        if pre != "none":
            out["n"] = _norm(h, pre, eps)[0] * one["pre_weight"] + one["pre_bias"]
        return out
    out = {}
    dh = x["dh"].astype(np.float64)
    if pre != "none":
        dn = x["dn"].astype(np.float64)
        hhat, hinv = _norm(x["h"].astype(np.float64), pre, eps)
        out["pre_weight"], out["pre_bias"] = (dn * hhat).sum(0), dn.sum(0)
        dh = dh + _norm_back(dn * one["pre_weight"], hhat, hinv, pre)
    out["residual"] = dh
    out["channel_scale"] = (dh * scale * drop(a * act, p, seed, offset)).sum(0)
    db = drop(dh * t, p, seed, offset)
    out["gate"] = db * a * slope
    da = db * act
    out["post_weight"], out["post_bias"] = (da * yhat).sum(0), da.sum(0)
    out["y"] = _norm_back(da * one["post_weight"], yhat, yinv, post)
    return out
