"""What is timed when the speed of the layer operators is measured: the gated
delta rule (one token, a prompt, a training step), the norm block (a block's
output normalised, gated, dropped out, scaled and added to the residual, then
normalised for the next block; forward and backward) and dropout by itself.

``run`` computes a case in its plain form, elementary torch operations in 32
bits rounded once at the end, or, where ``own`` is true, through
``cudacaml_amd.operators``.
"""

import math

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
CHUNK = 64


def _delta(name, kind, dtype, batch, tokens, key_heads, value_heads, key_dim, value_dim, sequences=0, fused=False,
           state=True):
    return {"name": name, "kind": kind, "dtype": dtype, "batch": batch, "tokens": tokens, "key_heads": key_heads,
            "value_heads": value_heads, "key_dim": key_dim, "value_dim": value_dim, "sequences": sequences,
            "fused": fused, "state": state}


def _norm(name, kind, dtype, rows, width, norm="rms", pre="rms", gate="none", residual=True, dropout=0.0, weight="f32",
          bias=False, channel=False):
    return {"name": name, "kind": kind, "dtype": dtype, "rows": rows, "width": width, "norm": norm, "pre": pre,
            "gate": gate, "residual": residual, "dropout": dropout, "weight": weight, "bias": bias, "channel": channel}


def listed():
    return [
        # One token for each of a few streams: a chat server at low load,
        # where the time of a call is its latency.
        _delta("delta_step_8_f16", "delta", "f16", 8, 1, 16, 16, 128, 128),
        # One token for each of many streams, two value heads to a key head:
        # bound by the states, which are read and written once.
        _delta("delta_step_256", "delta", "bf16", 256, 1, 16, 32, 128, 128),
        # A long prompt, its q, k and v slices of one projection's output, and
        # the state that decoding goes on from.
        _delta("delta_prompt_16384", "delta", "bf16", 1, 16384, 16, 32, 128, 128, fused=True),
        # A training step on whole sequences, forward and backward.
        _delta("delta_train_4x4096", "train", "bf16", 4, 4096, 16, 32, 128, 128, state=False),
        # A training step on packed sequences of very different lengths, in
        # single precision and with heads of odd sizes, with the gradient of
        # the states they begin from.
        _delta("delta_train_packed_f32", "train", "f32", 1, 5003, 4, 8, 72, 100, sequences=9),
        # The norm block between two layers while decoding: 16 rows.
        _norm("norm_step_16x4096", "norm", "bf16", 16, 4096),
        # The same in training, with dropout and a learned scale a channel.
        _norm("norm_train_16384x4096", "norm", "bf16", 16384, 4096, dropout=0.1, channel=True),
        # Its backward pass.
        _norm("norm_back_16384x4096", "norm_back", "bf16", 16384, 4096, dropout=0.1, channel=True),
        # The backward pass of the norm and gate over each head of a recurrent
        # layer's output: short rows, very many of them.
        _norm("norm_back_heads_128", "norm_back", "bf16", 262144, 128, pre="none", gate="silu", residual=False,
              weight="bf16"),
        # Layer norms with biases in single precision, an odd number of rows
        # of odd width, forward.
        _norm("norm_layer_3001x1111_f32", "norm", "f32", 3001, 1111, norm="layer", pre="layer", gate="sigmoid",
              dropout=0.25, bias=True),
        # Dropout of an activation on its way to the residual, and the
        # gradient through it; the second case is small and of odd width.
        {"name": "dropout_16384x8192", "kind": "dropout", "dtype": "bf16", "rows": 16384, "cols": 8192, "p": 0.1,
         "residual": True},
        {"name": "dropout_301x1001_f16", "kind": "dropout", "dtype": "f16", "rows": 301, "cols": 1001, "p": 0.5,
         "residual": False},
    ]


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    kind = rng.choice(["step", "prompt", "train", "norm", "norm_back", "dropout"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind in ("step", "prompt", "train"):
        group = rng.choice([1, 2, 4])
        key_heads = log(1, 16)
        value_heads = key_heads * group
        key_dim, value_dim = rng.choice([(128, 128), (64, 64), (64, 128), (rng.randrange(16, 129), rng.randrange(8, 257))])
        if kind == "step":
            batch = log(1, max(1, 4096 // value_heads))
            return {k: v for k, v in _delta("", "delta", dtype, batch, 1, key_heads, value_heads, key_dim, value_dim,
                                            fused=rng.random() < 0.5).items() if k != "name"}
        room = 262144 if dtype == "bf16" else 65536
        tokens = log(2, max(2, min(16384 if kind == "prompt" else 4096, room // value_heads)))
        batch = log(1, max(1, min(16, room // (tokens * value_heads))))
        sequences = 0
        if rng.random() < 0.4:
            tokens, batch = tokens * batch, 1
            tokens = min(tokens, 8192)
            sequences = log(1, 12)
        return {k: v for k, v in _delta("", "train" if kind == "train" else "delta", dtype, batch, tokens, key_heads,
                                        value_heads, key_dim, value_dim, sequences=sequences, fused=rng.random() < 0.5,
                                        state=rng.random() < 0.5).items() if k != "name"}
    if kind == "dropout":
        cols = log(1, 16384)
        return {"kind": "dropout", "dtype": dtype, "rows": log(1, (1 << 26) // cols), "cols": cols,
                "p": rng.choice([0.0, 0.1, 0.5, rng.random()]), "residual": rng.random() < 0.5}
    width = rng.choice([128, 1024, 4096, 8192, log(16, 16384), log(16, 16384)])
    norm, pre = rng.choice([("rms", "rms"), ("layer", "layer"), ("rms", "none"), ("none", "rms")])
    c = _norm("", kind, dtype, log(1, (1 << 25) // width), width, norm=norm, pre=pre,
              gate=rng.choice(["none", "silu", "sigmoid"]), residual=rng.random() < 0.7,
              dropout=rng.choice([0.0, 0.1, rng.random()]), weight=rng.choice(["f32", dtype]),
              bias=norm == "layer" or pre == "layer", channel=rng.random() < 0.5)
    return {k: v for k, v in c.items() if k != "name"}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _offsets(case, g):
    """Where each packed sequence begins: random cuts, the second sequence of
    one token and the third empty where there are that many."""
    n, t = case["sequences"], case["tokens"]
    cuts = sorted(torch.randint(0, t + 1, (n - 1,), generator=g).tolist())
    if n >= 4:
        cuts[1] = min(t, cuts[0] + 1)
        cuts[2] = cuts[1]
        cuts = sorted(cuts)
    return [0] + cuts + [t]


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(int(seed))
    d = TYPES[case["dtype"]]

    def normal(*shape, dtype=d, mean=0.0, std=1.0):
        return (torch.randn(shape, device=DEV, generator=gen) * std + mean).to(dtype)

    s = {"case": case, "seed": int(seed) * 7919 + 12345}
    if case["kind"] in ("delta", "train"):
        b, t, hk, hv, dk, dv = (case[x] for x in ("batch", "tokens", "key_heads", "value_heads", "key_dim", "value_dim"))
        q = torch.nn.functional.normalize(torch.randn(b, t, hk, dk, device=DEV, generator=gen), dim=-1)
        k = torch.nn.functional.normalize(torch.randn(b, t, hk, dk, device=DEV, generator=gen), dim=-1)
        if case["fused"]:
            whole = torch.empty(b, t, 2 * hk * dk + hv * dv, device=DEV, dtype=d)
            s["q"] = whole[:, :, : hk * dk].unflatten(2, (hk, dk))
            s["k"] = whole[:, :, hk * dk: 2 * hk * dk].unflatten(2, (hk, dk))
            s["v"] = whole[:, :, 2 * hk * dk:].unflatten(2, (hv, dv))
            s["q"].copy_(q)
            s["k"].copy_(k)
            s["v"].copy_(normal(b, t, hv, dv))
        else:
            s["q"], s["k"], s["v"] = q.to(d), k.to(d), normal(b, t, hv, dv)
        # the decay of a head: a rate that differs from head to head times a
        # softplus of the token's projection, as such layers have it
        rate = torch.exp(torch.rand(hv, device=DEV, generator=gen) * 3.0 - 2.0)
        s["g"] = (-rate * torch.nn.functional.softplus(normal(b, t, hv, dtype=torch.float32, mean=-2.0))).to(d)
        s["beta"] = torch.sigmoid(normal(b, t, hv, dtype=torch.float32)).to(d)
        n = case["sequences"] or b
        if case["sequences"]:
            cpu = torch.Generator()
            cpu.manual_seed(int(seed))
            s["cuts"] = _offsets(case, cpu)
            s["offsets"] = torch.tensor(s["cuts"], dtype=torch.int32, device=DEV)
        if case["state"]:
            s["state"] = normal(n, hv, dk, dv, dtype=torch.float32, std=0.1)
        if case["kind"] == "train":
            s["do"] = normal(b, t, hv, dv)
            if case["state"]:
                s["dstate_out"] = normal(n, hv, dk, dv, dtype=torch.float32, std=0.1)
    elif case["kind"] in ("norm", "norm_back"):
        r, w = case["rows"], case["width"]
        wt = TYPES[case["weight"]]
        s["y"] = normal(r, w)
        if case["gate"] != "none":
            s["gate"] = normal(r, w)
        if case["kind"] == "norm" and case["residual"]:
            s["residual"] = normal(r, w, std=2.0)
        if case["norm"] != "none":
            s["post_weight"] = normal(w, dtype=wt, mean=1.0, std=0.1)
            if case["bias"]:
                s["post_bias"] = normal(w, dtype=wt, std=0.1)
        if case["channel"]:
            s["channel_scale"] = normal(w, dtype=wt, mean=1.0, std=0.1)
        if case["pre"] != "none":
            s["pre_weight"] = normal(w, dtype=wt, mean=1.0, std=0.1)
            if case["bias"]:
                s["pre_bias"] = normal(w, dtype=wt, std=0.1)
        if case["kind"] == "norm_back":
            s["dh"] = normal(r, w)
            if case["pre"] != "none":
                s["dn"] = normal(r, w)
                s["h"] = normal(r, w, std=2.0)
    else:
        s["x"], s["dout"] = normal(case["rows"], case["cols"]), normal(case["rows"], case["cols"])
        if case["residual"]:
            s["residual"] = normal(case["rows"], case["cols"])
    if own:
        s["op"] = _operator(case)
        if case["kind"] == "train":
            s["saved"] = torch.empty(s["op"].saved_bytes(), dtype=torch.uint8, device=DEV)
    return s


# What multiplies a block's output before the residual is added.
RESIDUAL_SCALE = 0.5
EPS = 1e-6


def _operator(case):
    """The handle that a user's program makes once for its shapes."""
    from cudacaml_amd import operators as O

    if case["kind"] in ("delta", "train"):
        return O.GatedDelta(case["dtype"], case["batch"], case["tokens"], case["key_heads"], case["value_heads"],
                            case["key_dim"], case["value_dim"], sequences=case["sequences"] or None,
                            states=case["state"])
    if case["kind"] in ("norm", "norm_back"):
        return O.NormBlock(case["dtype"], case["rows"], case["width"], norm=case["norm"], pre=case["pre"],
                           gate=case["gate"], dropout=case["dropout"], scale=RESIDUAL_SCALE, eps=EPS,
                           weight_dtype=case["weight"])
    return O.Dropout(case["dtype"], case["rows"], case["cols"], case["p"], scale=RESIDUAL_SCALE)


# ---------------------------------------------------------------------------
# A pass
# ---------------------------------------------------------------------------

def run(state):
    kind = state["case"]["kind"]
    if kind in ("delta", "train"):
        return _delta_own(state) if own else _delta_plain(state)
    if kind in ("norm", "norm_back"):
        return _norm_own(state) if own else _norm_plain(state)
    return _dropout_own(state) if own else _dropout_plain(state)


PARAMS = ("post_weight", "post_bias", "channel_scale", "pre_weight", "pre_bias")


def _delta_own(s):
    op, e = s["op"], torch.empty_like
    q, k, v, g, beta = s["q"], s["k"], s["v"], s["g"], s["beta"]
    out = {"o": v.new_empty(v.shape)}
    end = e(s["state"]) if "state" in s else None
    op.forward(q, k, v, g, beta, out["o"], state=s.get("state"), state_out=end, offsets=s.get("offsets"),
               saved=s.get("saved"))
    if end is not None:
        out["state"] = end
    if s["case"]["kind"] == "train":
        out.update(dq=q.new_empty(q.shape), dk=k.new_empty(k.shape), dv=v.new_empty(v.shape), dg=e(g), dbeta=e(beta))
        if end is not None:
            out["dstate"] = e(end)
        op.backward(q, k, v, g, beta, s["do"], s["saved"], out["dq"], out["dk"], out["dv"], out["dg"], out["dbeta"],
                    dstate_out=s.get("dstate_out"), dstate=out.get("dstate"), offsets=s.get("offsets"))
    return out


def _norm_own(s):
    op, e, case = s["op"], torch.empty_like, s["case"]
    params = {n: s[n] for n in PARAMS if n in s}
    if case["kind"] == "norm":
        out = {"h": e(s["y"])}
        if case["pre"] != "none":
            out["n"] = e(s["y"])
        op.forward(s["y"], out["h"], out.get("n"), gate=s.get("gate"), residual=s.get("residual"), seed=s["seed"],
                   offset=3, **params)
        return out
    out = {"dy": e(s["y"])}
    if "gate" in s:
        out["dgate"] = e(s["y"])
    if case["residual"]:
        out["dresidual"] = e(s["y"])
    for n in params:
        out["d" + n] = e(params[n])
    op.backward(s["y"], s["dh"], out["dy"], dn=s.get("dn"), h=s.get("h"), gate=s.get("gate"), dgate=out.get("dgate"),
                dresidual=out.get("dresidual"), seed=s["seed"], offset=3,
                grads={n: out["d" + n] for n in params}, **params)
    return out


def _dropout_own(s):
    out = {"out": torch.empty_like(s["x"]), "dx": torch.empty_like(s["x"])}
    s["op"].forward(s["x"], out["out"], residual=s.get("residual"), seed=s["seed"], offset=3)
    s["op"].backward(s["dout"], out["dx"], seed=s["seed"], offset=3)
    return out


def _by_sequence(s):
    """For packed tokens, which token stands at each place of a table of the
    sequences, and which places hold one; None where the batch is the table."""
    cuts = s.get("cuts")
    if cuts is None:
        return None
    first = torch.tensor(cuts[:-1], device=DEV)[:, None]
    length = torch.tensor(cuts, device=DEV).diff()[:, None]
    at = torch.arange(max(b - a for a, b in zip(cuts, cuts[1:])), device=DEV)[None, :]
    return (first + at).clamp_max(cuts[-1] - 1), at < length


def _in_chunks(x, where):
    """[batch, tokens, heads, ...] as [sequence, head, chunk, CHUNK, ...] in 32
    bits; places that hold no token are zero, which leaves a state as it is."""
    x = x.float()
    if where is not None:
        index, live = where
        x = x[0][index] * live.reshape(live.shape + (1,) * (x.dim() - 2))
    pad = -x.shape[1] % CHUNK
    if pad:
        x = torch.cat([x, x.new_zeros((x.shape[0], pad) + x.shape[2:])], 1)
    x = x.reshape((x.shape[0], x.shape[1] // CHUNK, CHUNK) + x.shape[2:])
    return x.movedim(3, 1).contiguous()


def _from_chunks(x, where, like):
    x = x.movedim(1, 3)
    x = x.reshape((x.shape[0], x.shape[1] * CHUNK) + x.shape[3:])
    if where is None:
        return x[:, : like.shape[1]].to(like.dtype)
    index, live = where
    out = x.new_zeros((like.shape[1],) + x.shape[2:])
    out[index[live]] = x[:, : index.shape[1]][live]
    return out[None].to(like.dtype)


def _unit_lower_inverse(a):
    """(I + a)^-1 of strictly lower triangular a, a row at a time."""
    t = torch.eye(CHUNK, device=a.device).expand(a.shape).contiguous()
    for i in range(1, CHUNK):
        t[..., i, :i] = -(a[..., i, None, :i] @ t[..., :i, :i])[..., 0, :]
    return t


def _step_plain(s):
    """The recurrence itself, for one token of each sequence."""
    case = s["case"]
    group = case["value_heads"] // case["key_heads"]
    q, k = (s[n][:, 0].float().repeat_interleave(group, 1) for n in ("q", "k"))
    v, g, beta = (s[n][:, 0].float() for n in ("v", "g", "beta"))
    state = torch.exp(g)[..., None, None] * s["state"]
    u = beta[..., None] * (v - (k[..., None, :] @ state)[..., 0, :])
    state = state + k[..., :, None] * u[..., None, :]
    o = case["key_dim"] ** -0.5 * (q[..., None, :] @ state)[..., 0, :]
    return {"o": o[:, None].to(s["v"].dtype), "state": state}


def _delta_plain(s):
    case = s["case"]
    if case["tokens"] == 1 and case["kind"] == "delta" and "state" in s and "cuts" not in s:
        return _step_plain(s)
    group = case["value_heads"] // case["key_heads"]
    scale = case["key_dim"] ** -0.5
    where = _by_sequence(s)
    q = _in_chunks(s["q"], where).repeat_interleave(group, 1)
    k = _in_chunks(s["k"], where).repeat_interleave(group, 1)
    v, g, beta = _in_chunks(s["v"], where), _in_chunks(s["g"], where), _in_chunks(s["beta"], where)[..., None]
    c = g.cumsum(-1)
    low = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=DEV).tril()
    decay = torch.exp((c[..., :, None] - c[..., None, :]).masked_fill(~low, -math.inf))
    first, last, end = torch.exp(c)[..., None], torch.exp(c[..., -1:] - c)[..., None], torch.exp(c[..., -1])[..., None, None]
    kk = (decay * (k @ k.transpose(-1, -2))).tril(-1)
    t = _unit_lower_inverse(beta * kk)
    p = decay * (q @ k.transpose(-1, -2))
    n, heads, chunks = k.shape[:3]
    state = s["state"] if "state" in s else torch.zeros(n, heads, case["key_dim"], case["value_dim"], device=DEV)
    states, us, os = [], [], []
    for i in range(chunks):
        x = v[:, :, i] - first[:, :, i] * (k[:, :, i] @ state)
        u = t[:, :, i] @ (beta[:, :, i] * x)
        os.append(scale * (first[:, :, i] * (q[:, :, i] @ state) + p[:, :, i] @ u))
        states.append(state)
        us.append(u)
        state = end[:, :, i] * state + k[:, :, i].transpose(-1, -2) @ (last[:, :, i] * u)
    out = {"o": _from_chunks(torch.stack(os, 2), where, s["v"])}
    if "state" in s:
        out["state"] = state
    if case["kind"] == "delta":
        return out
    do = _in_chunks(s["do"], where) * scale
    grad = s["dstate_out"] if "dstate_out" in s else torch.zeros_like(state)
    final, grads, ys = state, [None] * chunks, [None] * chunks
    for i in reversed(range(chunks)):
        grads[i] = grad
        du = p[:, :, i].transpose(-1, -2) @ do[:, :, i] + last[:, :, i] * (k[:, :, i] @ grad)
        y = t[:, :, i].transpose(-1, -2) @ du
        grad = (end[:, :, i] * grad + q[:, :, i].transpose(-1, -2) @ (first[:, :, i] * do[:, :, i])
                - k[:, :, i].transpose(-1, -2) @ (first[:, :, i] * beta[:, :, i] * y))
        ys[i] = y
    if "state" in s:
        out["dstate"] = grad
    y, u, s0, e = torch.stack(ys, 2), torch.stack(us, 2), torch.stack(states, 2), torch.stack(grads, 2)
    after = torch.stack(states[1:] + [final], 2)
    m = decay * (do @ u.transpose(-1, -2))
    f = y @ u.transpose(-1, -2)
    b = -(beta * decay * f).tril(-1)
    from_o, from_y, from_u = do @ s0.transpose(-1, -2), y @ s0.transpose(-1, -2), u @ e.transpose(-1, -2)
    dq = first * from_o + m @ k
    dk = (m.transpose(-1, -2) @ q + last * from_u - first * beta * from_y + (b + b.transpose(-1, -2)) @ k)
    dbeta = (y * v).sum(-1) - first[..., 0] * (from_y * k).sum(-1) - (f * kk).sum(-1)
    # what a pair (t, s) gives grows with c_t and falls with c_s
    pair = m * (q @ k.transpose(-1, -2)) + b * (k @ k.transpose(-1, -2))
    dc = pair.sum(-1) - pair.sum(-2) + (first * (q * from_o - beta * k * from_y)).sum(-1) - (last * k * from_u).sum(-1)
    dc[..., -1] += (after * e).sum((-1, -2))
    dg = dc.flip(-1).cumsum(-1).flip(-1)
    summed = [z.unflatten(1, (-1, group)).sum(2) for z in (dq, dk)]
    out.update(dq=_from_chunks(summed[0], where, s["q"]), dk=_from_chunks(summed[1], where, s["k"]),
               dv=_from_chunks(beta * y, where, s["v"]), dg=_from_chunks(dg, where, s["g"]),
               dbeta=_from_chunks(dbeta, where, s["beta"]))
    return out


M0, M1, W0, W1, LOW = 0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85, 0xFFFFFFFF


def _kept(rows, cols, p, seed, offset):
    """Which values dropout keeps: Philox4x32-10 at counter (col / 8, row,
    offset), key seed, gives eight 16-bit draws, and a value is kept if its
    draw is at least round(65536 p). Also the scale of a kept value."""
    bar = int(round(p * 65536.0))
    groups = -(-cols // 8)
    row = torch.arange(rows, device=DEV)[:, None].expand(rows, groups)
    c = [torch.arange(groups, device=DEV)[None, :].expand(rows, groups), row,
         torch.full_like(row, offset & LOW), torch.full_like(row, offset >> 32)]
    k0, k1 = seed & LOW, (seed >> 32) & LOW
    for _ in range(10):
        a, b = c[0] * M0, c[2] * M1
        c = [(b >> 32 & LOW) ^ c[1] ^ k0, b & LOW, (a >> 32 & LOW) ^ c[3] ^ k1, a & LOW]
        k0, k1 = k0 + W0 & LOW, k1 + W1 & LOW
    halves = torch.stack([h for w in c for h in (w & 0xFFFF, w >> 16)], -1)
    return halves.reshape(rows, groups * 8)[:, :cols] >= bar, 0.0 if bar >= 65536 else 65536.0 / (65536 - bar)


def _dropped(x, p, seed, offset):
    if p == 0.0:
        return x
    keep, up = _kept(x.shape[0], x.shape[1], p, seed, offset)
    return torch.where(keep, x * up, torch.zeros_like(x))


def _dropout_plain(s):
    p = s["case"]["p"]
    out = RESIDUAL_SCALE * _dropped(s["x"].float(), p, s["seed"], 3)
    if "residual" in s:
        out = out + s["residual"].float()
    dx = RESIDUAL_SCALE * _dropped(s["dout"].float(), p, s["seed"], 3)
    return {"out": out.to(s["x"].dtype), "dx": dx.to(s["x"].dtype)}


def _normed(x, kind):
    """x centred and over its root mean square, and what it was divided by."""
    if kind == "none":
        return x, None
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    inv = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
    return x * inv, inv


def _normed_back(d, xhat, inv, kind):
    if kind == "none":
        return d
    d = d - xhat * (d * xhat).mean(-1, keepdim=True) - (d.mean(-1, keepdim=True) if kind == "layer" else 0.0)
    return d * inv


def _norm_plain(s):
    case = s["case"]
    f = {n: s[n].float() for n in PARAMS if n in s}
    y = s["y"].float()
    yhat, yinv = _normed(y, case["norm"])
    a = yhat * f.get("post_weight", 1.0) + f.get("post_bias", 0.0)
    b = a
    if "gate" in s:
        z = s["gate"].float()
        sig = 1.0 / (1.0 + torch.exp(-z))
        act = z * sig if case["gate"] == "silu" else sig
        b = a * act
    d = s["y"].dtype
    if case["kind"] == "norm":
        h = RESIDUAL_SCALE * f.get("channel_scale", 1.0) * _dropped(b, case["dropout"], s["seed"], 3)
        if "residual" in s:
            h = h + s["residual"].float()
        out = {"h": h.to(d)}
        if case["pre"] != "none":
            out["n"] = (_normed(h, case["pre"])[0] * f["pre_weight"] + f.get("pre_bias", 0.0)).to(d)
        return out
    out = {}
    dh = s["dh"].float()
    if case["pre"] != "none":
        hhat, hinv = _normed(s["h"].float(), case["pre"])
        dn = s["dn"].float()
        out["dpre_weight"] = (dn * hhat).sum(0)
        if "pre_bias" in s:
            out["dpre_bias"] = dn.sum(0)
        dh = dh + _normed_back(dn * f["pre_weight"], hhat, hinv, case["pre"])
    if case["residual"]:
        out["dresidual"] = dh
    if "channel_scale" in s:
        out["dchannel_scale"] = (dh * RESIDUAL_SCALE * _dropped(b, case["dropout"], s["seed"], 3)).sum(0)
    db = _dropped(dh * RESIDUAL_SCALE * f.get("channel_scale", 1.0), case["dropout"], s["seed"], 3)
    da = db
    if "gate" in s:
        da = db * act
        out["dgate"] = db * a * (sig * (1.0 + z * (1.0 - sig)) if case["gate"] == "silu" else sig * (1.0 - sig))
    if case["norm"] != "none":
        out["dpost_weight"] = (da * yhat).sum(0)
        if "post_bias" in s:
            out["dpost_bias"] = da.sum(0)
    out["dy"] = _normed_back(da * f.get("post_weight", 1.0), yhat, yinv, case["norm"])
    return {n: x.to(s[n[1:]].dtype if n[1:] in PARAMS else d) for n, x in out.items()}


# ---------------------------------------------------------------------------
# What a pass cannot do without, and what it gives
# ---------------------------------------------------------------------------

def work(case):
    z = SIZE[case["dtype"]]
    if case["kind"] in ("delta", "train"):
        hk, hv, dk, dv = (case[x] for x in ("key_heads", "value_heads", "key_dim", "value_dim"))
        tokens = case["batch"] * case["tokens"]
        states = (case["sequences"] or case["batch"]) * hv * dk * dv * 4 if case["state"] else 0
        qk, vo, gates = 2 * tokens * hk * dk * z, tokens * hv * dv * z, 2 * tokens * hv * z
        forward = {"bytes": qk + 2 * vo + gates + 2 * states, "flops": 6 * tokens * hv * dk * dv}
        if case["kind"] == "delta":
            return forward
        # q, k, v and the gates are read once for the whole step
        return {"bytes": forward["bytes"] + qk + 2 * vo + gates + 2 * states, "flops": 3 * forward["flops"]}
    if case["kind"] == "dropout":
        n = case["rows"] * case["cols"]
        return {"bytes": (4 + case["residual"]) * n * z, "flops": 24 * n}
    n, w, wz = case["rows"] * case["width"], case["width"], SIZE[case["weight"]]
    norm, pre, gate = case["norm"] != "none", case["pre"] != "none", case["gate"] != "none"
    params = norm * (1 + case["bias"]) + pre * (1 + case["bias"]) + case["channel"]
    draws = 12 if case["dropout"] else 0
    if case["kind"] == "norm":
        return {"bytes": (2 + gate + case["residual"] + pre) * n * z + params * w * wz, "flops": (12 + 8 * gate + draws) * n}
    return {"bytes": (3 + 2 * gate + case["residual"] + 2 * pre) * n * z + 2 * params * w * wz,
            "flops": (30 + 16 * gate + draws) * n}


def _exact_sequence(q, k, v, g, beta, state, scale, do, dstate_out):
    """One sequence of some heads, token by token: o, the last state and, with
    `do`, every gradient. Tensors are [tokens, heads, ...] in 64 bits."""
    tokens, back = v.shape[0], do is not None
    o, alpha, states = torch.zeros_like(v), torch.exp(g), []
    for t in range(tokens):
        if back:
            states.append(state)
        seen = alpha[t][:, None, None] * state
        u = beta[t][:, None] * (v[t] - (seen * k[t][:, :, None]).sum(1))
        state = seen + k[t][:, :, None] * u[:, None, :]
        o[t] = scale * (state * q[t][:, :, None]).sum(1)
    if not back:
        return o, state, None
    e = torch.zeros_like(state) if dstate_out is None else dstate_out
    dq, dk, dv, dg, db = (torch.zeros_like(x) for x in (q, k, v, g, beta))
    for t in reversed(range(tokens)):
        al, be, kt = alpha[t][:, None], beta[t][:, None], k[t][:, :, None]
        before = states.pop()
        seen_k = (before * kt).sum(1)
        left = v[t] - al * seen_k
        u = be * left
        now = al[..., None] * before + kt * u[:, None, :]
        dq[t] = scale * (now * do[t][:, None, :]).sum(2)
        e = e + scale * q[t][:, :, None] * do[t][:, None, :]
        du = (e * kt).sum(1)
        db[t] = (du * left).sum(1)
        dleft = be * du
        dv[t] = dleft
        dk[t] = (e * u[:, None, :]).sum(2) - al * (before * dleft[:, None, :]).sum(2)
        dg[t] = alpha[t] * ((before * e).sum((1, 2)) - (dleft * seen_k).sum(1))
        e = al[..., None] * (e - kt * dleft[:, None, :])
    return o, state, (dq, dk, dv, dg, db, e)


def _exact_delta(case, s):
    group, train = case["value_heads"] // case["key_heads"], case["kind"] == "train"
    hv, dk, dv = case["value_heads"], case["key_dim"], case["value_dim"]
    cuts = s.get("cuts")
    rows = range(len(cuts) - 1) if cuts else [None]
    longest = max(b - a for a, b in zip(cuts, cuts[1:])) if cuts else case["tokens"]
    steps = case["tokens"]
    # the heads of all rows go through the tokens together; a backward pass
    # keeps every token's states, so it takes as many heads at a time as fit
    lanes = hv if cuts else hv * case["batch"]
    some = lanes if not train else max(1, min(lanes, int(40e9 // (max(1, longest) * dk * dv * 8))))
    if steps * -(-lanes // some) > (90000 if not train else 25000):
        return None
    wide = {n: s[n].double() for n in ("q", "k", "v", "g", "beta", "do", "state", "dstate_out") if n in s}
    for n in ("q", "k"):
        wide[n] = wide[n].repeat_interleave(group, 2)
    names = ("q", "k", "v", "g", "beta")
    got = {n: torch.zeros_like(wide[n if n != "o" else "v"]) for n in ("o",) + (names if train else ())}
    n_states = len(cuts) - 1 if cuts else case["batch"]
    begin = wide.get("state", torch.zeros(n_states, hv, dk, dv, dtype=torch.float64, device=DEV))
    ends, dbegin = torch.zeros_like(begin), torch.zeros_like(begin)

    def lanes_of(x, i):  # [tokens, lanes, ...] of packed sequence i or of the whole batch
        if cuts:
            return x[0, cuts[i]:cuts[i + 1]]
        return x.transpose(0, 1).flatten(1, 2)

    for i in rows:
        part = {n: lanes_of(wide[n], i) for n in names + (("do",) if train else ())}
        st = begin[i] if cuts else begin.flatten(0, 1)
        dst = (wide["dstate_out"][i] if cuts else wide["dstate_out"].flatten(0, 1)) if "dstate_out" in wide else None
        for lo in range(0, lanes, some):
            sl = slice(lo, min(lanes, lo + some))
            o, end, grads = _exact_sequence(*(part[n][:, sl] for n in names), st[sl], dk ** -0.5,
                                            part["do"][:, sl] if train else None, None if dst is None else dst[sl])
            if cuts:
                got["o"][0, cuts[i]:cuts[i + 1], sl] = o
                ends[i, sl] = end
            else:
                at = torch.arange(sl.start, sl.stop, device=DEV)
                got["o"][at // hv, :, at % hv] = o.transpose(0, 1)
                ends[at // hv, at % hv] = end
            for n, d in zip(names, (grads or ())[:5]):
                if cuts:
                    got[n][0, cuts[i]:cuts[i + 1], sl] = d
                else:
                    got[n][at // hv, :, at % hv] = d.transpose(0, 1)
            if train:
                if cuts:
                    dbegin[i, sl] = grads[5]
                else:
                    dbegin[at // hv, at % hv] = grads[5]
    out = {"o": got["o"]}
    if "state" in s:
        out["state"] = ends
    if train:
        out.update({"d" + n: got[n] for n in names})
        for n in ("dq", "dk"):
            out[n] = out[n].unflatten(2, (-1, group)).sum(3)
        if "state" in s:
            out["dstate"] = dbegin
    return out


def _exact_norm(case, s):
    """The definition in 64 bits; gradients by automatic differentiation."""
    t = {n: s[n].double() for n in s if n in PARAMS + ("y", "gate", "residual", "dh", "dn", "h")}
    back = case["kind"] == "norm_back"
    wanted = [n for n in ("y", "gate") + PARAMS if n in t]
    if back:
        for n in wanted:
            t[n].requires_grad_(True)

    def norm(x, kind):
        if kind == "layer":
            x = x - x.mean(-1, keepdim=True)
        return x if kind == "none" else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)

    b = norm(t["y"], case["norm"]) * t.get("post_weight", 1.0) + t.get("post_bias", 0.0)
    if case["gate"] != "none":
        b = b * (torch.sigmoid(t["gate"]) if case["gate"] == "sigmoid" else t["gate"] * torch.sigmoid(t["gate"]))
    if case["dropout"]:
        keep, up = _kept(case["rows"], case["width"], case["dropout"], s["seed"], 3)
        b = torch.where(keep, b * up, 0.0)
    h = b * t.get("channel_scale", 1.0) * RESIDUAL_SCALE + t.get("residual", 0.0)

    def next_norm(x):
        return norm(x, case["pre"]) * t["pre_weight"] + t.get("pre_bias", 0.0)

    if not back:
        return {"h": h, "n": next_norm(h)} if case["pre"] != "none" else {"h": h}
    out, dh = {}, t["dh"]
    if case["pre"] != "none":  # from h as it was stored
        at = t["h"].clone().requires_grad_(True)
        mine = [n for n in ("pre_weight", "pre_bias") if n in t]
        got = torch.autograd.grad(next_norm(at), [at] + [t[n] for n in mine], t["dn"])
        dh = dh + got[0]
        out.update({"d" + n: x for n, x in zip(mine, got[1:])})
    if case["residual"]:
        out["dresidual"] = dh
    rest = [n for n in wanted if not n.startswith("pre_")]
    out.update({"d" + n: x for n, x in zip(rest, torch.autograd.grad(h, [t[n] for n in rest], dh))})
    return out


def exact(case, seed):
    s = prepare({**case}, seed)
    if case["kind"] in ("delta", "train"):
        return _exact_delta(case, s)
    if case["kind"] in ("norm", "norm_back"):
        return _exact_norm(case, s)
    keep, up = ((True, 1.0) if case["p"] == 0.0 else _kept(case["rows"], case["cols"], case["p"], s["seed"], 3))
    keep = torch.as_tensor(keep, device=DEV)
    out = torch.where(keep, RESIDUAL_SCALE * up * s["x"].double(), 0.0)
    return {"out": out + s["residual"].double() if "residual" in s else out,
            "dx": torch.where(keep, RESIDUAL_SCALE * up * s["dout"].double(), 0.0)}
