"""What is timed when the speed of the operators of an attending layer is
measured: attention (one token for each sequence over a cache, a chunk of a
prompt over a cache, a prompt, a training step), the norm and rotation of its
heads (with the write to the cache while decoding, in training, and backward)
and the embedding lookup with its gradient.

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
EPS = 1e-6


def _attention(name, kind, dtype, batch, tokens, heads, kv_heads, head_dim, sequences=0, keys=0, fused=False):
    """kind "prompt" (forward) or "train" (forward and backward); ``sequences``
    packed into a batch of 1, or ``keys`` in a cache."""
    return {"name": name, "op": "attention", "kind": kind, "dtype": dtype, "batch": batch, "tokens": tokens, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "sequences": sequences, "keys": keys, "fused": fused}


def _heads(name, kind, dtype, batch, tokens, heads, kv_heads, head_dim, rotary=0, interleaved=False, norm="rms", weight="f32",
           keys=0, far=0):
    """kind "forward" or "backward"; ``keys`` in the cache that is written, or
    0; positions from 0 or, with ``far``, up to it."""
    return {"name": name, "op": "heads", "kind": kind, "dtype": dtype, "batch": batch, "tokens": tokens, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "rotary": rotary or head_dim, "interleaved": interleaved, "norm": norm,
            "weight": weight, "keys": keys, "far": far}


def _embedding(name, dtype, tokens, vocab, width, weight, kind="train", accumulate=False):
    """kind "forward" or "train" (the lookup and its gradient)."""
    return {"name": name, "op": "embedding", "kind": kind, "dtype": dtype, "tokens": tokens, "vocab": vocab, "width": width,
            "weight": weight, "accumulate": accumulate}


def listed():
    return [
        # One token for each of a few conversations: latency.
        _attention("attend_step_4x1024_f16", "prompt", "f16", 4, 1, 16, 4, 128, keys=1024),
        # One token for each of many: bound by the cache, which is read once.
        _attention("attend_step_64x8192", "prompt", "bf16", 64, 1, 32, 8, 128, keys=8192),
        # A chunk of a prompt over what the cache holds of it.
        _attention("attend_chunk_512", "prompt", "bf16", 2, 512, 32, 8, 128, keys=8192),
        # A whole prompt, its q, k and v slices of one projection's output.
        _attention("attend_prompt_8192", "prompt", "bf16", 1, 8192, 32, 8, 128, fused=True),
        # A training step on packed sequences of very different lengths.
        _attention("attend_train_packed", "train", "bf16", 1, 8192, 16, 4, 128, sequences=5),
        # A training step in single precision, heads of an odd size.
        _attention("attend_train_f32", "train", "f32", 3, 701, 6, 2, 72),
        # The heads of one token for each of 16 conversations, written to the cache.
        _heads("heads_step_16", "forward", "bf16", 16, 1, 32, 8, 128, keys=512),
        # The heads of a training step, forward.
        _heads("heads_train_16384", "forward", "bf16", 4, 4096, 32, 8, 128),
        # Their gradients.
        _heads("heads_back_16384", "backward", "bf16", 4, 4096, 32, 8, 128),
        # Gradients of heads of which a part is rotated, at far positions.
        _heads("heads_back_odd_f32", "backward", "f32", 1, 1009, 12, 3, 80, rotary=32, interleaved=True, far=1 << 20),
        # Text of a training step through a table of 65536 words and back.
        _embedding("embed_train_16384", "bf16", 16384, 65536, 2048, "bf16"),
        # A few tokens of single precision onto the gradient of a tied table.
        _embedding("embed_train_301_f32", "f32", 301, 5003, 520, "f32", accumulate=True),
    ]


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))

    kind = rng.choice(["step", "chunk", "prompt", "train", "heads", "heads", "embedding"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    group = rng.choice([1, 2, 3, 4, 7, 8])
    kv_heads = log(1, 8)
    dim = rng.choice([64, 128, 128, rng.randrange(8, 129)])
    if kind in ("step", "chunk", "prompt", "train"):
        heads, most = kv_heads * group, 2.5e8 if dtype == "f32" else 1e9
        if kind == "step":
            keys = log(16, 16384)
            c = _attention("", "prompt", dtype, log(1, max(1, min(128, (1 << 27) // (keys * heads)))), 1, heads, kv_heads, dim,
                           keys=keys)
        elif kind == "chunk":
            keys = log(64, 8192)
            tokens = log(2, min(keys, 1024))
            c = _attention("", "prompt", dtype, log(1, max(1, min(16, int(most / 4 / (heads * keys * tokens))))), tokens, heads,
                           kv_heads, dim, keys=keys)
        else:
            tokens = log(2, min(8192, int(math.sqrt(most / 2 / heads))))
            batch = log(1, max(1, min(16, int(most / 2 / (heads * tokens * tokens)))))
            sequences = 0
            if rng.random() < 0.4:
                batch, sequences = 1, log(1, min(12, tokens))
            c = _attention("", kind, dtype, batch, tokens, heads, kv_heads, dim, sequences=sequences, fused=rng.random() < 0.5)
    elif kind == "heads":
        tokens, batch = log(1, 4096), log(1, 4)
        keys = 0
        which = rng.choice(["forward", "forward", "backward"])
        if which == "forward" and rng.random() < 0.4:
            tokens, batch = log(1, 32), log(1, 64)
            keys = tokens + log(1, 512)
        c = _heads("", which, dtype, batch, tokens, kv_heads * group if kv_heads * group < 33 else kv_heads, kv_heads, dim,
                   rotary=rng.choice([dim // 2 * 2, dim // 4 * 2]), interleaved=rng.random() < 0.4,
                   norm=rng.choice(["rms", "rms", "none"]), weight=rng.choice(["f32", dtype]), keys=keys,
                   far=0 if keys else rng.choice([0, log(4096, 1 << 22)]))
    else:
        width = rng.choice([512, 2048, log(8, 4096)])
        vocab = log(16, (1 << 27) // width)
        c = _embedding("", dtype, log(1, (1 << 25) // width), vocab, width, rng.choice(["f32", dtype]),
                       kind=rng.choice(["forward", "train", "train"]), accumulate=rng.random() < 0.3)
    return {k: v for k, v in c.items() if k != "name"}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _lengths(case):
    """How many keys the sequences of a cache have: spread from the tokens that
    the call brings to the whole cache."""
    low, n = case["tokens"], case["batch"]
    return [case["keys"] - (case["keys"] - low) * i // n for i in range(n)]


def _pieces(case):
    """The lengths of packed sequences: each about 2/3 of the one before, of
    four or more one of a single token and one empty."""
    n, t = case["sequences"], case["tokens"]
    size = [(2 / 3) ** i for i in range(n)]
    out = [int(t * x / sum(size)) for x in size]
    if n >= 4:
        out[-1], out[-2] = 0, 1
    out[0] += t - sum(out)
    return out


def _angles(case):
    """Radians a position of each rotated pair."""
    half = case["rotary"] // 2
    return torch.tensor([10000.0 ** (-i / half) for i in range(half)], dtype=torch.float32, device=DEV)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(int(seed))
    d = TYPES[case["dtype"]]

    def normal(*shape, dtype=d, mean=0.0, std=1.0):
        return (torch.randn(shape, device=DEV, generator=gen) * std + mean).to(dtype)

    def shuffled(values):
        order = torch.randperm(len(values), generator=gen, device=DEV).tolist()
        return [values[i] for i in order]

    s = {"case": case}
    if case["op"] == "attention":
        b, t, h, hk, dim = (case[x] for x in ("batch", "tokens", "heads", "kv_heads", "head_dim"))
        n = case["keys"] or t
        if case["fused"]:
            whole = normal(b, t, h + 2 * hk, dim)
            s["q"], s["k"], s["v"] = whole[:, :, :h], whole[:, :, h:h + hk], whole[:, :, h + hk:]
        else:
            s["q"], s["k"], s["v"] = normal(b, t, h, dim), normal(b, n, hk, dim), normal(b, n, hk, dim)
        if case["keys"]:
            s["lengths"] = torch.tensor(shuffled(_lengths(case)), dtype=torch.int32, device=DEV)
        if case["sequences"]:
            cuts = [0]
            for x in shuffled(_pieces(case)):
                cuts.append(cuts[-1] + x)
            s["cuts"], s["offsets"] = cuts, torch.tensor(cuts, dtype=torch.int32, device=DEV)
        if case["kind"] == "train":
            s["do"] = normal(b, t, h, dim)
    elif case["op"] == "heads":
        b, t, h, hk, dim = (case[x] for x in ("batch", "tokens", "heads", "kv_heads", "head_dim"))
        wt = TYPES[case["weight"]]
        # heads as a projection gives them: q, k and v side by side
        whole = normal(b, t, h + 2 * hk, dim, std=2.0)
        s["q"], s["k"], s["v"] = whole[:, :, :h], whole[:, :, h:h + hk], whole[:, :, h + hk:]
        s["frequencies"] = _angles(case)
        if case["norm"] != "none":
            s["q_weight"], s["k_weight"] = normal(dim, dtype=wt, mean=1.0, std=0.1), normal(dim, dtype=wt, mean=1.0, std=0.1)
        first = torch.zeros(b, 1, dtype=torch.int64, device=DEV)
        if case["keys"]:
            first = torch.randint(0, case["keys"] - t + 1, (b, 1), generator=gen, device=DEV)
        if case["far"]:
            first = torch.randint(0, case["far"], (b, 1), generator=gen, device=DEV)
        s["positions"] = (first + torch.arange(t, device=DEV)).to(torch.int32)
        if case["keys"]:
            s["k_cache"], s["v_cache"] = normal(b, case["keys"], hk, dim), normal(b, case["keys"], hk, dim)
        if case["kind"] == "backward":
            s["dq_out"], s["dk_out"] = normal(b, t, h, dim), normal(b, t, hk, dim)
    else:
        # words by their frequency in text: the r-th has about 1 / r of it
        u = torch.rand(case["tokens"], device=DEV, generator=gen, dtype=torch.float64)
        rank = (torch.exp(u * math.log(case["vocab"])) - 1.0).long().clamp(0, case["vocab"] - 1)
        s["ids"] = torch.randperm(case["vocab"], generator=gen, device=DEV)[rank].to(torch.int32)
        s["weight"] = normal(case["vocab"], case["width"], dtype=TYPES[case["weight"]], std=0.02)
        if case["kind"] == "train":
            s["dout"] = normal(case["tokens"], case["width"])
            if case["accumulate"]:
                s["before"] = normal(case["vocab"], case["width"], dtype=TYPES[case["weight"]])
    if own:
        s["handle"] = _handle(case)
        if case["op"] == "attention" and case["kind"] == "train":
            s["saved"] = torch.empty(s["handle"].saved_bytes(), dtype=torch.uint8, device=DEV)
    return s


def _scale(case):
    """A lookup's scale is the root of the width, as where a table is tied to
    the output's weights."""
    return math.sqrt(case["width"])


def _handle(case):
    """The handle that a user's program makes once for its shapes."""
    from cudacaml_amd import operators as O

    if case["op"] == "attention":
        return O.Attention(case["dtype"], case["batch"], case["tokens"], case["heads"], case["kv_heads"], case["head_dim"],
                           sequences=case["sequences"] or None, keys=case["keys"] or None)
    if case["op"] == "heads":
        return O.HeadNorm(case["dtype"], case["batch"], case["tokens"], case["heads"], case["kv_heads"], case["head_dim"],
                          norm=case["norm"], rotary=case["rotary"], interleaved=case["interleaved"], eps=EPS,
                          weight_dtype=case["weight"], keys=case["keys"] or None)
    return O.Embedding(case["dtype"], case["tokens"], case["vocab"], case["width"], scale=_scale(case),
                       weight_dtype=case["weight"])


# ---------------------------------------------------------------------------
# A pass
# ---------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if op == "attention":
        return _attention_own(state) if own else _attention_plain(state)
    if op == "heads":
        return _heads_own(state) if own else _heads_plain(state)
    return _embedding_own(state) if own else _embedding_plain(state)


def _attention_own(s):
    q, k, v, op = s["q"], s["k"], s["v"], s["handle"]
    out = {"o": q.new_empty(q.shape)}
    op.forward(q, k, v, out["o"], offsets=s.get("offsets"), lengths=s.get("lengths"), saved=s.get("saved"))
    if s["case"]["kind"] == "train":
        out.update(dq=q.new_empty(q.shape), dk=k.new_empty(k.shape), dv=v.new_empty(v.shape))
        op.backward(q, k, v, out["o"], s["do"], s["saved"], out["dq"], out["dk"], out["dv"], offsets=s.get("offsets"))
    return out


def _heads_own(s):
    q, k, op, case = s["q"], s["k"], s["handle"], s["case"]
    common = dict(frequencies=s["frequencies"], positions=s["positions"], q_weight=s.get("q_weight"), k_weight=s.get("k_weight"))
    if case["kind"] == "forward":
        out = {"q": q.new_empty(q.shape)}
        if case["keys"]:
            op.forward(q, k, out["q"], v=s["v"], k_cache=s["k_cache"], v_cache=s["v_cache"], **common)
            return {"q": out["q"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
        out["k"] = k.new_empty(k.shape)
        op.forward(q, k, out["q"], out["k"], **common)
        return out
    out = {"dq": q.new_empty(q.shape), "dk": k.new_empty(k.shape)}
    grads = {}
    if case["norm"] != "none":
        grads = {n: torch.empty_like(s[n]) for n in ("q_weight", "k_weight")}
    op.backward(q, k, s["dq_out"], s["dk_out"], out["dq"], out["dk"], grads=grads, **common)
    return {**out, **{"d" + n: x for n, x in grads.items()}}


def _embedding_own(s):
    case, op = s["case"], s["handle"]
    out = {"out": torch.empty(case["tokens"], case["width"], dtype=TYPES[case["dtype"]], device=DEV)}
    op.forward(s["ids"], s["weight"], out["out"])
    if case["kind"] == "train":
        # a gradient that is added to: a copy, so that a pass can be repeated
        out["dweight"] = s["before"].clone() if case["accumulate"] else torch.empty_like(s["weight"])
        op.backward(s["ids"], s["dout"], out["dweight"], accumulate=case["accumulate"])
    return out


def _seen(s):
    """Which keys a query sees: [batch, tokens, keys]."""
    case = s["case"]
    t, n = case["tokens"], case["keys"] or case["tokens"]
    at, key = torch.arange(t, device=DEV)[:, None], torch.arange(n, device=DEV)[None, :]
    if case["keys"]:
        length = s["lengths"].long()[:, None, None]
        return key <= length - t + at
    if case["sequences"]:
        which = torch.bucketize(torch.arange(t, device=DEV), s["offsets"].long(), right=True)
        return ((key <= at) & (which[:, None] == which[None, :]))[None]
    return (key <= at)[None]


def _grouped(x, case):
    """[batch, tokens, heads, dim] as [batch, kv head, head of the group x token, dim] in 32 bits."""
    b, t, dim = x.shape[0], x.shape[1], x.shape[3]
    return x.float().reshape(b, t, case["kv_heads"], -1, dim).permute(0, 2, 3, 1, 4).reshape(b, case["kv_heads"], -1, dim)


def _ungrouped(x, case, like):
    b, dim = x.shape[0], x.shape[3]
    return x.reshape(b, case["kv_heads"], -1, like.shape[1], dim).permute(0, 3, 1, 2, 4).reshape(like.shape).to(like.dtype)


def _attention_plain(s):
    case = s["case"]
    scale = case["head_dim"] ** -0.5
    group = case["heads"] // case["kv_heads"]
    q, k, v = _grouped(s["q"], case), _grouped(s["k"], case), _grouped(s["v"], case)
    hidden = ~_seen(s)[:, None, None]
    x = (scale * q) @ k.transpose(-1, -2)
    by_head = x.view(x.shape[0], x.shape[1], group, case["tokens"], -1)
    by_head.masked_fill_(hidden, -math.inf)
    x -= x.amax(-1, keepdim=True).clamp_min(-3e38)
    p = x.exp_()
    p /= p.sum(-1, keepdim=True).clamp_min(1e-30)
    if case["keys"]:  # what a cache holds behind its sequence's end is anything
        live = torch.arange(case["keys"], device=DEV)[None, :] < s["lengths"][:, None]
        v = torch.where(live[:, None, :, None], v, 0.0)
    o = p @ v
    out = {"o": _ungrouped(o, case, s["q"])}
    if case["kind"] == "train":
        do = _grouped(s["do"], case)
        out["dv"] = _ungrouped(p.transpose(-1, -2) @ do, case, s["v"])
        ds = do @ v.transpose(-1, -2)
        ds -= (do * o).sum(-1, keepdim=True)
        ds *= p
        out["dq"] = _ungrouped(scale * (ds @ k), case, s["q"])
        out["dk"] = _ungrouped(scale * (ds.transpose(-1, -2) @ q), case, s["k"])
    return out


def _turn(s):
    """Cosine and sine of each token and pair; positions are far enough that
    their angles need 64 bits."""
    a = s["positions"].double()[..., None] * s["frequencies"].double()
    return a.cos().float()[:, :, None], a.sin().float()[:, :, None]


def _pairs(x, case):
    """The first and second elements of the rotated pairs, and the rest."""
    r = case["rotary"]
    if case["interleaved"]:
        return x[..., 0:r:2], x[..., 1:r:2], x[..., r:]
    return x[..., : r // 2], x[..., r // 2: r], x[..., r:]


def _joined(a, b, rest, case):
    if case["interleaved"]:
        return torch.cat([torch.stack([a, b], -1).flatten(-2), rest], -1)
    return torch.cat([a, b, rest], -1)


def _heads_plain(s):
    case = s["case"]
    cos, sin = _turn(s)
    if case["kind"] == "forward":
        def forward(x, w):
            x = x.float()
            if w is not None:
                x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
            a, b, rest = _pairs(x, case)
            return _joined(a * cos - b * sin, b * cos + a * sin, rest, case)

        q, k = forward(s["q"], s.get("q_weight")).to(s["q"].dtype), forward(s["k"], s.get("k_weight")).to(s["k"].dtype)
        if not case["keys"]:
            return {"q": q, "k": k}
        row = torch.arange(case["batch"], device=DEV)[:, None].expand(-1, case["tokens"])
        s["k_cache"][row, s["positions"].long()] = k
        s["v_cache"][row, s["positions"].long()] = s["v"]
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}

    def backward(x, g, w):
        a, b, rest = _pairs(g.float(), case)
        g = _joined(a * cos + b * sin, b * cos - a * sin, rest, case)
        if w is None:
            return g, None
        x = x.float()
        inv = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
        x = x * inv
        dw = (g * x).sum((0, 1, 2))
        g = g * w.float()
        return (g - x * (g * x).mean(-1, keepdim=True)) * inv, dw

    dq, dqw = backward(s["q"], s["dq_out"], s.get("q_weight"))
    dk, dkw = backward(s["k"], s["dk_out"], s.get("k_weight"))
    out = {"dq": dq.to(s["q"].dtype), "dk": dk.to(s["k"].dtype)}
    if dqw is not None:
        out.update(dq_weight=dqw.to(s["q_weight"].dtype), dk_weight=dkw.to(s["k_weight"].dtype))
    return out


def _embedding_plain(s):
    case = s["case"]
    ids = s["ids"].long()
    out = {"out": (_scale(case) * s["weight"][ids].float()).to(TYPES[case["dtype"]])}
    if case["kind"] == "train":
        if case["accumulate"]:
            total = s["before"].float()
            if total is s["before"]:
                total = total.clone()
        else:
            total = torch.zeros(case["vocab"], case["width"], device=DEV)
        total.index_add_(0, ids, s["dout"].float(), alpha=_scale(case))
        out["dweight"] = total.to(s["weight"].dtype)
    return out


# ---------------------------------------------------------------------------
# What a pass cannot do without, and what it gives
# ---------------------------------------------------------------------------

def work(case):
    z = SIZE[case["dtype"]]
    if case["op"] == "attention":
        b, t, h, hk, dim = (case[x] for x in ("batch", "tokens", "heads", "kv_heads", "head_dim"))
        if case["keys"]:
            lengths = _lengths(case)
            pairs, held = sum(t * n - t * (t - 1) // 2 for n in lengths), sum(lengths)
        else:
            sizes = _pieces(case) if case["sequences"] else [t] * b
            pairs, held = sum(n * (n + 1) // 2 for n in sizes), b * t
        qo, kv = b * t * h * dim * z, held * hk * dim * z
        if case["kind"] == "prompt":
            return {"bytes": 2 * qo + 2 * kv, "flops": 4 * dim * pairs * h}
        # q, k and v are read once for the whole step
        return {"bytes": 4 * qo + 4 * kv, "flops": 14 * dim * pairs * h}
    if case["op"] == "heads":
        rows, h, hk, dim = case["batch"] * case["tokens"], case["heads"], case["kv_heads"], case["head_dim"]
        vectors = (2 * dim * SIZE[case["weight"]] if case["norm"] != "none" else 0) + 2 * case["rotary"] + 4 * rows
        if case["kind"] == "forward":
            return {"bytes": rows * (2 * h + 2 * hk + (2 * hk if case["keys"] else 0)) * dim * z + vectors,
                    "flops": 8 * rows * (h + hk) * dim}
        return {"bytes": 3 * rows * (h + hk) * dim * z + 2 * vectors, "flops": 18 * rows * (h + hk) * dim}
    n, w, wz = case["tokens"], case["width"], SIZE[case["weight"]]
    # words that come up more than once are read once: of the tokens' words by frequency, the different ones
    log_v = math.log(case["vocab"])
    different = min(case["vocab"], sum(-math.expm1(-n * math.log1p(1 / r) / log_v) for r in range(1, min(case["vocab"], 4096) + 1))
                    + sum(-math.expm1(-n / (r * log_v)) * max(1, r // 64) for r in _steps(4096, case["vocab"])))
    out = {"bytes": int(4 * n + different * w * wz + n * w * z), "flops": n * w}
    if case["kind"] == "train":
        out["bytes"] += int(n * w * z + (2 * different if case["accumulate"] else case["vocab"]) * w * wz)
        out["flops"] += 2 * n * w
    return out


def _steps(lo, hi):
    """Ranks from lo to hi, each standing for itself over 64 as many."""
    out, r = [], lo + 1
    while r <= hi:
        out.append(r)
        r += max(1, r // 64)
    return out


def _exact_attention(case, s):
    """The definition in 64 bits, a group of heads of a sequence at a time;
    gradients by automatic differentiation."""
    train, group = case["kind"] == "train", case["heads"] // case["kv_heads"]
    t = case["tokens"]
    parts = [(i, 0, t, 0, int(n)) for i, n in enumerate(s["lengths"].tolist())] if case["keys"] else \
            [(0, a, b, a, b) for a, b in zip(s["cuts"], s["cuts"][1:])] if case["sequences"] else \
            [(i, 0, t, 0, t) for i in range(case["batch"])]
    names = {"q": "dq", "k": "dk", "v": "dv"}
    out = {"o": torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)}
    if train:
        out.update({names[n]: torch.zeros(s[n].shape, dtype=torch.float64, device=DEV) for n in names})
    for row, qa, qb, ka, kb in parts:
        last = torch.arange(qb - qa, device=DEV) + (kb - ka) - (qb - qa)
        blind = torch.arange(kb - ka, device=DEV)[None, :] > last[:, None]
        for kv in range(case["kv_heads"]):
            if qb == qa or kb == ka:
                continue
            mine = slice(kv * group, (kv + 1) * group)
            q = s["q"][row, qa:qb, mine].double().transpose(0, 1).contiguous().requires_grad_(train)
            k, v = (s[n][row, ka:kb, kv].double().contiguous().requires_grad_(train) for n in ("k", "v"))
            x = (q @ k.t() / math.sqrt(case["head_dim"])).masked_fill(blind, -math.inf)
            p = torch.softmax(x, -1).masked_fill(blind, 0.0)
            o = p @ v
            out["o"][row, qa:qb, mine] = o.detach().transpose(0, 1)
            if train:
                do = s["do"][row, qa:qb, mine].double().transpose(0, 1)
                dq, dk, dv = torch.autograd.grad(o, (q, k, v), do)
                out["dq"][row, qa:qb, mine] = dq.transpose(0, 1)
                out["dk"][row, ka:kb, kv], out["dv"][row, ka:kb, kv] = dk, dv
    return out


def _exact_heads(case, s):
    """Pairs as complex numbers in 64 bits; gradients by automatic
    differentiation."""
    r = case["rotary"]
    angle = s["positions"].double()[..., None] * s["frequencies"].double()
    turn = torch.polar(torch.ones_like(angle), angle)[:, :, None]

    def f(x, w):
        if w is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w
        if not r:
            return x
        if case["interleaved"]:
            z = torch.complex(x[..., 0:r:2].contiguous(), x[..., 1:r:2].contiguous()) * turn
            head = torch.view_as_real(z).flatten(-2)
        else:
            z = torch.complex(x[..., : r // 2].contiguous(), x[..., r // 2: r].contiguous()) * turn
            head = torch.cat([z.real, z.imag], -1)
        return torch.cat([head, x[..., r:]], -1)

    out = {}
    for n in ("q", "k"):
        x = s[n].double().contiguous()
        w = s[n + "_weight"].double() if n + "_weight" in s else None
        if case["kind"] == "forward":
            out[n] = f(x, w)
            continue
        x.requires_grad_(True)
        wanted = [x] + ([w.requires_grad_(True)] if w is not None else [])
        got = torch.autograd.grad(f(x, w), wanted, s["d" + n + "_out"].double())
        out["d" + n] = got[0]
        if w is not None:
            out["d" + n + "_weight"] = got[1]
    if case["keys"]:
        row, at = torch.arange(case["batch"], device=DEV)[:, None], s["positions"].long()
        caches = {"k_cache": s["k_cache"].double(), "v_cache": s["v_cache"].double()}
        caches["k_cache"][row, at], caches["v_cache"][row, at] = out["k"], s["v"].double()
        return {"q": out["q"], **caches}
    return out


def exact(case, seed):
    s = prepare({**case}, seed)
    if case["op"] == "attention":
        return _exact_attention(case, s)
    if case["op"] == "heads":
        return _exact_heads(case, s)
    ids, scale = s["ids"].long(), math.sqrt(case["width"])
    out = {"out": s["weight"].double()[ids] * scale}
    if case["kind"] == "train":
        order = ids.argsort(stable=True)
        words, counts = ids[order].unique_consecutive(return_counts=True)
        # sums of runs of equal words, as differences of one running sum
        run_sum = (s["dout"].double()[order] * scale).cumsum(0)
        ends = run_sum[counts.cumsum(0) - 1]
        total = s["before"].double() if case["accumulate"] else torch.zeros(s["weight"].shape, dtype=torch.float64, device=DEV)
        total[words] += torch.cat([ends[:1], ends[1:] - ends[:-1]])
        out["dweight"] = total
    return out
