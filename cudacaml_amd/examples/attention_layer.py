"""A layer of an attending language model, trained on words and then run word by
word over a cache: the array graphs of this package for its products, and the
layer operators between them, all on residents that never leave the GPU.

    x  = embedding of the words, [tokens, width]        Embedding
    n  = norm(x)                                        NormBlock
    q, k, v = projections of n                          graph (matmul)
    q, k = norm and rotation of their heads             HeadNorm (serving: into the cache)
    o  = causal attention, heads in groups              Attention (serving: over the cache)
    y  = o Wo                                           graph (matmul)
    h  = x + norm(y), m = norm(h)                       NormBlock
    loss = mean((m We - target)^2)                      graph

    python -m cudacaml_amd.examples.attention_layer
"""

from __future__ import annotations

import numpy as np

from .. import backend_hip as H
from .. import dsl as D
from .. import grad as G
from .. import operators as O
from ..ir import F32, Graph
from ..runtime import Buffer
from .delta_layer import _vjp


class Sizes:
    def __init__(self, batch=2, tokens=48, width=64, heads=4, kv_heads=2, head_dim=16, vocab=40, out=16):
        self.batch, self.tokens, self.width = batch, tokens, width
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.vocab, self.out = vocab, out

    def rows(self):
        return self.batch * self.tokens


PROJECTIONS = ("wq", "wk", "wv")


def _projections(z, rows):
    n = D.param("n", F32, (rows, z.width))
    return [(name, D.matmul(n, D.param("w" + name, F32, (z.width, heads * z.head_dim))))
            for name, heads in (("q", z.heads), ("k", z.kv_heads), ("v", z.kv_heads))]


class Layer:
    """The compiled graphs, the operators' handles and the weights."""

    def __init__(self, z, seed=0):
        self.z = z
        self.made = []
        r, qd, kd = z.rows(), z.heads * z.head_dim, z.kv_heads * z.head_dim
        self.compiled, self.handles = {}, {}
        for one, rows, tokens, keys in (("", r, z.tokens, None), ("_one", z.batch, 1, z.tokens)):
            self.compiled["project" + one] = H.compile(Graph.create("project", _projections(z, rows)))
            y = D.matmul(D.param("o", F32, (rows, qd)), D.param("wo", F32, (qd, z.width)))
            self.compiled["mix" + one] = H.compile(Graph.create("mix", [("y", y)]))
            p = D.matmul(D.param("m", F32, (rows, z.width)), D.param("we", F32, (z.width, z.out)))
            self.compiled["predict" + one] = H.compile(Graph.create("predict", [("p", p)]))
            self.handles.update({
                "embed" + one: O.Embedding("f32", rows, z.vocab, z.width, scale=z.width ** 0.5),
                "first" + one: O.NormBlock("f32", rows, z.width, norm="none", pre="rms"),
                "turn" + one: O.HeadNorm("f32", z.batch, tokens, z.heads, z.kv_heads, z.head_dim, keys=keys),
                "attend" + one: O.Attention("f32", z.batch, tokens, z.heads, z.kv_heads, z.head_dim, keys=keys),
                "block" + one: O.NormBlock("f32", rows, z.width, norm="rms", pre="rms"),
            })
            if not one:
                self.compiled["mix_back"] = H.compile(_vjp("mix_back", [("y", y)], ["o", "wo"]))
        self.compiled["project_back"] = H.compile(_vjp("project_back", _projections(z, r), ["n"] + list(PROJECTIONS)))
        e = D.map2(D.sub, D.matmul(D.param("m", F32, (r, z.width)), D.param("we", F32, (z.width, z.out))),
                   D.param("target", F32, (r, z.out)))
        loss = D.reduce(D.add, D.const(F32, 0.0),
                        D.flatten(D.map(lambda d: D.mul(D.mul(d, d), D.const(F32, 1.0 / (r * z.out))), e)))
        self.compiled["loss"] = H.compile(G.grad(Graph.create("loss", [("loss", loss)]), "loss", ["m", "we"]))

        g = np.random.default_rng(seed)
        shapes = {"words": (z.vocab, z.width), "wq": (z.width, qd), "wk": (z.width, kd), "wv": (z.width, kd), "wo": (qd, z.width),
                  "we": (z.width, z.out), "first": (z.width,), "post": (z.width,), "pre": (z.width,), "qn": (z.head_dim,),
                  "kn": (z.head_dim,)}
        self.weights = {n: (np.ones(s) if len(s) == 1 else g.standard_normal(s) / np.sqrt(s[-1] if n == "words" else s[0])
                            ).astype(np.float32) for n, s in shapes.items()}
        self.frequencies = (100.0 ** (-np.arange(z.head_dim // 2) / (z.head_dim // 2))).astype(np.float32)
        self._upload()

    def _upload(self):
        for r in getattr(self, "device", {}).values():
            H.free_resident(r)
        self.device = {n: H.upload(w) for n, w in self.weights.items()}
        self.device["frequencies"] = H.upload(self.frequencies)

    # What a call makes on the way, freed when it ends.

    def _keep(self, r):
        self.made.append(r)
        return r

    def _empty(self, *shape):
        return self._keep(H.Resident(Buffer.alloc(4 * int(np.prod(shape))), F32, shape))

    def _graph(self, name, **inputs):
        out = dict(H.run_resident(self.compiled[name], inputs))
        self.made += out.values()
        return out

    def _done(self):
        for b in {id(r.buf): r.buf for r in self.made}.values():
            b.free()
        self.made = []

    def _heads(self, r, heads):
        """[rows, heads head_dim] as [batch, tokens, heads, head_dim]."""
        return O.Array(r.buf, "f32", (self.z.batch, r.shape[0] // self.z.batch, heads, self.z.head_dim))

    def _forward(self, ids, one="", cache=None, saved=None):
        """All of the layer's values; ``cache``: k and v, positions and lengths."""
        z, w, op = self.z, self.device, self.handles
        rows, qd = len(ids), z.heads * z.head_dim
        a = {"ids": self._keep(H.upload(np.ascontiguousarray(ids, dtype=np.int32)))}
        a.update({n: self._empty(rows, z.width) for n in ("x", "h0", "n", "h", "m")}, o=self._empty(rows, qd), qr=self._empty(rows, qd))
        op["embed" + one].forward(a["ids"], w["words"], a["x"])
        op["first" + one].forward(a["x"], a["h0"], a["n"], pre_weight=w["first"])
        a.update(self._graph("project" + one, n=a["n"], **{n: w[n] for n in PROJECTIONS}))
        q, qr, o = (self._heads(a[n], z.heads) for n in ("q", "qr", "o"))
        k, v = (self._heads(a[n], z.kv_heads) for n in ("k", "v"))
        turn = dict(frequencies=w["frequencies"], q_weight=w["qn"], k_weight=w["kn"])
        if cache:
            op["turn" + one].forward(q, k, qr, positions=cache["positions"], v=v, k_cache=cache["k"], v_cache=cache["v"], **turn)
            op["attend" + one].forward(qr, cache["k"], cache["v"], o, lengths=cache["lengths"])
        else:
            a["kr"] = self._empty(rows, z.kv_heads * z.head_dim)
            kr = self._heads(a["kr"], z.kv_heads)
            op["turn"].forward(q, k, qr, kr, **turn)
            op["attend"].forward(qr, kr, v, o, saved=saved)
        a.update(self._graph("mix" + one, o=a["o"], wo=w["wo"]))
        op["block" + one].forward(a["y"], a["h"], a["m"], residual=a["x"], post_weight=w["post"], pre_weight=w["pre"])
        return a

    def gradients(self, ids, target):
        """The loss for words ``ids`` [tokens] and ``target`` [tokens, out], and
        its gradient with respect to each weight."""
        z, r, w, op = self.z, self.z.rows(), self.device, self.handles
        saved = self._keep(op["attend"].saved())
        a = self._forward(ids, saved=saved)
        top = self._graph("loss", m=a["m"], we=w["we"], target=self._keep(H.upload(target)))
        grads = {n: self._empty(*s.shape) for n, s in self.weights.items() if n in ("words", "first", "post", "pre", "qn", "kn")}
        grads["we"] = top["dloss/dwe"]
        zero = self._keep(H.upload(np.zeros((r, z.width), np.float32)))
        dy, dx0, dx = (self._empty(r, z.width) for _ in range(3))
        op["block"].backward(a["y"], zero, dy, dn=top["dloss/dm"], h=a["h"], dresidual=dx0, post_weight=w["post"], pre_weight=w["pre"],
                             grads=dict(post_weight=grads["post"], pre_weight=grads["pre"]))
        back = self._graph("mix_back", o=a["o"], wo=w["wo"], dy=dy)
        grads["wo"] = back["ds/dwo"]
        d = {n: self._empty(*a[n].shape) for n in ("q", "k", "v")}
        at = {n: self._heads(a[n], z.heads if n in ("q", "qr", "o") else z.kv_heads) for n in ("q", "k", "v", "qr", "kr", "o")}
        dq, dk, dv = (self._heads(d[n], z.heads if n == "q" else z.kv_heads) for n in ("q", "k", "v"))
        op["attend"].backward(at["qr"], at["kr"], at["v"], at["o"], self._heads(back["ds/do"], z.heads), saved, dq, dk, dv)
        op["turn"].backward(at["q"], at["k"], dq, dk, dq, dk, frequencies=w["frequencies"], q_weight=w["qn"], k_weight=w["kn"],
                            grads=dict(q_weight=grads["qn"], k_weight=grads["kn"]))
        back = self._graph("project_back", n=a["n"], **{n: w[n] for n in PROJECTIONS}, **{"d" + n: t for n, t in d.items()})
        grads.update({n: back["ds/d" + n] for n in PROJECTIONS})
        op["first"].backward(a["x"], dx0, dx, dn=back["ds/dn"], h=a["h0"], pre_weight=w["first"], grads=dict(pre_weight=grads["first"]))
        op["embed"].backward(a["ids"], dx, grads["words"])
        loss = float(H.download(top["loss"]))
        grads = {n: H.download(t).reshape(self.weights[n].shape) for n, t in grads.items()}
        self._done()
        return loss, grads

    def step(self, ids, target, rate=0.1):
        """One step of training; the loss before it."""
        loss, grads = self.gradients(ids, target)
        for n, g in grads.items():
            self.weights[n] = (self.weights[n] - rate * g).astype(np.float32)
        self._upload()
        return loss

    def evaluate(self, ids):
        """The outputs for whole sequences in one pass."""
        a = self._forward(ids)
        out = H.download(self._graph("predict", m=a["m"], we=self.device["we"])["p"])
        self._done()
        return out

    def predict(self, ids):
        """The same a word at a time, with a cache of what came before."""
        z = self.z
        ids = ids.reshape(z.batch, z.tokens)
        cache = {n: O.Array.empty("f32", (z.batch, z.tokens, z.kv_heads, z.head_dim)) for n in ("k", "v")}
        out = np.empty((z.batch, z.tokens, z.out), np.float32)
        for t in range(z.tokens):
            at = [self._keep(H.upload(np.full(z.batch, x, np.int32))) for x in (t, t + 1)]
            cache.update(positions=O.Array(at[0].buf, "i32", (z.batch, 1)), lengths=at[1])
            a = self._forward(ids[:, t], "_one", cache)
            out[:, t] = H.download(self._graph("predict_one", m=a["m"], we=self.device["we"])["p"])
            self._done()
        for n in ("k", "v"):
            cache[n].free()
        return out.reshape(z.rows(), z.out)

    def release(self):
        for c in self.compiled.values():
            c.release()
        for op in self.handles.values():
            op.free()
        for r in self.device.values():
            H.free_resident(r)
        self.device = {}


def recall_task(z, seed):
    """Words, and for each the vector that stands for the word two before it."""
    g = np.random.default_rng(seed)
    ids = g.integers(0, z.vocab, (z.batch, z.tokens)).astype(np.int32)
    meaning = g.standard_normal((z.vocab, z.out)).astype(np.float32)
    target = meaning[np.roll(ids, 2, axis=1)]
    target[:, :2] = 0.0
    return ids.reshape(-1), target.reshape(z.rows(), z.out)


def main(steps=40):
    z = Sizes()
    layer = Layer(z)
    ids, target = recall_task(z, 1)
    for i in range(steps):
        loss = layer.step(ids, target)
        if i % 10 == 0 or i == steps - 1:
            print("step %2d loss %.4f" % (i, loss), flush=True)
    a, b = layer.predict(ids), layer.evaluate(ids)
    print("word by word against whole sequences: largest difference %.2g" % np.abs(a - b).max(), flush=True)
    layer.release()


if __name__ == "__main__":
    main()
