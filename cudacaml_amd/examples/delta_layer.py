"""A layer of a recurrent language model, trained and then run token by token:
the array graphs of this package for its products, and the layer operators
between them, all on residents that never leave the GPU.

    x  = the residual stream, [tokens, width]
    n  = norm(x)                                       NormBlock
    q, k, v, g, beta = projections of n                graph (matmul, maps)
    o  = gated delta rule                              GatedDelta
    y  = o Wo                                          graph (matmul)
    h  = x + drop(norm(y)), n' = norm(h)               NormBlock
    loss = mean((drop(n') We - target)^2)              Dropout, graph

Gradients of the graphs come from ``Grad``: the gradient of
``sum(output * given)`` is the vector-Jacobian product that a chain of
operators needs.

    python -m cudacaml_amd.examples.delta_layer
"""

from __future__ import annotations

import numpy as np

from .. import backend_hip as H
from .. import dsl as D
from .. import grad as G
from .. import operators as O
from ..ir import F32, I32, Graph
from ..runtime import Buffer


class Sizes:
    def __init__(self, batch=2, tokens=96, width=64, heads=2, key_dim=32, value_dim=32, out=16):
        self.batch, self.tokens, self.width, self.heads = batch, tokens, width, heads
        self.key_dim, self.value_dim, self.out = key_dim, value_dim, out

    def rows(self):
        return self.batch * self.tokens


def _unit_rows(x, heads, dim):
    """Each head of each row over its 2-norm."""
    n = x.shape[0]
    r = D.reshape((n * heads, dim), x)
    sq = D.reduce_rows(D.add, D.const(F32, 0.0), D.map(lambda e: D.mul(e, e), r))
    inv = D.map(lambda s: D.div(D.const(F32, 1.0), D.sqrt(D.add(s, D.const(F32, 1e-6)))), sq)
    row = D.map(lambda i: D.div(i, D.const(I32, dim)), D.iota((n * heads, dim)))
    return D.reshape((n, heads * dim), D.map2(D.mul, r, D.gather(row, inv)))


def _projections(z, rows):
    n = D.param("n", F32, (rows, z.width))

    def project(name, cols):
        return D.matmul(n, D.param(name, F32, (z.width, cols)))

    one = D.const(F32, 1.0)
    # a decay of softplus(-a) a token, about 0.3 at the start
    g = D.map(lambda a: D.neg(D.log(D.add(one, D.exp(D.sub(D.neg(a), one))))), project("wg", z.heads))
    beta = D.map(lambda b: D.div(one, D.add(one, D.exp(D.neg(b)))), project("wb", z.heads))
    return [("q", _unit_rows(project("wq", z.heads * z.key_dim), z.heads, z.key_dim)),
            ("k", _unit_rows(project("wk", z.heads * z.key_dim), z.heads, z.key_dim)),
            ("v", project("wv", z.heads * z.value_dim)), ("g", g), ("beta", beta)]


def _vjp(name, outputs, wrt):
    """The gradients of sum(output * given) over the outputs, ``given`` a
    parameter d<output> for each."""
    total = None
    for n, t in outputs:
        s = D.reduce(D.add, D.const(F32, 0.0), D.flatten(D.map2(D.mul, t, D.param("d" + n, F32, t.shape))))
        total = s if total is None else D.map2(D.add, total, s)
    return G.grad(Graph.create(name, [("s", total)]), "s", wrt)


PROJECTIONS = ("wq", "wk", "wv", "wg", "wb")


class Layer:
    """The compiled graphs, the operators' handles and the weights."""

    def __init__(self, z, seed=0, dropout=0.1):
        self.z = z
        r = z.rows()
        self.compiled = {
            "project": H.compile(Graph.create("project", _projections(z, r))),
            "project_back": H.compile(_vjp("project_back", _projections(z, r), ["n"] + list(PROJECTIONS))),
            "project_one": H.compile(Graph.create("project_one", _projections(z, z.batch))),
        }
        for suffix, rows in (("", r), ("_one", z.batch)):
            o = D.param("o", F32, (rows, z.heads * z.value_dim))
            y = D.matmul(o, D.param("wo", F32, (z.heads * z.value_dim, z.width)))
            self.compiled["mix" + suffix] = H.compile(Graph.create("mix", [("y", y)]))
            if not suffix:
                self.compiled["mix_back"] = H.compile(_vjp("mix_back", [("y", y)], ["o", "wo"]))
            n = D.param("m", F32, (rows, z.width))
            p = D.matmul(n, D.param("we", F32, (z.width, z.out)))
            self.compiled["predict" + suffix] = H.compile(Graph.create("predict", [("p", p)]))
        e = D.map2(D.sub, D.matmul(D.param("m", F32, (r, z.width)), D.param("we", F32, (z.width, z.out))),
                   D.param("target", F32, (r, z.out)))
        loss = D.reduce(D.add, D.const(F32, 0.0),
                        D.flatten(D.map(lambda d: D.mul(D.mul(d, d), D.const(F32, 1.0 / (r * z.out))), e)))
        self.compiled["loss"] = H.compile(G.grad(Graph.create("loss", [("loss", loss)]), "loss", ["m", "we"]))

        self.first = O.NormBlock("f32", r, z.width, norm="none", pre="rms")
        self.delta = O.GatedDelta("f32", z.batch, z.tokens, z.heads, z.heads, z.key_dim, z.value_dim, states=False)
        self.block = O.NormBlock("f32", r, z.width, norm="rms", pre="rms", dropout=dropout)
        self.drop = O.Dropout("f32", r, z.width, dropout)
        self.first_one = O.NormBlock("f32", z.batch, z.width, norm="none", pre="rms")
        self.delta_one = O.GatedDelta("f32", z.batch, 1, z.heads, z.heads, z.key_dim, z.value_dim)
        self.block_one = O.NormBlock("f32", z.batch, z.width, norm="rms", pre="rms")

        g = np.random.default_rng(seed)
        kd, vd = z.heads * z.key_dim, z.heads * z.value_dim
        shapes = {"wq": (z.width, kd), "wk": (z.width, kd), "wv": (z.width, vd), "wg": (z.width, z.heads),
                  "wb": (z.width, z.heads), "wo": (vd, z.width), "we": (z.width, z.out), "first": (z.width,),
                  "post": (z.width,), "pre": (z.width,)}
        self.weights = {n: (np.ones(s) if len(s) == 1 else g.standard_normal(s) / np.sqrt(s[0])).astype(np.float32)
                        for n, s in shapes.items()}
        self._upload()

    def _upload(self):
        for r in getattr(self, "device", {}).values():
            H.free_resident(r)
        self.device = {n: H.upload(w) for n, w in self.weights.items()}

    def _graph(self, name, **inputs):
        return dict(H.run_resident(self.compiled[name], inputs))

    @staticmethod
    def _empty(*shape):
        return H.Resident(Buffer.alloc(4 * int(np.prod(shape))), F32, shape)

    def _view(self, r, rows, dim=None):
        """A [rows, heads (dim)] resident as [batch, tokens, heads(, dim)]."""
        z = self.z
        shape = (z.batch, rows // z.batch, z.heads) + (() if dim is None else (dim,))
        return O.Array(r.buf, "f32", shape)

    def _heads(self, p, rows):
        z = self.z
        return [self._view(p["q"], rows, z.key_dim), self._view(p["k"], rows, z.key_dim),
                self._view(p["v"], rows, z.value_dim), self._view(p["g"], rows), self._view(p["beta"], rows)]

    def step(self, x, target, seed, rate=0.1):
        """One training step on ``x`` [tokens, width] and ``target``; the loss."""
        z, r, w = self.z, self.z.rows(), self.device
        x, target = H.upload(x), H.upload(target)
        e = lambda *s: self._empty(*(s or (r, z.width)))  # noqa: E731
        h0, n0 = e(), e()
        self.first.forward(x, h0, n0, pre_weight=w["first"])
        p = self._graph("project", n=n0, **{k: w[k] for k in PROJECTIONS})
        heads = self._heads(p, r)
        o = e(r, z.heads * z.value_dim)
        saved = self.delta.saved()
        self.delta.forward(*heads, self._view(o, r, z.value_dim), saved=saved)
        y = self._graph("mix", o=o, wo=w["wo"])["y"]
        h, n1, m = e(), e(), e()
        params = dict(post_weight=w["post"], pre_weight=w["pre"])
        self.block.forward(y, h, n1, residual=x, seed=seed, **params)
        self.drop.forward(n1, m, seed=seed, offset=1)
        top = self._graph("loss", m=m, we=w["we"], target=target)

        grads = {n: self._empty(*self.weights[n].shape) for n in ("first", "post", "pre")}
        grads["we"] = top["dloss/dwe"]
        dn1, dh, dy = e(), H.upload(np.zeros((r, z.width), np.float32)), e()
        self.drop.backward(top["dloss/dm"], dn1, seed=seed, offset=1)
        self.block.backward(y, dh, dy, dn=dn1, h=h, seed=seed, grads=dict(post_weight=grads["post"], pre_weight=grads["pre"]),
                            **params)
        back = self._graph("mix_back", o=o, wo=w["wo"], dy=dy)
        grads["wo"] = back["ds/dwo"]
        d = {n: e(r, z.heads * s) for n, s in (("q", z.key_dim), ("k", z.key_dim), ("v", z.value_dim), ("g", 1), ("beta", 1))}
        self.delta.backward(*heads, self._view(back["ds/do"], r, z.value_dim), saved, *self._heads(d, r))
        back2 = self._graph("project_back", n=n0, **{k: w[k] for k in PROJECTIONS}, **{"d" + n: t for n, t in d.items()})
        grads.update({n: back2["ds/d" + n] for n in PROJECTIONS})
        dx = e()
        self.first.backward(x, dh, dx, dn=back2["ds/dn"], h=h0, grads=dict(pre_weight=grads["first"]), pre_weight=w["first"])

        loss = float(H.download(top["loss"]))
        for n, t in grads.items():
            self.weights[n] = (self.weights[n] - rate * H.download(t).reshape(self.weights[n].shape)).astype(np.float32)
        held = {id(t.buf): t.buf for t in [x, target, h0, n0, o, y, h, n1, m, dn1, dh, dy, dx, saved]
                + list(grads.values()) + list(d.values()) + list(p.values()) + list(top.values()) + list(back.values())
                + list(back2.values())}
        for b in held.values():
            b.free()
        self._upload()
        return loss

    def predict(self, x):
        """The outputs for ``x`` without dropout, a token at a time: what a
        server does, with one state a sequence and head."""
        z, w = self.z, self.device
        x = x.reshape(z.batch, z.tokens, z.width)
        e = lambda *s: self._empty(*(s or (z.batch, z.width)))  # noqa: E731
        state = H.upload(np.zeros((z.batch, z.heads, z.key_dim, z.value_dim), np.float32))
        out = np.empty((z.batch, z.tokens, z.out), np.float32)
        for t in range(z.tokens):
            xt = H.upload(np.ascontiguousarray(x[:, t]))
            h0, n0, o, h, n1 = e(), e(), e(z.batch, z.heads * z.value_dim), e(), e()
            self.first_one.forward(xt, h0, n0, pre_weight=w["first"])
            p = self._graph("project_one", n=n0, **{k: w[k] for k in PROJECTIONS})
            self.delta_one.forward(*self._heads(p, z.batch), self._view(o, z.batch, z.value_dim), state=state, state_out=state)
            y = self._graph("mix_one", o=o, wo=w["wo"])["y"]
            self.block_one.forward(y, h, n1, residual=xt, post_weight=w["post"], pre_weight=w["pre"])
            q = self._graph("predict_one", m=n1, we=w["we"])["p"]
            out[:, t] = H.download(q)
            for b in [xt, h0, n0, o, h, n1, y, q] + list(p.values()):
                b.buf.free()
        state.buf.free()
        return out.reshape(z.rows(), z.out)

    def evaluate(self, x):
        """The same outputs from one pass over whole sequences."""
        z, r, w = self.z, self.z.rows(), self.device
        x = H.upload(x)
        h0, n0, o, h, n1 = (self._empty(r, c) for c in (z.width, z.width, z.heads * z.value_dim, z.width, z.width))
        self.first.forward(x, h0, n0, pre_weight=w["first"])
        p = self._graph("project", n=n0, **{k: w[k] for k in PROJECTIONS})
        self.delta.forward(*self._heads(p, r), self._view(o, r, z.value_dim))
        y = self._graph("mix", o=o, wo=w["wo"])["y"]
        plain = O.NormBlock("f32", r, z.width, norm="rms", pre="rms")
        plain.forward(y, h, n1, residual=x, post_weight=w["post"], pre_weight=w["pre"])
        q = self._graph("predict", m=n1, we=w["we"])["p"]
        out = H.download(q)
        for b in [x, h0, n0, o, h, n1, y, q] + list(p.values()):
            b.buf.free()
        return out

    def release(self):
        for c in self.compiled.values():
            c.release()
        for op in (self.first, self.delta, self.block, self.drop, self.first_one, self.delta_one, self.block_one):
            op.free()
        for r in self.device.values():
            H.free_resident(r)
        self.device = {}


def recall_task(z, seed):
    """Inputs and targets of a task that needs a memory: the target at a token
    is the sum of the sequence's first columns so far, decayed."""
    g = np.random.default_rng(seed)
    x = g.standard_normal((z.batch, z.tokens, z.width)).astype(np.float32)
    target = np.zeros((z.batch, z.tokens, z.out), np.float32)
    run = np.zeros((z.batch, z.out), np.float32)
    for t in range(z.tokens):
        run = 0.7 * run + 0.5 * x[:, t, :z.out]
        target[:, t] = run
    return x.reshape(z.rows(), z.width), target.reshape(z.rows(), z.out)


def main(steps=20):
    z = Sizes()
    layer = Layer(z)
    x, target = recall_task(z, 1)
    for i in range(steps):
        loss = layer.step(x, target, seed=i)
        if i % 5 == 0 or i == steps - 1:
            print("step %2d loss %.4f" % (i, loss), flush=True)
    a, b = layer.predict(x), layer.evaluate(x)
    print("token by token against whole sequences: largest difference %.2g" % np.abs(a - b).max(), flush=True)
    layer.release()


if __name__ == "__main__":
    main()
