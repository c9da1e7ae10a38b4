"""What attention, the norm of its heads and the embedding refuse of arrays that
lie in one another, against every address, without a device."""

import numpy as np
import pytest

from cudacaml_amd import _lib
from cudacaml_amd import operators as O

DIM, SIZE, BASE = 4, 4, 1 << 20


def _places(at, counts, steps):
    """The first places, in elements, of all heads of an array."""
    i = np.indices(counts).reshape(3, -1)
    return at + (i * np.array(steps)[:, None]).sum(0)


def _meet(x, y):
    return bool((np.abs(x[:, None] - y[None, :]) < DIM).any())


def _steps(g, counts):
    """Distances along the axes in an order of their own, with something between
    neighbours or not, and of any sign but the tokens'."""
    steps, reach = [0, 0, 0], DIM
    for axis in g.permutation(3):
        steps[axis] = int(reach + g.choice([0, 0, 3, DIM, 2 * DIM]))
        reach += steps[axis] * (max(counts[axis], 2) - 1)
        if axis != 1 and g.random() < 0.2:
            steps[axis] *= -1
    return steps, reach


def _heads(at, steps):
    return (BASE + at * SIZE, *steps)


def _far(at):
    return (at << 24, 1 << 16, 1 << 10, 1 << 6)


@pytest.mark.parametrize("seed", range(4))
def test_attention_refuses_results_within_inputs_wherever_they_meet(seed):
    """o moved along q by any distance, with q's steps: refused if a head of one
    lies in a head of the other, and not otherwise; of two results too."""
    g = np.random.default_rng(seed)
    L, seen = _lib.lib(), [0, 0]
    for _ in range(400):
        b, t, hk, group = (int(x) for x in g.integers(1, 5, 4))
        h = hk * group
        counts = (b, t, h)
        steps, reach = _steps(g, counts)
        desc = _lib.AttentionDesc(0, b, t, 0, 0, h, hk, DIM, 1.0)
        # about as far as the array reaches, mostly by whole steps and a little
        by = int(sum(int(g.integers(-n, n + 1)) * s for n, s in zip(counts, steps)) + g.integers(-DIM, DIM + 1)) if g.random() < 0.8 else int(
            g.integers(-reach, reach))
        at = 4 * reach
        io = O.Attention._forward_io.pack(*_heads(at, steps), *_far(2), *_far(3), *_heads(at + by, steps), 0, 0, 4098)
        rc, msg = L.cchip_attention_forward(desc, io, None, 0, None), _lib.lib().cchip_last_error().decode()
        met = _meet(_places(at, counts, steps), _places(at + by, counts, steps))
        assert rc == 1 and ("o is written over q" if met else "saved is not aligned") in msg, (counts, steps, by, msg)
        seen[met] += 1
        # dk beside dq: fewer heads, with the same steps
        back = [*_far(2), *_far(3), *_far(4), *_far(5), *_far(6), *_heads(at, steps), *_heads(at + by, steps), *_far(7)]
        rc, msg = L.cchip_attention_backward(desc, O.Attention._backward_io.pack(*back, 0, 0, 4098), None, 0, None), _lib.lib().cchip_last_error().decode()
        met = _meet(_places(at, counts, steps), _places(at + by, (b, t, hk), steps))
        assert rc == 1 and ("dq and dk are written to one place" if met else "saved is not aligned") in msg, (counts, hk, steps, by, msg)
    assert min(seen) > 50


@pytest.mark.parametrize("seed", range(2))
def test_head_norm_refuses_results_within_inputs_wherever_they_meet(seed):
    """All but the very place."""
    g = np.random.default_rng(10 + seed)
    L = _lib.lib()
    none = (0, 0, 0, 0)
    for _ in range(300):
        b, t, h, hk = (int(x) for x in g.integers(1, 5, 4))
        counts = (b, t, h)
        steps, reach = _steps(g, counts)
        desc = _lib.HeadNormDesc(0, 0, b, t, 0, h, hk, DIM, DIM, 0, 1, 1e-6)
        by = int(sum(int(g.integers(-n, n + 1)) * s for n, s in zip(counts, steps)) + (g.integers(-DIM, DIM + 1) if g.random() < 0.5 else 0))
        at = 4 * reach
        # the sum of a weight's gradient has no workspace, which is refused last
        back = [*_heads(at, steps), *_far(2), *none, *none, *none, *none, *none, *_far(3), *_far(4), *_heads(at + by, steps), *_far(5),
                0, 4096, 0, 0, 4096, 0]
        rc, msg = L.cchip_head_norm_backward(desc, O.HeadNorm._io.pack(*back), None, 0, None), _lib.lib().cchip_last_error().decode()
        met = _meet(_places(at, counts, steps), _places(at + by, counts, steps))
        assert rc == 1 and ("dq is written over q" if met else "workspace needs") in msg, (counts, steps, by, msg)
        back[0:4], back[28:32] = _far(3), _heads(at, steps)  # the gradient, which dq may take the place of
        rc, msg = L.cchip_head_norm_backward(desc, O.HeadNorm._io.pack(*back), None, 0, None), _lib.lib().cchip_last_error().decode()
        assert rc == 1 and ("not head for head" if met and by else "workspace needs") in msg, (counts, steps, by, msg)


def test_attention_refuses_tensors_in_its_workspace():
    L = _lib.lib()
    t = lambda p, h=4: (p << 24, 100 * 8 * h, 8 * h, 8)  # noqa: E731
    desc = _lib.AttentionDesc(0, 2, 100, 0, 0, 4, 2, 8, 1.0)
    back = [*t(1), *t(2, 2), *t(3, 2), *t(4), *t(5), *t(6), *t(7, 2), *t(8, 2)]
    need = O.Attention("f32", 2, 100, 4, 2, 8).workspace_bytes(backward=True)
    assert need < 1 << 24  # the first address that a tensor has
    for at in range(8):
        io = O.Attention._backward_io.pack(*back, 0, 0, 1 << 28)
        rc, msg = L.cchip_attention_backward(desc, io, ((at + 1) << 24) - need + 16, need, None), L.cchip_last_error().decode()
        assert rc == 1 and "lies in the workspace" in msg
    cache = _lib.AttentionDesc(0, 2, 1, 0, 4096, 4, 2, 8, 1.0)
    need = O.Attention("f32", 2, 1, 4, 2, 8, keys=4096).workspace_bytes()
    words = [*t(1), 2 << 24, 1 << 16, 16, 8, 3 << 24, 1 << 16, 16, 8, *t(4)]
    for p in (1 << 24, 2 << 24, 3 << 24, 4 << 24):
        io = O.Attention._forward_io.pack(*words, 0, 4096, 0)
        rc, msg = L.cchip_attention_forward(cache, io, p - need + 16, need, None), L.cchip_last_error().decode()
        assert need > 0 and rc == 1 and "lies in the workspace" in msg
    for p in (1, 2, 3, 4):  # and `saved`, which a forward call writes
        rc, msg = L.cchip_attention_forward(desc, O.Attention._forward_io.pack(*back[:16], 0, 0, p << 24), None, 0, None), L.cchip_last_error().decode()
        assert rc == 1 and "what the forward pass saves" in msg


@pytest.mark.parametrize("seed", range(2))
def test_embedding_refuses_rows_within_its_table(seed):
    g = np.random.default_rng(20 + seed)
    L, seen = _lib.lib(), [0, 0]
    for _ in range(300):
        vocab, tokens = (int(x) for x in g.integers(1, 9, 2))
        step, by = int(DIM + g.choice([0, 0, 2, DIM, 9])), int(g.integers(-120, 120))
        desc = _lib.EmbeddingDesc(0, 0, tokens, vocab, DIM, 1.0)
        met = _meet(_places(0, (1, vocab, 1), (0, step, 0)), _places(by, (1, tokens, 1), (0, step, 0)))
        table, rows = BASE, BASE + by * SIZE
        seen[met] += 1
        if not met:  # taken, which only a device can show
            continue
        for fn, words in ((L.cchip_embedding_forward, [4096, table, step, rows, step, 0, 0, 0, 0, 0]),
                          (L.cchip_embedding_backward, [4096, 0, 0, 0, 0, rows, step, table, step, 0])):
            rc = fn(desc, O.Embedding._io.pack(*words), *((None,) if fn is L.cchip_embedding_forward else (None, 0, None)))
            assert rc == 1 and "is written over" in L.cchip_last_error().decode(), (vocab, tokens, step, by)
    assert min(seen) > 30
