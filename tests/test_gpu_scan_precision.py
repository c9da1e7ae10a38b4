"""Float prefix sums over many small tiles are as close as few roundings can
be: the error of whole scans of positive values against that of rounding the
exact sums once."""

import numpy as np
import pytest

from cudacaml_amd import backend_hip as H
from cudacaml_amd import dsl as D
from cudacaml_amd.ir import F32, F64, Graph

pytestmark = pytest.mark.gpu


# Chains of up to 256 tiles round a prefix where it is published, where it is
# read and where it joins an element: sqrt(3) roundings. The bound of 2^25
# doubles is above what a running sum of long doubles is itself off there; the
# exact sums are further down.
@pytest.mark.parametrize("dtype,shape,seeds,most", [(F32, (900_001,), 24, 1.75), (F64, (900_001,), 24, 1.75),
                                                    (F32, (30, 60_000), 8, 1.75), (F64, (1 << 25,), 5, 4.5)], ids=str)
def test_error_of_sums(device, dtype, shape, seeds, most):
    wide = np.float64 if dtype is F32 else np.longdouble
    x = D.param("x", dtype, shape)
    c = H.compile(Graph.create("s", [("p", (D.scan if len(shape) == 1 else D.scan_rows)(D.add, D.const(dtype, 0), x))]))
    err = once = 0.0
    try:
        for seed in range(seeds):
            v = np.random.default_rng(seed).random(shape).astype(dtype.np)
            e = np.cumsum(v.astype(wide), axis=-1)
            got = dict(H.run(c, [("x", v)]))["p"]
            err += float(((got - e) ** 2).sum() / (e ** 2).sum())
            once += float(((e.astype(dtype.np) - e) ** 2).sum() / (e ** 2).sum())
    finally:
        c.release()
    assert np.sqrt(err / once) <= most


@pytest.mark.parametrize("dtype", [F32, F64], ids=lambda d: d.name)
@pytest.mark.parametrize("n", [300_000, 3_000_000])
def test_zeros_infinities_and_nan(device, dtype, n):
    """A sum that overflows stays infinite, infinities of both signs give NaN
    from there on, and -0 stays -0 from an initial -0."""
    def scan(init, v):
        c = H.compile(Graph.create("s", [("p", D.scan(D.add, D.const(dtype, init), D.param("x", dtype, (n,))))]))
        try:
            return dict(H.run(c, [("x", v)]))["p"]
        finally:
            c.release()

    v = np.full(n, -0.0, dtype.np)
    assert np.signbit(scan(-0.0, v)).all()
    assert not np.signbit(scan(0.0, v)).any()
    v = np.ones(n, dtype.np)
    v[n // 3] = np.inf
    got = scan(0, v)
    np.testing.assert_array_equal(got[: n // 3], np.arange(1, n // 3 + 1))
    assert (got[n // 3:] == np.inf).all()
    v[n // 2] = -np.inf
    got = scan(0, v)
    assert (got[n // 3:n // 2] == np.inf).all() and np.isnan(got[n // 2:]).all()
    big = np.finfo(dtype.np).max
    v = np.zeros(n, dtype.np)
    v[[5, n // 2]] = big
    got = scan(0, v)
    assert (got[5:n // 2] == big).all() and (got[n // 2:] == np.inf).all()


# A prefix of a long chain is carried to 70 bits and more, whatever look-backs
# it came through: it is rounded where it is read and where it joins an
# element, sqrt(2) roundings, and the tiles' own totals add less than a fifth
# of one. The exact sums come from the values' two halves as integers, as a
# running sum of 2^25 long doubles is three roundings off itself.
@pytest.mark.parametrize("n,seeds", [(1 << 25, 3), (25_000_001, 2)])
def test_long_chains_of_doubles_round_prefixes_once(device, n, seeds):
    c = H.compile(Graph.create("s", [("p", D.scan(D.add, D.const(F64, 0), D.param("x", F64, (n,))))]))
    try:
        for seed in range(seeds):
            v = np.random.default_rng(100 + seed).random(n)
            high = np.floor(v * 2.0 ** 26)
            low = (v * 2.0 ** 26 - high) * 2.0 ** 27
            e = (np.cumsum(high.astype(np.int64)).astype(np.longdouble) * 2.0 ** 27 +
                 np.cumsum(low.astype(np.int64)).astype(np.longdouble)) * 2.0 ** -53
            once = float(((e.astype(np.float64) - e) ** 2).sum())
            for _ in range(2):
                got = dict(H.run(c, [("x", v)]))["p"]
                assert np.sqrt(float(((got - e) ** 2).sum()) / once) <= 1.75
    finally:
        c.release()


def test_infinities_nan_and_zeros_of_long_chains(device):
    """As above, through the chain of a row too long for two passes."""
    n = 21_000_000
    c = H.compile(Graph.create("s", [("p", D.scan(D.add, D.const(F64, -0.0), D.param("x", F64, (n,))))]))
    scan = lambda v: dict(H.run(c, [("x", v)]))["p"]  # noqa: E731
    try:
        assert np.signbit(scan(np.full(n, -0.0))).all()
        v = np.ones(n)
        v[n // 3] = np.inf
        got = scan(v)
        np.testing.assert_array_equal(got[: n // 3], np.arange(1, n // 3 + 1))
        assert (got[n // 3:] == np.inf).all()
        v[n // 2] = -np.inf
        got = scan(v)
        assert (got[n // 3:n // 2] == np.inf).all() and np.isnan(got[n // 2:]).all()
        big = np.finfo(np.float64).max
        v = np.zeros(n)
        v[[5, n // 2]] = big
        got = scan(v)
        assert (got[5:n // 2] == big).all() and (got[n // 2:] == np.inf).all()
        v = np.full(n, 5e-324)  # sums of the smallest number are exact
        np.testing.assert_array_equal(scan(v), np.arange(1, n + 1) * 5e-324)
    finally:
        c.release()
