"""Gradients of gated units in fp16 whose inner gradients dG = D U act'(G) and dU = D act(G) leave the type's range though the results do not: against the formulas in 64 bits."""
import numpy as np
import pytest

from layers import CALC, TINY, UNIT, decode, encode
from test_gpu_gate import Unit, held, near
from test_gpu_gate_tails import value_and_slope

pytestmark = pytest.mark.gpu
T = "f16"
# blocks that split the sums, tiles, a batch in parts
SHAPES = [(40, 24, 30), (300, 100, 257), (20001, 20, 8)]


def kept(a):
    return decode(encode(a, T), T)


def unit(m, k, n, Y, Wg, Wu, D, seed=1, kind="silu", bias=False):
    """A unit of normal values times the given magnitudes (of Y and D: numbers, or an array over rows and columns)."""
    rng = np.random.default_rng(seed)
    u = Unit(m, k, n, T, seed, kind=kind, bias=bias)
    u.Y, u.D = kept(rng.standard_normal((m, k)) * Y), kept(rng.standard_normal((m, n)) * D)
    u.W = kept(np.concatenate([rng.standard_normal((n, k)) * Wg, rng.standard_normal((n, k)) * Wu]) * k ** -0.5)
    u.dY, u.dW, u.dD = held(u.Y, T, k), held(u.W, T, k), held(u.D, T, n)
    return u


def check(u, got):
    """As the gradients' other tests count roundings; what lies below the type's range between the products is off by half of its last place, which lies 2^39 below the bound
    of the row or column: 2-norms of the rows of Y and W, 1.13 for a derivative, at least 1 for a value."""
    c, e, n = CALC[T], UNIT[T], u.n
    g, p, dg, dp = u.projections()
    v, kv, s, ks = value_and_slope(g, u.kind)
    ds, dv = 1.1 * dg + c * ks, np.abs(s) * dg + 1.1 * dg * dg + c * kv
    D = np.abs(u.D)
    P = np.concatenate([u.D * p * s, u.D * v], 1)
    dP = np.concatenate([D * (np.abs(p) * ds + np.abs(s) * dp + dp * ds), D * dv], 1) + 3 * c * np.abs(P)
    y, w = np.linalg.norm(u.Y, axis=1)[:, None], np.linalg.norm(u.W, axis=1)[None, :]
    b = np.zeros(2 * n) if u.b is None else np.abs(u.b)
    most = np.concatenate([1.13 * D * (y * w[:, n:] + b[n:]), D * np.maximum(y * w[:, :n] + b[:n], 1)], 1)
    last = 1.01 * 2.0 ** -38 * most
    assert np.abs(P).max() > 65504 or np.median(np.abs(P[P != 0])) < 2.0 ** -22 or most.max() / most[most > 0].min() > 2.0 ** 20, "nothing leaves the range"

    def result(x, d, terms, mag):
        d = d + 2 * (terms + 2) * c * mag
        assert np.abs(x).max() < 65000 and np.median(np.abs(x)) > 0
        return x, d + e * (np.abs(x) + d) + TINY[T]
    rows = dP + e * (np.abs(P) + dP) + last.max(1)[:, None]
    cols = dP + e * (np.abs(P) + dP) + last.max(0)[None, :]
    near(got[0].get(), *result(P @ u.W, rows @ np.abs(u.W), 2 * n, (np.abs(P) + rows) @ np.abs(u.W)))
    near(got[1].get(), *result(P.T @ u.Y, cols.T @ np.abs(u.Y), u.m, (np.abs(P) + cols).T @ np.abs(u.Y)))


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("kind", ["silu", "gelu", "none"])
def test_beyond_the_range(cla, kind, m, k, n):
    """dG around 2^15 and up to 2^19, beside weights of 2^-14 and rows of 2^-10."""
    u = unit(m, k, n, 2.0 ** -10, 2.0 ** -14 * k ** 0.5, 2.0 ** 14, 2.0 ** 12, kind=kind)
    check(u, u.backward((True, True, False)))


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("a", [10, -10])
def test_below_the_range(cla, a, m, k, n):
    """dG around 2^-27: beside large weights the gradient of Y, beside large rows that of W is an ordinary number."""
    u = unit(m, k, n, 2.0 ** a, 2.0 ** -a, 2.0 ** (-8 - a), 2.0 ** -18)
    g, p, _, _ = u.projections()
    v, _, s, _ = value_and_slope(g, u.kind)
    P = u.D * p * s
    assert np.median(np.abs(P)) < 2.0 ** -25
    got = u.backward()
    check(u, got)
    big = got[0].get() if a < 0 else got[1].get()[:n]
    want = P @ u.W[:n] + (u.D * v) @ u.W[n:] if a < 0 else P.T @ u.Y
    assert np.linalg.norm(big - want) < 0.05 * np.linalg.norm(want)  # (2^-25 of 2^-17 or more; nothing of them was left where they vanished)


@pytest.mark.parametrize("m,k,n", SHAPES)
def test_rows_and_columns_of_unlike_magnitudes(cla, m, k, n):
    rng = np.random.default_rng(m)
    D = 2.0 ** rng.uniform(-16, 0, (m, 1)) * 2.0 ** rng.uniform(-8, 0, (1, n))
    u = unit(m, k, n, 2.0 ** rng.uniform(-6, 4, (m, 1)), 1.0, 1.0, D, bias=True)
    u.b = kept(np.random.default_rng(2).standard_normal(2 * n))
    from devmem import DevBuf
    u.dB = DevBuf.from_numpy(encode(u.b, T))
    check(u, u.backward((True, True, False)))


@pytest.mark.parametrize("m,k,n", SHAPES)
def test_rows_without_a_gradient_change_nothing(cla, m, k, n):
    """The largest values in rows of Y whose incoming gradient is 0: the gradient of W is that of zeros in their place, bit by bit."""
    u = unit(m, k, n, 1.0, 1.0, 1.0, 1.0)
    u.D[1::3], u.Y[1::3] = 0.0, 0.0
    u.dD, u.dY = held(u.D, T, n), held(u.Y, T, k)
    clean = [o.get() for o in u.backward()]
    u.Y[1::3] = 65504.0 * np.sign(np.random.default_rng(3).standard_normal(u.Y[1::3].shape))
    u.dY = held(u.Y, T, k)
    for a, b in zip(clean, [o.get() for o in u.backward()]):
        assert np.array_equal(a, b)


def test_gradients_beyond_the_type_are_infinite(cla):
    """What does not fit the result is infinite there, and there alone."""
    u = unit(40, 24, 30, 1.0, 1.0, 1.0, 1.0)
    u.D[5] = 60000.0
    u.dD = held(u.D, T, u.n)
    g = [o.get() for o in u.backward()]
    ref = unit(40, 24, 30, 1.0, 1.0, 1.0, 1.0)
    want = [o.get() for o in ref.backward()]
    assert not np.isfinite(g[0][5]).all() and not np.isnan(g[0]).any()
    rest = np.arange(40) != 5
    assert np.array_equal(g[0][rest], want[0][rest])


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("kind", ["relu", "sigmoid"])
def test_gates_shut_by_their_bias(cla, kind, m, k, n):
    """Gates whose bias is -infinity give nothing; the others' gradients, dG up to 2^19, are what they are without them: each side rounds every dG and dU by half a step or by half of the last
    place 2^39 below its row's or column's bound, and the result by half a step."""
    from devmem import DevBuf
    u = unit(m, k, n, 2.0 ** -10, 2.0 ** -14 * k ** 0.5, 2.0 ** 14 if kind == "relu" else 2.0 ** -4, 2.0 ** 12 if m < 1000 else 2.0 ** 11, kind=kind, bias=True)
    u.b = np.zeros(2 * n)
    u.b[n:] = 40.0 if kind == "relu" else 120.0
    shut = np.arange(n) % 3 == 1
    u.D[:, shut] = 0.0
    u.dD, u.dB = held(u.D, T, n), DevBuf.from_numpy(encode(u.b, T))
    clean = [o.get() for o in u.backward((True, True, False))[:2]]
    g, p, _, _ = u.projections()
    v, _, s, _ = value_and_slope(g, kind)
    P = np.abs(np.concatenate([u.D * p * s, u.D * v], 1))
    assert P.max() > 2 * 65504
    u.D[:, shut] = 30000.0
    u.b[:n][shut] = -np.inf
    u.dD, u.dB = held(u.D, T, n), DevBuf.from_numpy(encode(u.b, T))
    got = [o.get() for o in u.backward((True, True, False))[:2]]
    y, w = np.linalg.norm(u.Y, axis=1)[:, None], np.linalg.norm(u.W, axis=1)[None, :]
    most = np.abs(u.D) * np.maximum(1.13 * (y * w[:, n:] + u.b[n:]), y * w[:, :n] + 1)
    last = 2.0 ** -38 * most
    rows, cols = P * 2.0 ** -11 + last.max(1)[:, None], P * 2.0 ** -11 + last.max(0).repeat(2).reshape(n, 2).T.reshape(-1)[None, :]
    for x, c, off in ((got[0], clean[0], rows @ np.abs(u.W)), (got[1], clean[1], cols.T @ np.abs(u.Y))):
        assert np.isfinite(c).all() and np.median(np.abs(c)) > 0
        near(x, c, 2.1 * (off + 2.0 ** -11 * np.abs(c) + TINY[T]))
    assert not got[1][:n][shut].any() and not got[1][n:][shut].any()
