"""The activations of gated units and their derivatives where they are small: what an output may be off by is counted relative to the value itself (or, where a derivative is
a sum of two terms, to their magnitudes), so that a form which loses its digits to a difference is seen."""
import numpy as np
import pytest
from scipy.special import erfc, expit

from devmem import DevBuf, hip
from layers import BYTES, CALC, TINY, TYPE_IDS, UNIT, decode, encode

pytestmark = pytest.mark.gpu
KINDS = ["sigmoid", "silu", "gelu", "gelu_tanh", "relu", "none"]
LEAST = {"f64": 2.0 ** -1000, "f32": 2.0 ** -110, "bf16": 2.0 ** -110, "f16": 2.0 ** -110}  # below: intermediates are zero or have lost digits at the end of the range


def value_and_slope(x, kind):
    """(value, its error in half steps of the computing type, derivative, its error) in 64 bits. A value carries 40 half steps of its own (exp, erfc: at most 16 units of the last
    place; 1 / x, sums, products) and what its argument is off by (a: how many half steps, relative, twice that for this oracle's own) times the argument times the function's logarithmic derivative."""
    with np.errstate(all="ignore"):
        zero = np.zeros_like(x)

        def off(terms):  # (magnitude, half steps of the argument, argument's weight)
            return sum(np.nan_to_num(np.abs(m)) * (40 + np.nan_to_num(a * w, nan=0.0, posinf=0.0)) for m, a, w in terms)
        if kind in ("sigmoid", "silu"):
            l, m = expit(x), expit(-x)
            if kind == "sigmoid":
                return l, off([(l, 4, np.abs(x) * m)]), l * m, off([(l * m, 4, np.abs(x))])
            return x * l, off([(x * l, 4, np.abs(x) * m)]), l + x * l * m, off([(l, 4, np.abs(x) * m), (x * l * m, 4, np.abs(x))])
        if kind == "gelu":
            p, d = 0.5 * erfc(-x / np.sqrt(2)), np.exp(-x * x / 2) / np.sqrt(2 * np.pi)
            xd = np.where(d > 0, x * d, 0.0)
            return x * p, off([(x * p, 4, np.where(p > 0, np.abs(x) * d / p, 0.0))]), p + xd, off([(p, 4, np.where(p > 0, np.abs(x) * d / p, 0.0)), (xd, 4, x * x)])
        if kind == "gelu_tanh":
            c = 2 * np.sqrt(2 / np.pi)
            t = c * (x + 0.044715 * x ** 3)
            l, m = expit(t), expit(-t)
            w = np.where(l * m > 0, x * l * m * c * (1 + 0.134145 * x * x), 0.0)
            return x * l, off([(x * l, 20, np.abs(t) * m)]), l + w, off([(l, 20, np.abs(t) * m), (w, 20, np.abs(t))])
        if kind == "relu":
            return np.maximum(x, 0), zero, (x > 0).astype(float), zero
        return x, zero, np.ones_like(x), zero


def points(t):
    far = {"f64": [1e100, 1e200], "f32": [1e20, 3e38], "bf16": [1e20, 3e38], "f16": [65504.0]}[t]
    x = np.concatenate([np.linspace(-13, 20, 331), np.linspace(-1.4, -0.6, 41), [0.0, -0.0, 30.0, -30.0, 100.0, -100.0], far, [-v for v in far]])
    return decode(encode(x, t), t)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("t", ["f64", "f32", "bf16", "f16"])
@pytest.mark.parametrize("n", [1, 2048])
def test_relative_errors(cla, t, kind, n):
    """Rows (x, 1) and weights (1, 0), (0, 1): the gate is x, the other projection 1, exactly. n outputs alike, on blocks that split the sums and on tiles; an incoming
    gradient of 1 in one of them leaves derivative and value as the gradient of Y."""
    x = points(t)
    m = x.size
    Y = np.stack([x, np.ones(m)], 1)
    W = np.concatenate([np.tile([1.0, 0.0], (n, 1)), np.tile([0.0, 1.0], (n, 1))])
    D = np.zeros((m, n))
    D[:, n // 3] = 1.0
    dY, dW, dD = (DevBuf.from_numpy(encode(a, t)) for a in (Y, W, D))
    dO, dG = DevBuf(m * n * BYTES[t]), DevBuf(m * 2 * BYTES[t])
    need = cla.gate_workspace(TYPE_IDS[t], m, 2, n, True)
    ws = DevBuf(need)
    args = (cla.ACTIVATIONS[kind], TYPE_IDS[t], dY.ptr, m, 2, 2, dW.ptr, 2, None, n)
    cla.gate_dev_async(*args, dO.ptr, n)
    cla.gate_backward_dev_async(*args, dD.ptr, n, dG.ptr, 2, None, 2, None, ws.ptr, need)
    assert hip().hipDeviceSynchronize() == 0
    kept = encode(np.zeros(0), t).dtype
    out, grad = decode(dO.to_numpy((m, n), kept), t), decode(dG.to_numpy((m, 2), kept), t)
    v, kv, s, ks = value_and_slope(x, kind)

    def near(got, want, k, roundings):
        d = CALC[t] * k + LEAST[t] * (1 + np.abs(x) * (np.abs(x) < 1e3))
        bound = d + roundings * UNIT[t] * 1.01 * (np.abs(want) + d) + TINY[t]
        off = np.abs(got - want)
        at = int(np.argmax(np.where(np.isnan(off), np.inf, off - bound)))
        assert np.all(off <= bound), (x[at], got[at], want[at], bound[at])
    near(out[:, 0], v, kv, 1)
    assert np.array_equal(out, np.repeat(out[:, :1], n, 1))
    near(grad[:, 1], v, kv, 1)  # (rounded to the type once: the second time there is nothing left to round)
    near(grad[:, 0], s, ks, 1)
