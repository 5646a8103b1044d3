"""8-bit products whose scales' product leaves fp32's range though the result does not."""
import numpy as np
import pytest

from devmem import DevBuf, hip
from layers import BYTES, CALC, TINY, TYPE_IDS, UNIT, decode, encode, quantise

pytestmark = pytest.mark.gpu
# rows that a product quantises itself, rows streamed past the weights, tiles (and their largest shape)
SHAPES = [(3, 2000, 40), (20, 2000, 100), (700, 2000, 700), (2100, 130, 4096)]


def run(cla, Y, W, scales, t, bias=None, gate=None):
    m, n = Y.shape[0], W.shape[1] // (2 if gate else 1)
    h = cla.ClaQ8(*W.shape).set_values(W, scales)
    dY, dO, ws = DevBuf.from_numpy(encode(Y, t)), DevBuf(m * n * BYTES[t]), DevBuf(h.workspace(m))
    dB = None if bias is None else DevBuf.from_numpy(encode(bias, t))
    b = None if bias is None else dB.ptr
    if gate:
        h.gate_dev_async(cla.ACTIVATIONS[gate], dY.ptr, TYPE_IDS[t], m, Y.shape[1], b, dO.ptr, n, ws.ptr, ws.nbytes)
    else:
        h.lmm_dev_async(dY.ptr, TYPE_IDS[t], m, Y.shape[1], b, dO.ptr, n, ws.ptr, ws.nbytes)
    assert hip().hipDeviceSynchronize() == 0
    return decode(dO.to_numpy((m, n), encode(np.zeros(0), t).dtype), t)


def exact(Y, W, scales):
    q, s = quantise(Y)
    return (q.astype(np.float64) @ W.astype(np.float64)) * s.astype(np.float64)[:, None] * scales.astype(np.float64)  # (whole numbers below 2^53)


@pytest.mark.parametrize("gate", [None, "sigmoid"])
@pytest.mark.parametrize("t", ["f64", "f32", "bf16"])
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_small_scales(cla, t, m, k, n, gate):
    """Scales of rows around 2^-75, of columns around 2^-65, sums beyond 2^19: each result off by the roundings of two products and its own."""
    rng = np.random.default_rng(k + n)
    Y = decode(encode((0.25 + rng.random((m, k))) * 2.0 ** -68, t), t)
    W = rng.integers(64, 128, (k, n)).astype(np.int8)
    scales = ((0.5 + rng.random(n)) * 2.0 ** -65).astype(np.float32)
    want = exact(Y, W, scales)
    if gate:  # (the gate's sums are next to 0)
        want = 0.5 * want[:, n // 2:]
    off = np.abs(run(cla, Y, W, scales, t, gate=gate) - want)
    assert np.abs(want).min() > 2.0 ** -125
    assert np.all(off <= (5 * CALC[t] + 1.01 * UNIT[t]) * np.abs(want) + (2.0 ** -100 if t == "f64" else TINY[t]) * (gate == "sigmoid") * np.abs(want) + TINY[t])


@pytest.mark.parametrize("t", ["f64", "f32", "bf16"])
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_large_scales(cla, t, m, k, n):
    """Scales of rows and columns around 2^100: sums of 0 give the bias; others leave fp32 with their sign, and are numbers in fp64."""
    rng = np.random.default_rng(k)
    Y = decode(encode(rng.standard_normal((m, k)) * 2.0 ** 106, t), t)
    W = rng.integers(-127, 128, (k, n)).astype(np.int8)
    W[:, ::3] = 0
    scales = ((0.5 + rng.random(n)) * 2.0 ** 100).astype(np.float32)
    bias = decode(encode(rng.standard_normal(n), t), t)
    got = run(cla, Y, W, scales, t, bias=bias)
    assert np.array_equal(got[:, ::3], np.tile(bias[::3], (m, 1)))
    want = exact(Y, W, scales)
    if t == "f64":
        assert np.all(np.abs(got - (want + bias)) <= 5 * CALC[t] * (np.abs(want) + np.abs(bias)))
    else:
        there = np.abs(want) > 1e39
        assert there.sum() > 0.6 * want.size and np.array_equal(got[there], np.where(want[there] > 0, np.inf, -np.inf))


@pytest.mark.parametrize("m,k,n", SHAPES)
def test_a_zero_scale_and_one_that_is_not_finite(cla, m, k, n):
    rng = np.random.default_rng(k)
    Y = decode(encode(rng.standard_normal((m, k)), "f32"), "f32")
    Y[1] = 0.0
    W = rng.integers(-127, 128, (k, n)).astype(np.int8)
    scales = (0.5 + rng.random(n)).astype(np.float32)
    scales[2], scales[5] = 0.0, np.nan
    got, rest = run(cla, Y, W, scales, "f32"), np.arange(n) != 5
    want = exact(Y, W[:, rest], scales[rest])
    assert np.isnan(got[:, 5]).all() and not got[1, rest].any() and not got[:, 2].any()
    assert np.all(np.abs(got[:, rest] - want) <= 5 * CALC["f32"] * np.abs(want))
