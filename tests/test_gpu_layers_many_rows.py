"""Layers' products of more rows than one launch takes (blocks times threads are below 2^32), and widths at their limits."""
import ctypes as C

import numpy as np
import pytest

from devmem import DevBuf, hip

pytestmark = pytest.mark.gpu
LAUNCH = (1 << 32) - 1


def fill(nbytes, byte):
    b = DevBuf(nbytes)
    assert hip().hipMemset(b.ptr, byte, nbytes) == 0
    return b


def write(b, at, a):
    assert hip().hipMemcpy(b.ptr + at, a.ctypes.data_as(C.c_void_p), a.nbytes, 1) == 0


def read(b, at, n, dtype):
    out = np.empty(n, dtype)
    assert hip().hipMemcpy(out.ctypes.data_as(C.c_void_p), b.ptr + at, out.nbytes, 2) == 0
    return out


def sync():
    assert hip().hipDeviceSynchronize() == 0


def test_rows_to_8_bits(cla):
    """2^28 + 37 rows of one value, 16 rows to a block."""
    m, split = (1 << 28) + 37, LAUNCH // 256 * 16
    assert split < m
    dY, dQ, dS = fill(2 * m, 0x40), fill(m + 64, 99), fill(4 * m, 0)  # (bf16 0x4040: 3)
    other = [0, split - 1, split, m - 1]
    for i, at in enumerate(other):
        write(dY, 2 * at, np.array([0xC000 + 16 * i], np.uint16))
    cla.quantize_rows_dev_async(dY.ptr, 2, m, 1, 1, dQ.ptr, 1, dS.ptr)
    sync()
    q, s = dQ.to_numpy(m + 64, np.int8), dS.to_numpy(m, np.float32)
    top = np.full(m, 3.0, np.float32)
    sign = np.full(m, 127, np.int8)
    for i, at in enumerate(other):
        top[at], sign[at] = -np.array([(0xC000 + 16 * i) << 16], np.uint32).view(np.float32)[0], -127
    assert np.all(q[m:] == 99) and np.array_equal(q[:m], sign) and np.array_equal(s, top * (np.float32(1) / np.float32(127)))


def test_product_of_8_bit_rows(cla):
    """The most rows that a call takes, into one column: three launches."""
    m, k = (1 << 31) - 1, 16
    split = LAUNCH // 256 * 64
    dQ, dS, dO = fill(m * k, 1), fill(4 * m, 0x3C), fill(2 * m + 64, 0x5A)
    for at in (0, split - 1, split, 2 * split, m - 1):
        write(dQ, at * k, np.full(k, 5, np.int8))
    h = cla.ClaQ8(k, 1).set_values(np.ones((k, 1)), np.ones(1))
    h.lmm_quantized_dev_async(dQ.ptr, k, dS.ptr, m, None, dO.ptr, 3, 1)
    sync()
    s = np.full(4, 0x3C, np.uint8).view(np.float32)[0]
    for a, b, five in ((0, 1000, 0), (split - 500, split + 500, 499), (split - 500, split + 500, 500), (2 * split - 64, m, 64), (2 * split - 64, m, m - 1 - 2 * split + 64)):
        got = read(dO, 2 * a, b - a, np.float16)
        want = np.full(b - a, np.float16(16 * s))
        for at in (0, split - 1, split, 2 * split, m - 1):
            if a <= at < b:
                want[at - a] = np.float16(80 * s)
        assert np.array_equal(got, want) and got[five] == np.float16(80 * s)
    assert np.all(read(dO, 2 * m, 64, np.uint8) == 0x5A)


def test_gated_unit(cla):
    m = (1 << 30) + 5
    split = LAUNCH // 256 * 64
    dY, dO = fill(8 * m, 0x40), fill(8 * m + 64, 0x5A)
    x = np.full(8, 0x40, np.uint8).view(np.float64)[0]
    other = [0, split - 1, split, m - 1]
    for at in other:
        write(dY, 8 * at, np.array([3.0]))
    dW = DevBuf.from_numpy(np.array([[0.5], [2.0]]))
    cla.gate_dev_async(cla.ACTIVATIONS["none"], 0, dY.ptr, m, 1, 1, dW.ptr, 1, None, 1, dO.ptr, 1)
    sync()
    for a, b in ((0, 1000), (split - 500, split + 5), (m - 5, m)):
        got = read(dO, 8 * a, b - a, np.float64)
        want = np.full(b - a, 0.5 * x * (2 * x))
        for at in other:
            if a <= at < b:
                want[at - a] = 9.0
        assert np.allclose(got, want, rtol=2.0 ** -51, atol=0)
    assert np.all(read(dO, 8 * m, 64, np.uint8) == 0x5A)


@pytest.mark.parametrize("t", [0, 1, 2, 3])
def test_gradients_of_too_many_rows_are_refused(cla, t):
    """... in front of the first launch (the pointers are a small buffer's)."""
    m = 1 << 30
    b, need = DevBuf(1024), cla.gate_workspace(t, m, 1, 1, True)
    with pytest.raises(cla.ClaError, match="fewer rows") as e:
        cla.gate_backward_dev_async(1, t, b.ptr, m, 1, 1, b.ptr, 1, None, 1, b.ptr, 1, None, 1, b.ptr, 1, None, b.ptr, need)
    assert e.value.code == cla.ERR_UNSUPPORTED
    sync()


def test_most_columns_of_an_8_bit_matrix(cla):
    k, n = 3, 1 << 21
    rng = np.random.default_rng(1)
    W = rng.standard_normal((k, n))
    h = cla.ClaQ8(k, n).set(W)
    v, s = h.get()
    scale = np.abs(W).max(0).astype(np.float32) * (np.float32(1) / np.float32(127))
    assert np.array_equal(s, scale) and np.array_equal(v, np.clip(np.rint(W / scale.astype(np.float64)), -127, 127).astype(np.int8))
    Y = rng.standard_normal((20, k))
    out, _ = h.lmm(Y)
    r = np.abs(Y).max(1).astype(np.float32) * (np.float32(1) / np.float32(127))
    q = np.clip(np.rint(Y / r.astype(np.float64)[:, None]), -127, 127)
    assert np.allclose(out, (q @ v.astype(float)) * r.astype(np.float64)[:, None] * s.astype(np.float64), rtol=4e-16, atol=0)
