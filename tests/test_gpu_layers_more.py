"""Layers' products in the types and at the addresses that their first tests leave out, with those tests' tolerances."""
import numpy as np
import pytest

from devmem import DevBuf, hip
from layers import BYTES, TYPE_IDS, decode, encode
from test_gpu_gate import KINDS, TYPES, Shifted, Unit, held
from test_gpu_q8 import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m", [5, 130, 1100])
def test_activations_of_gated_units_in_fp16(cla, kind, m):
    u = Unit(m, 48, 40 if m < 1000 else 300, "f16", m, kind=kind)
    u.W *= 4.0
    u.dW = held(u.W, "f16", u.k)
    u.check_forward(u.forward().get())
    u.check_backward(u.backward())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("m,n", [(5, 96), (70, 96), (700, 1400)])
def test_activations_of_8_bit_gated_units(cla, kind, t, m, n):
    c = Case(cla, m, 100, n, t, seed=m, gated=True)
    c.call(kind)
    c.check(c.result(), kind)


class Behind:
    """An output one element behind an aligned address, sentinels around it; what Unit's checks take for an output."""

    def __init__(self, rows, cols, t):
        self.rows, self.cols, self.t = rows, cols, t
        self.buf = DevBuf((rows * cols + 1) * BYTES[t] + 64)
        assert hip().hipMemset(self.buf.ptr, 0x5A, self.buf.nbytes) == 0
        self.ptr = self.buf.ptr + BYTES[t]

    def get(self):
        b = BYTES[self.t]
        raw = self.buf.to_numpy(self.buf.nbytes, np.uint8)
        end = (self.rows * self.cols + 1) * b
        assert np.all(raw[:b] == 0x5A) and np.all(raw[end:] == 0x5A), "bytes around an output were written"
        return decode(raw[b:end].copy().view(encode(np.zeros(0), self.t).dtype).reshape(self.rows, self.cols), self.t)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,k,n", [(3, 96, 40), (90, 97, 33), (700, 96, 200), (3001, 20, 9)])
def test_gradients_at_odd_places(cla, t, m, k, n):
    u = Unit(m, k, n, t, m)
    for name in ("dY", "dW", "dD", "dB"):
        setattr(u, name, Shifted(getattr(u, name), t))
    outs = Behind(m, k, t), Behind(2 * n, k, t), Behind(1, 2 * n, t)
    need = cla.gate_workspace(TYPE_IDS[t], m, k, n, True)
    ws = DevBuf(need)
    cla.gate_backward_dev_async(*u.args(), u.dD.ptr, n, outs[0].ptr, k, outs[1].ptr, k, outs[2].ptr, ws.ptr, need)
    assert hip().hipDeviceSynchronize() == 0
    u.check_backward(outs)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m", [2, 30, 700])
def test_8_bit_products_at_odd_places(cla, t, m):
    """Rows, bias and output one element behind an aligned address."""
    c = Case(cla, m, 90, 700, t, seed=m)
    c.dY, c.dB = Shifted(c.dY, t), Shifted(c.dB, t)
    out = Behind(m, 700, t)
    c.h.lmm_dev_async(c.dY.ptr, TYPE_IDS[t], m, 90, c.dB.ptr, out.ptr, 700, c.dW.ptr, c.bytes)
    assert hip().hipDeviceSynchronize() == 0
    c.check(out.get())
