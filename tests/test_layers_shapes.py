"""Shapes that the host forms of the layers' products refuse before the library reads or writes an array (in whose place a recorder stands)."""
import ctypes as C

import numpy as np
import pytest


class Recorder:
    """Stands for the library: takes every call, keeps its arguments."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def f(*a):
            self.calls.append((name, a))
            return 1 << 20 if name == "cla_q8_create" else 0
        return f


@pytest.fixture
def rec(monkeypatch):
    from systemds_amd import capi
    r = Recorder()
    monkeypatch.setattr(capi, "load_library", lambda: r)
    monkeypatch.setattr(capi, "_initialised", True)
    return r


def refused(match, f, *a, **k):
    from systemds_amd import capi
    with pytest.raises(capi.ClaError, match=match) as e:
        f(*a, **k)
    assert e.value.code == capi.ERR_INVALID


def values(p, n):
    return np.ctypeslib.as_array(C.cast(p, C.POINTER(C.c_double)), (n,)).copy()


def test_gate(rec):
    from systemds_amd import capi
    Y, W, D = np.arange(33 * 7.0).reshape(33, 7), np.ones((10, 7)), np.ones((33, 5))
    for f, more in ((capi.gate, ()), (capi.gate_backward, (D,))):
        refused("W", f, "silu", Y, np.ones((11, 7)), *more)       # an odd number of rows: whose last one belongs to no projection
        refused("W", f, "silu", Y, np.ones(70), *more)
        refused("W", f, "silu", Y, np.ones((0, 7)), *more)
        refused("Y", f, "silu", np.ones((7, 33)), W, *more)       # whole rows if it were flat
        refused("Y", f, "silu", np.ones(33 * 7 - 1), W, *more)
        refused("bias", f, "silu", Y, W, *more, bias=np.ones(9))
        refused("activation", f, "swish", Y, W, *more)
    for grad in (np.ones((10, 5)), np.ones((34, 5)), np.ones((33, 4)), np.ones((5, 33)), np.ones(10 * 5)):
        refused("grad", capi.gate_backward, "silu", Y, W, grad)
    assert rec.calls == []
    capi.gate("silu", Y, W, np.ones((1, 10)))
    capi.gate(capi.ACTIVATIONS["silu"], Y.ravel(), W)
    capi.gate_backward("silu", Y, W, D.ravel())
    capi.gate_backward("silu", np.asfortranarray(Y), W[:, ::-1], np.zeros((33, 10))[:, ::2])
    for name, a in rec.calls:
        assert a[0] == 1 and a[2] == 33 and a[3] == 7 and a[6] == 5 and np.array_equal(values(a[1], 33 * 7), Y.ravel())
    assert capi.gate("silu", np.zeros((0, 7)), W)[0].shape == (0, 5)


def test_8_bit_matrix(rec):
    from systemds_amd import capi
    h = capi.ClaQ8(7, 10)
    rec.calls.clear()
    refused("W", h.set, np.ones((10, 7)))                         # transposed: as many values
    refused("W", h.set, np.ones(69))
    refused("values", h.set_values, np.ones((10, 7), np.int8), np.ones(10))
    refused("8-bit whole numbers", h.set_values, np.full((7, 10), 200), np.ones(10))
    refused("8-bit whole numbers", h.set_values, np.full((7, 10), 0.5), np.ones(10))
    refused("scales", h.set_values, np.ones((7, 10), np.int8), np.ones(9))
    for f in (h.lmm, lambda *a, **k: h.gate("silu", *a, **k)):
        refused("Y", f, np.ones((7, 4)))
        refused("Y", f, np.ones(20))
        refused("bias", f, np.ones((4, 7)), bias=np.ones(7))
    refused("activation", h.gate, "swish", np.ones((4, 7)))
    assert rec.calls == []
    h.set(np.ones((7, 10)))
    h.set(np.ones(70))
    h.set_values(np.full((7, 10), -128), np.ones((10, 1)))
    assert h.lmm(np.ones(14), np.ones(10))[0].shape == (2, 10) and h.gate(1, np.ones((3, 7)))[0].shape == (3, 5)
    assert [n for n, _ in rec.calls] == ["cla_q8_set", "cla_q8_set", "cla_q8_set_values", "cla_q8_lmm", "cla_q8_gate"]
    h.h = None


def test_chain_of_a_block(rec):
    """The multiply chain's vectors are as long as the block's columns and rows."""
    from systemds_amd import capi
    blk = object.__new__(capi.ClaBlock)
    blk.lib, blk.h, blk.n_rows, blk.n_cols = rec, None, 9, 4
    refused("mmchain", blk.mmchain, np.ones(3))
    refused("mmchain", blk.mmchain, np.ones(5), np.ones(9), 1)
    for ctype in (1, 2):
        refused("mmchain", blk.mmchain, np.ones(4), np.ones(8), ctype)
    assert rec.calls == []
    blk.mmchain(np.ones((4, 1)))
    blk.mmchain(np.ones(4), np.ones((9, 1)), 1)
    assert [n for n, _ in rec.calls] == ["cla_mmchain", "cla_mmchain"]
