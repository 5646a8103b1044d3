"""Gated units act(Y t(Wg) + bg) * (Y t(Wu) + bu) and their gradients against the formulas in 64 bits, with tolerances that count every rounding
between (a sum of n terms: 2 (n + 2) half steps of the computing type of the sum of the terms' magnitudes), and against differences."""
import numpy as np
import pytest

from devmem import DevBuf, hip
from layers import BYTES, CALC, TINY, TYPE_IDS, UNIT, act, decode, encode, gated_bound

pytestmark = pytest.mark.gpu
TYPES = ["f64", "f32", "bf16", "f16"]
KINDS = ["sigmoid", "silu", "gelu", "gelu_tanh", "relu", "none"]


def sync():
    assert hip().hipDeviceSynchronize() == 0


class Out:
    """A device output with sentinels behind its rows and its end."""

    def __init__(self, rows, cols, ld, t):
        self.rows, self.cols, self.ld, self.t = rows, cols, ld, t
        self.buf = DevBuf(max(rows * ld * BYTES[t], 1) + 64)
        assert hip().hipMemset(self.buf.ptr, 0x5A, self.buf.nbytes) == 0
        sync()

    def get(self):
        sync()
        raw = self.buf.to_numpy(self.buf.nbytes, np.uint8)
        n = self.rows * self.ld * BYTES[self.t]
        assert np.all(raw[n:] == 0x5A), "bytes behind an output were written"
        o = raw[:n].view(encode(np.zeros(0), self.t).dtype).reshape(self.rows, self.ld)
        assert np.all(np.ascontiguousarray(o[:, self.cols:]).view(np.uint8) == 0x5A), "values behind a row were written"
        return decode(np.ascontiguousarray(o[:, :self.cols]), self.t)


def held(a, t, ld):
    host = np.zeros((a.shape[0], ld), encode(a[:0, :0], t).dtype)
    host[:, :a.shape[1]] = encode(a, t)
    return DevBuf.from_numpy(host)


class Unit:
    def __init__(self, m, k, n, t, seed, kind="silu", bias=True, apart=0):
        rng = np.random.default_rng(seed)
        self.m, self.k, self.n, self.t, self.kind, self.apart = m, k, n, t, kind, apart

        def values(*shape, by=1.0):
            return decode(encode(rng.standard_normal(shape) * by, t), t)
        self.Y, self.W, self.D = values(m, k), values(2 * n, k, by=k ** -0.5), values(m, n)
        if m > 4:
            self.Y[m - 2] = 0.0
        self.b = values(2 * n, by=0.3) if bias else None
        self.dY, self.dW, self.dD = held(self.Y, t, k + apart), held(self.W, t, k + apart), held(self.D, t, n + apart)
        self.dB = None if self.b is None else DevBuf.from_numpy(encode(self.b, t))

    def args(self):
        from systemds_amd import capi
        return (capi.ACTIVATIONS[self.kind], TYPE_IDS[self.t], self.dY.ptr, self.m, self.k, self.k + self.apart, self.dW.ptr, self.k + self.apart,
                None if self.dB is None else self.dB.ptr, self.n)

    def forward(self, stream=None, out=None):
        from systemds_amd import capi
        out = out or Out(self.m, self.n, self.n + self.apart, self.t)
        capi.gate_dev_async(*self.args(), out.buf.ptr, self.n + self.apart, stream=stream)
        return out

    def outs(self):
        a = self.apart
        return Out(self.m, self.k, self.k + a, self.t), Out(2 * self.n, self.k, self.k + a, self.t), Out(1, 2 * self.n, 2 * self.n, self.t)

    def backward(self, which=(True, True, True), stream=None, outs=None, ws=None):
        from systemds_amd import capi
        a = self.apart
        outs = outs or self.outs()
        need = capi.gate_workspace(TYPE_IDS[self.t], self.m, self.k, self.n, True)
        self.ws = ws or DevBuf(need + 64)
        assert hip().hipMemset(self.ws.ptr, 0xFF, need + 64) == 0  # (NaN in every type)
        sync()
        p = [o.buf.ptr if w else None for o, w in zip(outs, which)]
        capi.gate_backward_dev_async(*self.args(), self.dD.ptr, self.n + a, p[0], self.k + a, p[1], self.k + a, p[2], self.ws.ptr, need, stream)
        sync()
        assert np.all(self.ws.to_numpy(need + 64, np.uint8)[need:] == 0xFF), "bytes behind the workspace were written"
        return outs

    def projections(self):
        """(G, U) and how far the kernel's may be off."""
        c = CALC[self.t]
        x, mag = self.Y @ self.W.T, np.abs(self.Y) @ np.abs(self.W.T)
        d = 2 * (self.k + 2) * c * mag
        if self.b is not None:
            x = x + self.b
            d = d + c * (np.abs(x) + d)
        n = self.n
        return x[:, :n], x[:, n:], d[:, :n], d[:, n:]

    def check_forward(self, got):
        g, u, dg, du = self.projections()
        v, _ = act(g, self.kind)
        near(got, v * u, gated_bound(g, u, dg, du, self.kind, self.t))

    def check_backward(self, got, which=(True, True, True)):
        t, c, e = self.t, CALC[self.t], UNIT[self.t]
        g, u, dg, du = self.projections()
        v, s = act(g, self.kind)
        # slopes: second derivatives are at most 1.1, the formula's own roundings 16 (1 + |g| + |g|^3) half steps (1 - tanh^2 loses 12, times up to
        # 0.4 |g| + 0.054 |g|^3); next to the corner of max(x, 0) either slope
        ds = 1.1 * dg + 16 * c * (1 + np.abs(g) + np.abs(g) ** 3)
        if self.kind == "relu":
            ds = np.where(np.abs(g) <= dg, 1.0, 0.0)
        dv = np.abs(s) * dg + 1.1 * dg * dg + 16 * c * (1 + np.abs(g))
        D = np.abs(self.D)
        P = np.concatenate([self.D * u * s, self.D * v], 1)
        dP = np.concatenate([D * (np.abs(u) * ds + np.abs(s) * du + du * ds), D * dv], 1) + 3 * c * np.abs(P)
        dR = dP + e * (np.abs(P) + dP) + TINY[t]                       # rounded to the type between the products
        aP, aW, aY = np.abs(P) + dR, np.abs(self.W), np.abs(self.Y)

        def result(x, d, terms, mag):
            d = d + 2 * (terms + 2) * c * mag
            return x, d + e * (np.abs(x) + d) + TINY[t]
        if which[0]:
            near(got[0].get(), *result(P @ self.W, dR @ aW, 2 * self.n, aP @ aW))
        if which[1]:
            near(got[1].get(), *result(P.T @ self.Y, dR.T @ aY, self.m, aP.T @ aY))
        if which[2]:
            x, b = result(P.sum(0), dP.sum(0), self.m, (np.abs(P) + dP).sum(0))
            near(got[2].get()[0], x, b)
        for o, w in zip(got, which):
            if not w:
                assert np.all(o.buf.to_numpy(o.buf.nbytes, np.uint8) == 0x5A)


def near(got, want, bound):
    assert np.isfinite(got).all()
    off = np.abs(got - want)
    at = np.unravel_index(np.argmax(off - bound), off.shape)
    assert np.all(off <= bound), (at, got[at], want[at], off[at], bound[at])


# few rows (weights streamed), tiles of every shape, edges of all of them; values a row not whole 16 bytes
SHAPES = [(1, 1, 1), (1, 64, 16), (2, 100, 17), (16, 130, 33), (17, 301, 40), (40, 64, 64), (64, 65, 130), (65, 64, 1), (66, 200, 100), (129, 17, 65), (200, 1000, 129),
          (1000, 127, 70), (257, 512, 300)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_forward(cla, t, m, k, n):
    u = Unit(m, k, n, t, m + k + n, bias=(m + n) % 2 == 0)
    u.check_forward(u.forward().get())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (1, 64, 16), (3, 7, 5), (16, 130, 33), (64, 65, 130), (100, 64, 3), (257, 200, 100), (1000, 33, 70), (2000, 40, 24), (700, 300, 257)])
def test_backward(cla, t, m, k, n):
    u = Unit(m, k, n, t, m + k + n, bias=m % 2 == 0)
    u.check_backward(u.backward())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("t", ["f64", "f32", "bf16"])
def test_activations(cla, kind, t):
    for m in (5, 130):
        u = Unit(m, 48, 40, t, m, kind=kind)
        u.W *= 4.0
        u.dW = held(u.W, t, u.k)
        u.check_forward(u.forward().get())
        u.check_backward(u.backward())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m", [3, 90, 300])
def test_rows_apart(cla, t, m):
    u = Unit(m, 90, 35, t, m, apart=3)
    u.check_forward(u.forward().get())
    u.check_backward(u.backward())


class Shifted:
    """A copy of a device buffer that begins one element behind an aligned address."""

    def __init__(self, buf, t):
        raw = np.concatenate([np.zeros(BYTES[t], np.uint8), buf.to_numpy(buf.nbytes, np.uint8)])
        self.buf = DevBuf.from_numpy(raw)
        self.ptr = self.buf.ptr + BYTES[t]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m", [3, 90, 700])
def test_operands_at_odd_places(cla, t, m):
    """Operands, biases and the incoming gradient one element behind an aligned address; outputs, too."""
    u = Unit(m, 96, 40, t, m)
    for name in ("dY", "dW", "dD", "dB"):
        setattr(u, name, Shifted(getattr(u, name), t))
    u.check_forward(u.forward().get())
    u.check_backward(u.backward())
    from systemds_amd import capi
    want = u.forward().get()
    odd = DevBuf(m * 40 * BYTES[t] + 64)
    capi.gate_dev_async(*u.args(), odd.ptr + BYTES[t], 40)
    sync()
    raw = odd.to_numpy(odd.nbytes, np.uint8)[BYTES[t]:BYTES[t] * (1 + m * 40)].copy()
    assert np.array_equal(decode(raw.view(encode(np.zeros(0), t).dtype).reshape(m, 40), t), want)


@pytest.mark.parametrize("t", TYPES)
def test_two_streams_at_once(cla, t):
    """The gradients of two units queued on two streams, each with a workspace of its own, several times over."""
    import ctypes as C
    from systemds_amd import capi
    lib, streams, units = hip(), [C.c_void_p(), C.c_void_p()], []
    for i, s in enumerate(streams):
        assert lib.hipStreamCreate(C.byref(s)) == 0
        u = Unit(900, 130, 70, t, i + 1)
        u.got = u.backward()  # (allocates)
        units.append(u)
    need = capi.gate_workspace(TYPE_IDS[t], 900, 130, 70, True)
    for _ in range(6):
        for u, s in zip(units, streams):
            o = u.got
            capi.gate_backward_dev_async(*u.args(), u.dD.ptr, 70, o[0].buf.ptr, 130, o[1].buf.ptr, 130, o[2].buf.ptr, u.ws.ptr, need, s.value)
    sync()
    for u, s in zip(units, streams):
        u.check_backward(u.got)
        assert lib.hipStreamDestroy(s) == 0


@pytest.mark.parametrize("t,m,k,n", [("bf16", 2100, 256, 2048), ("f16", 4100, 136, 1100), ("f64", 2050, 70, 2049), ("f32", 2050, 72, 2050)])
def test_large_tiles(cla, t, m, k, n):
    u = Unit(m, k, n, t, 3)
    u.check_forward(u.forward().get())
    u.check_backward(u.backward())


@pytest.mark.parametrize("t", TYPES)
def test_many_rows_into_few_weights(cla, t):
    """The sums over the batch in parts, whose last one is short."""
    u = Unit(20001, 20, 8, t, 5)
    a, b = u.backward(), u.backward()
    u.check_backward(a)
    for x, y in zip(a, b):
        assert np.array_equal(x.get(), y.get())  # bit by bit


@pytest.mark.parametrize("which", [(True, False, False), (False, True, False), (False, False, True), (True, False, True)])
@pytest.mark.parametrize("m", [9, 1500])
def test_gradients_that_are_not_wanted(cla, which, m):
    u = Unit(m, 40, 24, "bf16", m)
    u.check_backward(u.backward(which), which)


@pytest.mark.parametrize("kind", ["sigmoid", "silu", "gelu", "gelu_tanh", "none"])
def test_gradients_against_differences(cla, kind):
    """sum(out * D) at 2^-14 to either side of a direction, in fp64: off by the third derivative (h^2 / 6 of a third derivative along a direction of norm 1, below
    40 here with |D|, |U| and the inner derivatives around 1 each over m n = 210 outputs) and the sums' roundings over 2 h."""
    rng = np.random.default_rng(2)
    m, k, n, h = 21, 12, 10, 2.0 ** -14
    Y, W, b, D = rng.standard_normal((m, k)), rng.standard_normal((2 * n, k)) * k ** -0.5, 0.3 * rng.standard_normal(2 * n), rng.standard_normal((m, n))
    grads = cla.gate_backward(kind, Y, W, D, b)

    def loss(y, w, c):
        return float(np.sum(cla.gate(kind, y, w, c)[0] * D))
    for i, x in enumerate((Y, W, b)):
        for _ in range(3):
            v = rng.standard_normal(x.shape)
            v /= np.linalg.norm(v)
            at = [[Y, W, b], [Y, W, b]]
            at[0][i], at[1][i] = x + h * v, x - h * v
            diff = (loss(*at[0]) - loss(*at[1])) / (2 * h)
            assert abs(diff - float(np.sum(grads[i] * v))) <= h * h / 6 * 40 + 2.0 ** -50 * m * n * 8 / h


def test_host_forms(cla):
    rng = np.random.default_rng(3)
    Y, W = rng.standard_normal((33, 7)), rng.standard_normal((10, 7))
    Y[3] = 0.0
    out, nnz = cla.gate("relu", Y, W)
    x = Y @ W.T
    assert np.allclose(out, np.maximum(x[:, :5], 0) * x[:, 5:], rtol=0, atol=1e-13) and nnz == np.count_nonzero(out) < 165
    out, nnz = cla.gate("silu", np.zeros((0, 7)), W)
    assert out.shape == (0, 5) and nnz == 0
    gy, gw, gb = cla.gate_backward("silu", np.zeros((0, 7)), W, np.zeros((0, 5)))
    assert gy.shape == (0, 7) and not gw.any() and not gb.any()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m", [5, 100])
def test_values_that_are_not_finite_stay_in_their_rows(cla, t, m):
    u = Unit(m, 50, 20, t, 1)
    clean, grads = u.forward().get(), [o.get() for o in u.backward()]
    u.Y[2, 7] = np.nan
    u.dY = held(u.Y, t, u.k)
    got = u.forward().get()
    rest = np.arange(m) != 2
    assert np.isnan(got[2]).all() and np.array_equal(got[rest], clean[rest])
    back = [o.get() for o in u.backward()]
    assert np.isnan(back[0][2]).all() and np.array_equal(back[0][rest], grads[0][rest])
    assert np.isnan(back[1]).all() and np.isnan(back[2]).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,n", [(5, 20), (100, 20), (1030, 1100), (2100, 2050)])
def test_row_ends_inside_16_bytes(cla, t, m, n):
    """What lies behind a row (the next row's first values, infinities and NaN here) stays out of its sums, in Y and in W, on every shape of tile and for every end."""
    for k in (2 + 64, 3 + 64, 6 + 64, 31) if m < 1000 else (70,):
        u = Unit(m, k, n, t, 1)
        clean = u.forward().get()
        u.Y[1::7, 0] = np.inf
        u.W[3::50, 0] = np.nan
        u.dY, u.dW = held(u.Y, t, k), held(u.W, t, k)
        got = u.forward().get()
        rows, cols = np.ones(m, bool), np.ones(n, bool)
        rows[1::7] = False
        bad = np.arange(3, 2 * n, 50)
        cols[bad % n] = False
        assert np.array_equal(got[np.ix_(rows, cols)], clean[np.ix_(rows, cols)])
        assert np.isnan(got[:, ~cols]).all()


def test_infinite_bias_beyond_the_batch(cla):
    """Rows that round the batch up are zeros in the sums whatever the bias is."""
    u = Unit(67, 24, 9, "bf16", 1)
    u.b[3] = np.inf
    u.dB = DevBuf.from_numpy(encode(u.b, "bf16"))
    gw = u.backward()[1].get()
    assert np.isfinite(gw[[0, 1, 2, 4, 5]]).all()


def test_captured_and_replayed(cla):
    """Forward and backward captured on a stream of their own, replayed on new values, with eager calls of the same unit in another workspace between."""
    import ctypes as C
    lib = hip()
    stream, graph, run = C.c_void_p(), C.c_void_p(), C.c_void_p()
    assert lib.hipStreamCreate(C.byref(stream)) == 0
    for m, t in ((3, "bf16"), (1300, "f32")):
        u, other = Unit(m, 72, 40, t, m), Unit(m, 72, 40, t, m + 1)
        out, outs = u.forward(), u.backward()  # (allocates)
        ws = u.ws
        from systemds_amd import capi
        need = capi.gate_workspace(TYPE_IDS[t], m, 72, 40, True)
        assert lib.hipStreamBeginCapture(stream, 0) == 0
        u.forward(stream.value, out)
        capi.gate_backward_dev_async(*u.args(), u.dD.ptr, 40, outs[0].buf.ptr, 72, outs[1].buf.ptr, 72, outs[2].buf.ptr, ws.ptr, need, stream.value)
        assert lib.hipStreamEndCapture(stream, C.byref(graph)) == 0
        assert lib.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0)) == 0
        for turn in range(4):
            u.Y = decode(encode(np.random.default_rng(turn).standard_normal((m, 72)), t), t)
            new = encode(u.Y, t)
            assert lib.hipMemcpy(C.c_void_p(u.dY.ptr), new.ctypes.data_as(C.c_void_p), C.c_size_t(new.nbytes), 1) == 0
            for o in (out, *outs):
                assert lib.hipMemset(o.buf.ptr, 0x5A, o.buf.nbytes) == 0
            sync()
            assert lib.hipGraphLaunch(run, stream) == 0
            other.check_forward(other.forward().get())
            other.check_backward(other.backward())
            sync()
            u.check_forward(out.get())
            u.check_backward(outs)
        assert lib.hipGraphExecDestroy(run) == 0 and lib.hipGraphDestroy(graph) == 0
    assert lib.hipStreamDestroy(stream) == 0


@pytest.mark.parametrize("m", [2, 150])
def test_a_block_of_layers(cla, m):
    """A feed-forward block in 8 bits as a program runs it: rows quantised, gated unit, its output quantised, product; against the same steps in 64 bits on the values
    that each step was given, and the 16-bit unit beside it within what 8 bits lose (a row's values are off by s / 2 at most)."""
    rng = np.random.default_rng(m)
    k, n, t = 96, 80, "bf16"
    u = Unit(m, k, n, t, m, bias=False)
    down = rng.standard_normal((n, k)) * n ** -0.5
    hu, hd = cla.ClaQ8(k, 2 * n).set(u.W.T), cla.ClaQ8(n, k).set(down)
    ws = DevBuf(max(hu.workspace(m), hd.workspace(m)))
    mid, out = Out(m, n, n, t), Out(m, k, k, t)
    null = cla.TYPES[t]
    for h in (hu, hd):
        h.set_stream(None)
    hu.gate_dev_async(1, u.dY.ptr, null, m, k, None, mid.buf.ptr, n, ws.ptr, ws.nbytes)
    hd.lmm_dev_async(mid.buf.ptr, null, m, n, None, out.buf.ptr, k, ws.ptr, ws.nbytes)
    sixteen = u.forward().get()
    from layers import quantise
    x, w = mid.get(), None
    q, s = quantise(x)
    v, c = hd.get()
    p = (q.astype(np.int64) @ v.astype(np.int64)) * s.astype(np.float64)[:, None] * c.astype(np.float64)
    near(out.get(), p, 2.0 ** -7.9 * np.abs(p) + 1e-30)
    # the unit itself: projections off by what rounding of either side to 8 bits loses
    q, s = quantise(u.Y)
    v, c = hu.get()
    dy, dw = s.astype(np.float64)[:, None] / 2, c.astype(np.float64)[None, :] / 2
    lost = dy * np.abs(u.W.T).sum(0)[None, :] + np.abs(u.Y).sum(1)[:, None] * dw + k * dy * dw
    g, up, dg, du = u.projections()
    near(x, sixteen, 2 * gated_bound(g, up, dg + lost[:, :n], du + lost[:, n:], "silu", t))


def test_refusals_of_workspaces(cla):
    u = Unit(70, 24, 9, "f32", 1)
    from systemds_amd import capi
    need = capi.gate_workspace(1, 70, 24, 9, True)
    o = u.outs()
    ws = DevBuf(need)

    def call(p, n):
        capi.gate_backward_dev_async(*u.args(), u.dD.ptr, 9, o[0].buf.ptr, 24, o[1].buf.ptr, 24, o[2].buf.ptr, p, n)
    for p, n in ((None, need), (ws.ptr, need - 1), (ws.ptr + 8, need)):
        with pytest.raises(capi.ClaError, match="workspace of") as e:
            call(p, n)
        assert e.value.code == capi.ERR_INVALID
    call(ws.ptr, need)
    sync()
