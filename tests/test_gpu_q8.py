"""8-bit matrices: rows quantised, products with a scale for each row and column, gated units, against the definition in 64 bits (sums of whole numbers
are exact in both; what is left are the roundings of scales, biases and outputs, counted below)."""
import numpy as np
import pytest

from devmem import DevBuf, hip
from layers import BYTES, CALC, TINY, TYPE_IDS, UNIT, act, decode, encode, gated_bound, quantise

pytestmark = pytest.mark.gpu
TYPES = ["f64", "f32", "bf16", "f16"]


def sync():
    assert hip().hipDeviceSynchronize() == 0


def rows_of(rng, m, k, t):
    Y = decode(encode(rng.standard_normal((m, k)) * np.where(rng.random(k) < 0.05, 12.0, 1.0), t), t)
    if m > 3:
        Y[m - 2] = 0.0
        Y[1, :] *= 2.0 ** -10
    return Y


def run_quantise(cla, Y, t, ld=None, ldq=None, off=0):
    m, k = Y.shape
    ld, ldq = ld or k, ldq or k
    host = np.full((m, ld), 0, encode(Y[:0, :0], t).dtype)
    host[:, :k] = encode(Y, t)
    buf = np.concatenate([np.zeros(off, host.dtype), host.reshape(-1)])
    dY, dQ, dS = DevBuf.from_numpy(buf), DevBuf.from_numpy(np.full(m * ldq + 64, 99, np.int8)), DevBuf(4 * m)
    cla.quantize_rows_dev_async(dY.ptr + off * BYTES[t], TYPE_IDS[t], m, k, ld, dQ.ptr, ldq, dS.ptr)
    sync()
    q = dQ.to_numpy(m * ldq + 64, np.int8)
    assert np.all(q[m * ldq:] == 99)
    q = q[:m * ldq].reshape(m, ldq)
    assert np.all(q[:, k:] == 99), "bytes behind a row were written"
    return q[:, :k], dS.to_numpy(m, np.float32)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,k", [(1, 1), (3, 7), (5, 8), (9, 100), (4, 2047), (2, 2049), (3, 8192), (2, 8200), (2, 20001), (300, 33)])
def test_rows_to_8_bits(cla, t, m, k):
    rng = np.random.default_rng(m * 31 + k)
    Y = rows_of(rng, m, k, t)
    q, s = run_quantise(cla, Y, t)
    want, scale = quantise(Y)
    assert np.array_equal(s, scale) and np.array_equal(q, want)
    q2, s2 = run_quantise(cla, Y, t, ld=k + 3, ldq=k + 5, off=1)  # rows and bytes at odd places
    assert np.array_equal(s2, scale) and np.array_equal(q2, want)


@pytest.mark.parametrize("t", TYPES)
def test_quotients_next_to_a_half(cla, t):
    """Rows whose values lie on and next to whole numbers and halves of the scale, at scales over the type's range."""
    rng = np.random.default_rng(5)
    lo, hi = {"f64": (-300, 120), "f32": (-140, 120), "bf16": (-125, 120), "f16": (-12, 9)}[t]
    Y = np.empty((257, 509))
    for i in range(257):
        e = rng.integers(lo, hi)
        top = decode(encode(np.array([(1 + rng.random()) * 2.0 ** e]), t), t)[0]
        step = float(np.float32(top) * (np.float32(1) / np.float32(127))) if top < 3e38 else top / 127
        x = (rng.integers(-254, 255, 509) / 2.0) * step * (1 + rng.integers(-2, 3, 509) * 2.0 ** -24)
        x[0] = top
        Y[i] = np.clip(decode(encode(x, t), t), -top, top)
    want, scale = quantise(Y)
    q, s = run_quantise(cla, Y, t)
    assert np.array_equal(s, scale)
    assert np.array_equal(q, want)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("k", [5, 3000])
def test_rows_that_are_not_finite(cla, t, k):
    rng = np.random.default_rng(k)
    Y = rows_of(rng, 6, k, t)
    Y[0, k - 1], Y[2, 0], Y[3, k // 2] = np.nan, np.inf, -np.inf
    q, s = run_quantise(cla, Y, t)
    want, scale = quantise(Y)
    assert np.array_equal(np.isnan(s), [True, False, True, True, False, False])
    assert np.array_equal(s[[1, 4, 5]], scale[[1, 4, 5]])
    assert np.all(q[[0, 2, 3]] == 0) and np.array_equal(q[[1, 4, 5]], want[[1, 4, 5]])


class Case:
    """A matrix, rows and what the product may be off by."""

    def __init__(self, cla, m, k, n, t, seed, bias=True, gated=False, ld_out=None, ld_y=None):
        rng = np.random.default_rng(seed)
        self.m, self.k, self.n, self.t, self.gated = m, k, n, t, gated
        self.nout = n // 2 if gated else n
        self.ld = ld_out or self.nout
        self.ldy = ld_y or k
        self.W = rng.integers(-128, 128, (k, n)).astype(np.int8)
        self.ws = (0.01 * (0.5 + rng.random(n)) / np.sqrt(k)).astype(np.float32)
        self.Y = rows_of(rng, m, k, t)
        self.b = decode(encode(rng.standard_normal(n), t), t) if bias else None
        self.h = cla.ClaQ8(k, n).set_values(self.W, self.ws)
        host = np.zeros((m, self.ldy), encode(self.Y[:0, :0], t).dtype)
        host[:, :k] = encode(self.Y, t)
        self.dY = DevBuf.from_numpy(host)
        self.dB = None if self.b is None else DevBuf.from_numpy(encode(self.b, t))
        self.dO = DevBuf(m * self.ld * BYTES[t] + 64)
        self.clear()
        self.bytes = self.h.workspace(m)
        self.dW = DevBuf(self.bytes)

    def clear(self):
        n = self.dO.nbytes
        assert hip().hipMemset(self.dO.ptr, 0x5A, n) == 0
        sync()

    def call(self, kind="silu"):
        b = None if self.dB is None else self.dB.ptr
        if self.gated:
            from systemds_amd import capi
            self.h.gate_dev_async(capi.ACTIVATIONS[kind], self.dY.ptr, TYPE_IDS[self.t], self.m, self.ldy, b, self.dO.ptr, self.ld, self.dW.ptr, self.bytes)
        else:
            self.h.lmm_dev_async(self.dY.ptr, TYPE_IDS[self.t], self.m, self.ldy, b, self.dO.ptr, self.ld, self.dW.ptr, self.bytes)

    def result(self):
        sync()
        raw = self.dO.to_numpy(self.dO.nbytes, np.uint8)
        assert np.all(raw[self.m * self.ld * BYTES[self.t]:] == 0x5A), "bytes behind the output were written"
        o = raw[:self.m * self.ld * BYTES[self.t]].view(encode(np.zeros(0), self.t).dtype).reshape(self.m, self.ld)
        assert np.all(o[:, self.nout:].view(np.uint8) == 0x5A), "values behind a row were written"
        return decode(np.ascontiguousarray(o[:, :self.nout]), self.t)

    def check(self, got, kind="silu"):
        """sums: rounded to the computing type, times (scale * scale), plus bias: four roundings (each relative to what it rounds), then the type's own."""
        t, c = self.t, CALC[self.t]
        q, s = quantise(self.Y)
        p = (q.astype(np.int64) @ self.W.astype(np.int64)).astype(np.float64) * s.astype(np.float64)[:, None] * self.ws.astype(np.float64)
        x = p if self.b is None else p + self.b
        d = 3.01 * c * np.abs(p) + c * np.abs(x)
        if self.gated:
            g, u, h = x[:, :self.nout], x[:, self.nout:], self.nout
            v, _ = act(g, kind)
            x, bound = v * u, gated_bound(g, u, d[:, :h], d[:, h:], kind, t)
        else:
            bound = d + UNIT[t] * (np.abs(x) + d) + TINY[t]
        assert np.isfinite(got).all()
        off = np.abs(got - x)
        worst = np.unravel_index(np.argmax(off - bound), off.shape)
        assert np.all(off <= bound), (worst, got[worst], x[worst], off[worst], bound[worst])


# few rows (weights streamed), tiles of every shape, edges of all of them
SHAPES = [(1, 1, 1), (1, 64, 16), (2, 100, 17), (16, 128, 33), (17, 300, 40), (33, 129, 64), (64, 65, 130), (65, 64, 1), (66, 200, 100), (129, 16, 129),
          (200, 1000, 257), (1000, 127, 100), (257, 2000, 515)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_product(cla, t, m, k, n):
    c = Case(cla, m, k, n, t, seed=m + k + n, bias=(m + n) % 2 == 0)
    c.call()
    c.check(c.result())


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,k,n", [(1, 64, 2), (3, 100, 34), (16, 200, 256), (40, 77, 62), (64, 512, 130), (65, 64, 4), (100, 300, 258), (300, 129, 770)])
def test_gated(cla, t, m, k, n):
    c = Case(cla, m, k, n, t, seed=m + k + n, bias=m % 2 == 0, gated=True)
    c.call()
    c.check(c.result())


@pytest.mark.parametrize("kind", ["sigmoid", "silu", "gelu", "gelu_tanh", "relu", "none"])
@pytest.mark.parametrize("t", ["f64", "bf16"])
@pytest.mark.parametrize("m", [5, 70])
def test_activations(cla, kind, t, m):
    c = Case(cla, m, 100, 96, t, seed=m, gated=True)
    c.call(kind)
    c.check(c.result(), kind)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("t,m,k,n", [("bf16", 2100, 256, 4096), ("f16", 4100, 130, 2050), ("f64", 2050, 70, 4098), ("f32", 2050, 70, 4100)])
def test_large_tiles(cla, t, m, k, n, gated):
    c = Case(cla, m, k, n, t, seed=3, gated=gated)
    c.call()
    c.check(c.result())


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m", [3, 90])
def test_rows_apart(cla, t, m, gated):
    """Leading dimensions beyond the rows, of operands and output, odd ones among them."""
    c = Case(cla, m, 90, 70, t, seed=m, gated=gated, ld_out=75, ld_y=93)
    c.call()
    c.check(c.result())


@pytest.mark.parametrize("m", [4, 100])
def test_rows_that_are_not_finite_stay_to_themselves(cla, m):
    c = Case(cla, m, 70, 50, "f32", seed=1)
    c.call()
    clean = c.result()
    c.Y[2, 3] = np.inf
    c.dY = DevBuf.from_numpy(encode(c.Y, "f32"))
    c.call()
    got = c.result()
    assert np.isnan(got[2]).all()
    rest = np.arange(m) != 2
    assert np.array_equal(got[rest], clean[rest])


def test_longest_sums(cla):
    """131,071 terms of -128 * -128 (values and rows as they are): the largest sum that 32 bits hold."""
    k = 131071
    h = cla.ClaQ8(k, 3).set_values(np.full((k, 3), -128, np.int8), np.ones(3, np.float32))
    ldq = 131072
    for m in (1, 65):
        dQ, dS, dO = DevBuf.from_numpy(np.full((m, ldq), -128, np.int8)), DevBuf.from_numpy(np.ones(m, np.float32)), DevBuf(m * 3 * 8)
        h.lmm_quantized_dev_async(dQ.ptr, ldq, dS.ptr, m, None, dO.ptr, TYPE_IDS["f64"], 3)
        sync()
        assert np.all(dO.to_numpy((m, 3)) == 128.0 * 128.0 * k)


@pytest.mark.parametrize("m", [2, 80])
def test_rows_quantised_once_for_two_matrices(cla, m):
    """Quantised, then two products and a gated unit on the same rows: what the calls from fp32 give, bit by bit; bytes behind the rows do not matter."""
    rng = np.random.default_rng(m)
    k, n, t = 83, 40, TYPE_IDS["f32"]
    Y = rows_of(rng, m, k, "f32")
    hs = [cla.ClaQ8(k, n).set(rng.standard_normal((k, n))) for _ in range(2)]
    dY, ldq = DevBuf.from_numpy(encode(Y, "f32")), 96
    dQ, dS = DevBuf.from_numpy(np.full((m, ldq), 77, np.int8)), DevBuf(4 * m)
    cla.quantize_rows_dev_async(dY.ptr, t, m, k, k, dQ.ptr, ldq, dS.ptr)
    ws = DevBuf(hs[0].workspace(m))
    for h in hs:
        a, b = DevBuf(m * n * 4), DevBuf(m * n * 4)
        h.lmm_quantized_dev_async(dQ.ptr, ldq, dS.ptr, m, None, a.ptr, t, n)
        h.lmm_dev_async(dY.ptr, t, m, k, None, b.ptr, n, ws.ptr, ws.nbytes)
        sync()
        assert np.array_equal(a.to_numpy((m, n), np.float32), b.to_numpy((m, n), np.float32))
        h.gate_quantized_dev_async(1, dQ.ptr, ldq, dS.ptr, m, None, a.ptr, t, n // 2)
        h.gate_dev_async(1, dY.ptr, t, m, k, None, b.ptr, n // 2, ws.ptr, ws.nbytes)
        sync()
        assert np.array_equal(a.to_numpy((m, n // 2), np.float32), b.to_numpy((m, n // 2), np.float32))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("by_column", [False, True])
@pytest.mark.parametrize("k,n", [(1, 1), (70, 33), (129, 65), (2500, 10)])
def test_weights_from_any_type(cla, t, by_column, k, n):
    """Columns are quantised as rows are; values come back as they were set."""
    rng = np.random.default_rng(k)
    W = decode(encode(rng.standard_normal((k, n)), t), t)
    want, scale = quantise(W.T)
    src = encode(W.T if by_column else W, t)
    ld = src.shape[1] + 2
    host = np.zeros((src.shape[0], ld), src.dtype)
    host[:, :src.shape[1]] = src
    d = DevBuf.from_numpy(host)
    h = cla.ClaQ8(k, n).set_dev(d.ptr, TYPE_IDS[t], ld, by_column)
    v, s = h.get()
    assert np.array_equal(v, want.T) and np.array_equal(s, scale)
    if t == "f64" and not by_column:
        v, s = cla.ClaQ8(k, n).set(W).get()
        assert np.array_equal(v, want.T) and np.array_equal(s, scale)
    dV = DevBuf.from_numpy(np.ascontiguousarray(want if by_column else want.T))
    dS = DevBuf.from_numpy(scale)
    v, s = h.set_values_dev(dV.ptr, k if by_column else n, dS.ptr, by_column).get()
    assert np.array_equal(v, want.T) and np.array_equal(s, scale)


def test_host_forms(cla):
    """The forms on host arrays return the number of non-zeros, as the other drivers do."""
    rng = np.random.default_rng(8)
    k, n, m = 60, 24, 37
    W, Y, b = rng.standard_normal((k, n)), rng.standard_normal((m, k)), rng.standard_normal(n)
    Y[5] = 0.0
    h = cla.ClaQ8(k, n).set(W)
    v, s = h.get()
    q, r = quantise(Y)
    p = (q.astype(np.int64) @ v.astype(np.int64)) * r.astype(np.float64)[:, None] * s.astype(np.float64)
    out, nnz = h.lmm(Y)
    assert np.allclose(out, p, rtol=4e-16, atol=0) and nnz == np.count_nonzero(out) == n * (m - 1)
    out, nnz = h.gate("silu", Y, b)
    x = p + b
    g, u = x[:, :12], x[:, 12:]
    assert np.all(np.abs(out - act(g, "silu")[0] * u) <= gated_bound(g, u, 2.0 ** -51 * np.abs(p[:, :12]) + 2.0 ** -53 * np.abs(g), 2.0 ** -51 * np.abs(p[:, 12:]) +
                                                                  2.0 ** -53 * np.abs(u), "silu", "f64"))
    assert nnz == np.count_nonzero(out)
    out, nnz = h.lmm(np.zeros((0, k)))
    assert out.shape == (0, n) and nnz == 0


def test_rows_of_a_compressed_block(cla, ora):
    """A compressed block's rows in 8 bits, and a product on them: what the decompressed rows give."""
    from conftest import mixed_block
    n_rows = 70001
    specs, n_cols = mixed_block(3, n_rows)
    blk = cla.build_block(n_rows, n_cols, specs)
    D, _ = blk.decompress()
    want, scale = quantise(D)
    ldq = 32
    dQ, dS = DevBuf.from_numpy(np.zeros((n_rows, ldq), np.int8)), DevBuf(4 * n_rows)
    blk.quantize_rows_dev_async(dQ.ptr, ldq, dS.ptr)
    sync()
    assert np.array_equal(dS.to_numpy(n_rows, np.float32), scale)
    assert np.array_equal(dQ.to_numpy((n_rows, ldq), np.int8)[:, :n_cols], want)
    h = cla.ClaQ8(n_cols, 40).set(np.random.default_rng(1).standard_normal((n_cols, 40)))
    v, s = h.get()
    dO = DevBuf(n_rows * 40 * 8)
    h.lmm_quantized_dev_async(dQ.ptr, ldq, dS.ptr, n_rows, None, dO.ptr, TYPE_IDS["f64"], 40)
    sync()
    p = (want.astype(np.int64) @ v.astype(np.int64)) * scale.astype(np.float64)[:, None] * s.astype(np.float64)
    assert np.allclose(dO.to_numpy((n_rows, 40)), p, rtol=4e-16, atol=0)
    blk.close()


def test_rows_of_a_compressed_block_captured(cla):
    """... captured behind a first call, replayed when other products of the block have come and grown their own scratch."""
    import ctypes as C

    from conftest import mixed_block
    lib, n_rows = hip(), 30011
    specs, n_cols = mixed_block(4, n_rows)
    blk = cla.build_block(n_rows, n_cols, specs)
    stream, graph, run = C.c_void_p(), C.c_void_p(), C.c_void_p()
    assert lib.hipStreamCreate(C.byref(stream)) == 0
    blk.set_stream(stream.value)
    dQ, dS = DevBuf(n_rows * 32), DevBuf(4 * n_rows)
    blk.quantize_rows_dev_async(dQ.ptr, 32, dS.ptr)
    assert lib.hipStreamSynchronize(stream) == 0
    want, scale = dQ.to_numpy((n_rows, 32), np.int8), dS.to_numpy(n_rows, np.float32)
    assert lib.hipStreamBeginCapture(stream, 0) == 0
    blk.quantize_rows_dev_async(dQ.ptr, 32, dS.ptr)
    assert lib.hipStreamEndCapture(stream, C.byref(graph)) == 0
    assert lib.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0)) == 0
    for turn in range(3):
        blk.aggregate("min", "row")
        blk.tsmm()
        assert lib.hipMemset(dQ.ptr, 0, dQ.nbytes) == 0 and lib.hipMemset(dS.ptr, 0, dS.nbytes) == 0
        sync()
        assert lib.hipGraphLaunch(run, stream) == 0
        sync()
        got = dQ.to_numpy((n_rows, 32), np.int8)
        assert np.array_equal(got[:, :n_cols], want[:, :n_cols]) and np.array_equal(dS.to_numpy(n_rows, np.float32), scale)
    assert lib.hipGraphExecDestroy(run) == 0 and lib.hipGraphDestroy(graph) == 0
    blk.close()
    assert lib.hipStreamDestroy(stream) == 0


def test_two_threads_on_two_matrices(cla):
    """Calls on two handles (streams of their own) from two threads, each checked against its own definition."""
    import threading
    cases = [Case(cla, 90, 300, 200, "bf16", seed=s) for s in (1, 2)]
    errors = []

    def work(c):
        try:
            for _ in range(10):
                c.call()
                c.check(c.result())
        except BaseException as e:  # noqa: BLE001 - reported by the assertion below
            errors.append(repr(e))
    threads = [threading.Thread(target=work, args=(c,)) for c in cases]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


def test_captured_and_replayed(cla):
    """A call captured into a graph on a stream of its own, replayed with new rows in its buffers and eager calls of the same matrix between."""
    import ctypes as C
    lib = hip()
    stream, graph, run = C.c_void_p(), C.c_void_p(), C.c_void_p()
    assert lib.hipStreamCreate(C.byref(stream)) == 0
    for m, gated in ((1, False), (150, True)):
        c = Case(cla, m, 200, 96, "bf16", seed=m, gated=gated)
        c.h.set_stream(stream.value)
        assert lib.hipStreamBeginCapture(stream, 0) == 0
        c.call()
        assert lib.hipStreamEndCapture(stream, C.byref(graph)) == 0
        assert lib.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0)) == 0
        rng = np.random.default_rng(m)
        other = Case(cla, m, 200, 96, "bf16", seed=m + 1, gated=gated)
        for turn in range(4):
            c.Y = rows_of(rng, m, 200, "bf16")
            new = encode(c.Y, "bf16")
            assert lib.hipMemcpy(C.c_void_p(c.dY.ptr), new.ctypes.data_as(C.c_void_p), C.c_size_t(new.nbytes), 1) == 0
            c.clear()
            other.call()
            assert lib.hipGraphLaunch(run, stream) == 0
            other.call()
            c.check(c.result())
            other.check(other.result())
        assert lib.hipGraphExecDestroy(run) == 0 and lib.hipGraphDestroy(graph) == 0
        c.h.close()
    assert lib.hipStreamDestroy(stream) == 0


def test_no_rows(cla):
    h = cla.ClaQ8(10, 4).set(np.ones((10, 4)))
    assert h.workspace(0) >= 0
    h.lmm_dev_async(None, 0, 0, 10, None, None, 4, None, 0)
    h.gate_dev_async(1, None, 0, 0, 10, None, None, 2, None, 0)
    cla.quantize_rows_dev_async(None, 0, 0, 10, 10, None, 10, None)


def test_refusals(cla):
    def refused(code, match, f, *a, **k):
        with pytest.raises(cla.ClaError, match=match) as e:
            f(*a, **k)
        assert e.value.code == code
    for k, n in ((0, 4), (4, 0), (131072, 4), (4, (1 << 21) + 1)):
        refused(-1, "invalid 8-bit matrix", cla.ClaQ8, k, n)
    h = cla.ClaQ8(20, 5)
    d = DevBuf(1 << 16)
    p, ws = d.ptr, h.workspace(4)
    refused(cla.ERR_STATE, "without values", h.lmm_dev_async, p, 0, 4, 20, None, p, 5, p, ws)
    refused(cla.ERR_STATE, "without values", h.get)
    h.set(np.ones((20, 5)))
    ok = (p, 1, 4, 20, None, p + 8192, 5, p + 16384, ws)

    def but(**kw):
        names = ("y", "t", "m", "ldy", "b", "o", "ldo", "ws", "bytes")
        return [kw.get(x, v) for x, v in zip(names, ok)]
    h.lmm_dev_async(*ok)
    refused(cla.ERR_INVALID, "type 4", h.lmm_dev_async, *but(t=4))
    refused(cla.ERR_INVALID, "-1 rows", h.lmm_dev_async, *but(m=-1))
    refused(cla.ERR_INVALID, "Y is null", h.lmm_dev_async, *but(y=None))
    refused(cla.ERR_INVALID, "Y is not aligned", h.lmm_dev_async, *but(y=p + 2))
    refused(cla.ERR_INVALID, "leading dimension 19 of Y", h.lmm_dev_async, *but(ldy=19))
    refused(cla.ERR_INVALID, "the output is null", h.lmm_dev_async, *but(o=None))
    refused(cla.ERR_INVALID, "leading dimension 4 of the output", h.lmm_dev_async, *but(ldo=4))
    refused(cla.ERR_INVALID, "bias is not aligned", h.lmm_dev_async, *but(b=p + 1))
    refused(cla.ERR_INVALID, "workspace of", h.lmm_dev_async, *but(bytes=ws - 1))
    refused(cla.ERR_INVALID, "workspace of", h.lmm_dev_async, *but(ws=None))
    refused(cla.ERR_INVALID, "workspace of", h.lmm_dev_async, *but(ws=p + 8))
    refused(cla.ERR_INVALID, "even number of columns", h.gate_dev_async, 1, *ok)
    refused(cla.ERR_INVALID, "activation 6", h.gate_dev_async, 6, *ok)
    refused(cla.ERR_INVALID, "multiple of 16", h.lmm_quantized_dev_async, p, 20, p + 4096, 4, None, p + 8192, 1, 5)
    refused(cla.ERR_INVALID, "not aligned", h.lmm_quantized_dev_async, p + 4, 32, p + 4096, 4, None, p + 8192, 1, 5)
    refused(cla.ERR_INVALID, "scales is null", h.lmm_quantized_dev_async, p, 32, None, 4, None, p + 8192, 1, 5)
    refused(cla.ERR_INVALID, "W is null", h.set_dev, None, 0, 5)
    refused(cla.ERR_INVALID, "leading dimension 4 of W", h.set_dev, p, 0, 4)
    refused(cla.ERR_INVALID, "leading dimension 5 of W", h.set_dev, p, 0, 5, True)
    refused(cla.ERR_INVALID, "the values is null", h.set_values_dev, None, 5, p)
    blk = cla.ClaBlock(10, 3)
    refused(cla.ERR_STATE, "not finalized", blk.quantize_rows_dev_async, p, 16, p)
    blk.add_const([0, 1, 2], [1.0, 2.0, 3.0])
    blk.finalize()
    refused(cla.ERR_INVALID, "leading dimension 2", blk.quantize_rows_dev_async, p, 2, p)
    sync()
