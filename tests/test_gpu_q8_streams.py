"""A compressed block's rows to 8 bits, and an 8-bit matrix, on several streams and in several graphs."""
import ctypes as C

import numpy as np
import pytest

from devmem import DevBuf, hip

pytestmark = pytest.mark.gpu


def ok(rc):
    assert rc == 0, rc


def streams(n):
    out = [C.c_void_p() for _ in range(n)]
    for s in out:
        ok(hip().hipStreamCreate(C.byref(s)))
    return out


N_ROWS, N_COLS, LDQ = 500_009, 40, 48  # (three chunks of decoded rows)


def block(cla, seed=1):
    rng = np.random.default_rng(seed)
    blk = cla.ClaBlock(N_ROWS, N_COLS)
    for c in range(N_COLS):
        blk.add_ddc([c], rng.standard_normal((200, 1)), rng.integers(0, 200, N_ROWS).astype(np.uint8))
    blk.finalize()
    return blk


class Out:
    def __init__(self):
        self.q, self.s = DevBuf(N_ROWS * LDQ), DevBuf(4 * N_ROWS)

    def clear(self):
        ok(hip().hipMemset(self.q.ptr, 0, self.q.nbytes))
        ok(hip().hipMemset(self.s.ptr, 0, self.s.nbytes))

    def get(self):
        return self.q.to_numpy((N_ROWS, LDQ), np.int8)[:, :N_COLS], self.s.to_numpy(N_ROWS, np.float32)

    def same(self, want):
        q, s = self.get()
        assert np.array_equal(s, want[1]) and np.array_equal(q, want[0])


def first(blk):
    o = Out()
    blk.quantize_rows_dev_async(o.q.ptr, LDQ, o.s.ptr)
    ok(hip().hipDeviceSynchronize())
    return o.get()


def test_a_block_that_changes_streams(cla):
    """Calls of one block, queued on streams in turn, an output to each."""
    blk = block(cla)
    want, ss, outs = first(blk), streams(3), [Out() for _ in range(6)]
    for turn in range(2):
        for o in outs:
            o.clear()
        ok(hip().hipDeviceSynchronize())
        for i, o in enumerate(outs):
            blk.set_stream(ss[i % 3].value)
            blk.quantize_rows_dev_async(o.q.ptr, LDQ, o.s.ptr)
        ok(hip().hipDeviceSynchronize())
        for o in outs:
            o.same(want)
    blk.close()
    for s in ss:
        ok(hip().hipStreamDestroy(s))


def test_graphs_of_one_block_at_once(cla):
    """Two graphs of one block (the first of them its first call) replayed at once, beside a call of the block on a third stream."""
    lib, blk, ss, outs, runs = hip(), block(cla), streams(3), [Out() for _ in range(3)], []
    for s, o in zip(ss[:2], outs):
        graph, run = C.c_void_p(), C.c_void_p()
        blk.set_stream(s.value)
        ok(lib.hipStreamBeginCapture(s, 0))
        blk.quantize_rows_dev_async(o.q.ptr, LDQ, o.s.ptr)
        ok(lib.hipStreamEndCapture(s, C.byref(graph)))
        ok(lib.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0)))
        runs.append((graph, run))
    blk.set_stream(ss[2].value)
    want = first(blk)
    for turn in range(4):
        for o in outs:
            o.clear()
        ok(lib.hipDeviceSynchronize())
        for s, (_, run) in zip(ss, runs):
            ok(lib.hipGraphLaunch(run, s))
        blk.quantize_rows_dev_async(outs[2].q.ptr, LDQ, outs[2].s.ptr)
        ok(lib.hipDeviceSynchronize())
        for o in outs:
            o.same(want)
    for graph, run in runs:
        ok(lib.hipGraphExecDestroy(run))
        ok(lib.hipGraphDestroy(graph))
    blk.close()
    for s in ss:
        ok(lib.hipStreamDestroy(s))


def test_chunks_go_with_the_block(cla):
    """What captured calls hold is freed with the block."""
    from devmem import free_device_bytes
    lib, (s,), o = hip(), streams(1), Out()

    def once():
        blk, graph = block(cla), C.c_void_p()
        blk.set_stream(s.value)
        blk.quantize_rows_dev_async(o.q.ptr, LDQ, o.s.ptr)
        for _ in range(3):
            ok(lib.hipStreamBeginCapture(s, 0))
            blk.quantize_rows_dev_async(o.q.ptr, LDQ, o.s.ptr)
            ok(lib.hipStreamEndCapture(s, C.byref(graph)))
            ok(lib.hipGraphDestroy(graph))
        ok(lib.hipDeviceSynchronize())
        blk.close()
    once()
    before = free_device_bytes()
    for _ in range(3):
        once()
    assert free_device_bytes() > before - (64 << 20)
    ok(lib.hipStreamDestroy(s))


def test_values_replaced_while_products_are_on_their_way(cla):
    """Products queued on one stream see the values that the matrix had, though it is on another stream when they are replaced; later ones the new values."""
    rng = np.random.default_rng(4)
    lib, (a, b), m, k, n = hip(), streams(2), 4096, 4096, 4096
    Y = DevBuf.from_numpy(rng.standard_normal((m, k)).astype(np.float32))
    h = cla.ClaQ8(k, n)
    W = [rng.integers(-127, 128, (k, n)).astype(np.int8) for _ in range(2)]
    scales = np.ones(n, np.float32)
    ws, want = DevBuf(h.workspace(m)), []
    for w in W:
        h.set_values(w, scales)
        o = DevBuf(m * n * 4)
        h.lmm_dev_async(Y.ptr, 1, m, k, None, o.ptr, n, ws.ptr, ws.nbytes)
        ok(lib.hipDeviceSynchronize())
        want.append(o.to_numpy((m, n), np.float32))
    dW, dS = [DevBuf.from_numpy(np.ascontiguousarray(w.T)) for w in W], DevBuf.from_numpy(scales)
    outs = [DevBuf(m * n * 4) for _ in range(6)]
    for turn in range(2):
        h.set_values_dev(dW[0].ptr, k, dS.ptr, True)
        h.set_stream(a.value)
        for o in outs[:5]:
            h.lmm_dev_async(Y.ptr, 1, m, k, None, o.ptr, n, ws.ptr, ws.nbytes)
        h.set_stream(b.value)
        h.set_values_dev(dW[1].ptr, k, dS.ptr, True)
        h.lmm_dev_async(Y.ptr, 1, m, k, None, outs[5].ptr, n, ws.ptr, ws.nbytes)
        ok(lib.hipDeviceSynchronize())
        for i, o in enumerate(outs):
            assert np.array_equal(o.to_numpy((m, n), np.float32), want[i == 5])
    h.close()
    for s in (a, b):
        ok(lib.hipStreamDestroy(s))
