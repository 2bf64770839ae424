"""The operators around a language model's matrix products as a program uses them: together, captured into graphs, on
streams of their own, over buffers whose offsets pass 32 bits."""
import ctypes
import threading

import numpy as np
import pytest

from libnd4j_amd import harness
from libnd4j_amd.native import Nd4jError
from training_views import COMPUTE, STORAGE, SUFFIXES, Vec, View, extra

pytestmark = pytest.mark.gpu

EPS = 1e-5


@pytest.fixture(scope="module")
def dev():
    return harness.Device()


class Model(object):
    """tokens -> scaled embedding -> layer norm -> logits (the embedding table again) -> log probabilities of the next tokens,
    and back: everything but the products of matrices, which are numpy's, runs through the library"""

    def __init__(self, dev, S, vocabulary=50, width=24, rows=17, seed=0):
        self.dev, self.S = dev, S
        rs = np.random.RandomState(seed)
        T = STORAGE[S]
        self.table = (rs.randn(vocabulary, width) / 4).astype(T)
        self.gain, self.bias = (1 + rs.randn(width) / 8).astype(T), (rs.randn(width) / 8).astype(T)
        self.tokens = rs.randint(0, vocabulary, rows)
        self.tokens[3] = self.tokens[5] = self.tokens[0]
        self.tokens[-1] = -1
        self.next = rs.randint(0, vocabulary, rows)
        self.next[-1] = -1  # padding
        self.scale, self.weight, self.h_weight = 1.5, rs.randn(rows), rs.randn(rows) / 8

    def run(self, gradients=True):
        dev, S, T, C = self.dev, self.S, STORAGE[self.S], COMPUTE[self.S]
        ops, (v, d), n = dev.ops, self.table.shape, len(self.tokens)
        call = lambda name: getattr(ops, "amd_exec" + name + S)  # noqa: E731
        W, K, NEXT = View(dev, v, d, "dense", T, self.table), Vec(dev, self.tokens, np.int64), Vec(dev, self.next, np.int64)
        E, Z = View(dev, n, d, "dense", T), View(dev, n, d, "dense", T)
        G, B, M, I = Vec(dev, self.gain, T), Vec(dev, self.bias, T), Vec(dev, np.zeros(n), C), Vec(dev, np.zeros(n), C)
        call("Embedding")(extra(dev, x=W, z=E), W.ptr, W.info_ptr, K.ptr, n, E.ptr, E.info_ptr, self.scale)
        call("LayerNorm")(extra(dev, x=E, z=Z), E.ptr, E.info_ptr, G.ptr, B.ptr, Z.ptr, Z.info_ptr, M.ptr, I.ptr, EPS)
        z = Z.get()
        # products of matrices come out in f order here as often as not
        logits = View(dev, n, v, "forder", T, (z.astype(np.float64) @ self.table.astype(np.float64).T))
        lp, ls, h = (Vec(dev, np.zeros(n), C) for _ in range(3))
        call("TokenLogProbs")(extra(dev, x=logits), logits.ptr, logits.info_ptr, NEXT.ptr, lp.ptr, ls.ptr, h.ptr, 0, None, None, None, 0)
        loss = float((lp.get().astype(np.float64) * self.weight + h.get().astype(np.float64) * self.h_weight).sum())
        if not gradients:
            return loss
        dl = View(dev, n, v, "dense", T)
        a, b = Vec(dev, self.weight, C), Vec(dev, self.h_weight, C)
        call("TokenLogProbsBp")(extra(dev, x=logits, z=dl), logits.ptr, logits.info_ptr, NEXT.ptr, ls.ptr, h.ptr, a.ptr, b.ptr, dl.ptr, dl.info_ptr)
        dlogits = dl.get().astype(np.float64)
        dz = View(dev, n, d, "dense", T, dlogits @ self.table.astype(np.float64))
        dtable = View(dev, v, d, "dense", T, dlogits.T @ z.astype(np.float64))  # the table as the last product's operand
        de, dg, db = View(dev, n, d, "dense", T), Vec(dev, np.zeros(d), T), Vec(dev, np.zeros(d), T)
        call("LayerNormBp")(extra(dev, x=E, y=dz, z=de), E.ptr, E.info_ptr, G.ptr, M.ptr, I.ptr, dz.ptr, dz.info_ptr, de.ptr, de.info_ptr, dg.ptr,
                            db.ptr, None, 0)
        call("EmbeddingBp")(extra(dev, x=de, z=dtable), de.ptr, de.info_ptr, K.ptr, n, dtable.ptr, dtable.info_ptr, self.scale, 1, None, 0)
        grads = [dtable.get(), dg.get(), db.get()]
        # clipped in place, as one step of training does
        held = [dtable, dg, db]
        tables = dev.upload(np.array([t.ptr for t in held], dtype=np.int64))
        offsets = Vec(dev, np.cumsum([0] + [g.size for g in grads]), np.int64)
        norm = Vec(dev, [0.0], C)
        total = sum(g.size for g in grads)
        call("ClipByGlobalNorm")(extra(dev), tables.ptr, tables.ptr, offsets.ptr, 3, total, 0.5, norm.ptr, None, 0)
        clipped = [dtable.get(), dg.get(), db.get()]
        return loss, grads, clipped, float(norm.get()[0])


def test_a_training_step_in_double_against_differences(dev):
    """central differences of the loss over the table, gain and bias: an error of order h^2 and one of eps / h"""
    m = Model(dev, "Double")
    loss, (dtable, dg, db), clipped, norm = m.run()
    h = 1e-5
    for array, grad, places in ((m.table, dtable, [(int(m.tokens[0]), 3), (int(m.next[2]), 0), (7, 23)]), (m.gain, dg, [0, 11]), (m.bias, db, [5, 23])):
        for at in places:
            old = array[at]
            array[at] = old + h
            up = m.run(False)
            array[at] = old - h
            down = m.run(False)
            array[at] = old
            assert abs((up - down) / (2 * h) - grad[at]) < 1e-7 * (1 + abs(grad[at])), at
    want = np.sqrt(sum((g ** 2).sum() for g in (dtable, dg, db)))
    assert abs(norm - want) < 1e-12 * want and want > 0.5
    for c, g in zip(clipped, (dtable, dg, db)):
        assert np.allclose(c, g * (0.5 / want), rtol=1e-14, atol=0)


@pytest.mark.parametrize("S,bound", [("Float", 1e-4), ("Half", 0.05)])
def test_a_training_step_in_other_types(dev, S, bound):
    """Against the step in double, by the norm of the difference.  Every value passes about ten roundings of the type on its
    way through products of 24 and 50 terms: some hundred roundings of 6e-8 or 5e-4."""
    exact, rounded = Model(dev, "Double"), Model(dev, S)
    exact.table, exact.gain, exact.bias = (v.astype(np.float64) for v in (rounded.table, rounded.gain, rounded.bias))
    want, got = exact.run(), rounded.run()
    assert abs(got[0] - want[0]) < bound * (1 + abs(want[0]))
    for g, w in zip(got[1], want[1]):
        assert np.linalg.norm(g.astype(np.float64) - w) < bound * np.linalg.norm(w)
    again = rounded.run()
    for g, w in zip(got[1] + got[2], again[1] + again[2]):
        assert np.array_equal(g, w)  # the same bits every time


class Calls(object):
    """One call of every operator on buffers of its own, on a stream of the caller's choice"""

    def __init__(self, dev, stream, S="Float", rows=37, width=300, vocabulary=900, seed=0, scratch=True):
        self.dev, self.stream, self.S = dev, stream, S
        T, C = STORAGE[S], COMPUTE[S]
        self.rs = np.random.RandomState(seed)
        self.rows, self.width, self.vocabulary = rows, width, vocabulary
        V = lambda r, n: View(dev, r, n, "dense", T)  # noqa: E731
        self.table, self.x, self.z, self.dz, self.dx, self.dtable = V(vocabulary, width), V(rows, width), V(rows, width), V(rows, width), V(rows, width), V(vocabulary, width)
        self.logits, self.dlogits = V(rows, 5003), V(rows, 5003)
        self.tokens, self.next = Vec(dev, np.zeros(rows), np.int64), Vec(dev, np.zeros(rows), np.int64)
        self.gain, self.bias, self.dg, self.db = (Vec(dev, np.zeros(width), T) for _ in range(4))
        self.mean, self.inv, self.lp, self.ls, self.h, self.a = (Vec(dev, np.zeros(rows), C) for _ in range(6))
        self.top, self.top_lp = Vec(dev, np.zeros(rows * 6), np.int64), Vec(dev, np.zeros(rows * 6), C)
        self.norm = Vec(dev, [0.0], C)
        self.clipped = V(vocabulary, width), V(1, width)
        self.tables = dev.upload(np.array([[self.dtable.ptr, self.dg.ptr], [self.clipped[0].ptr, self.clipped[1].ptr]], dtype=np.int64))
        self.offsets = Vec(dev, [0, vocabulary * width, (vocabulary + 1) * width], np.int64)
        self.total = (vocabulary + 1) * width
        o = dev.ops
        sizes = [o.amd_scratchLayerNormBp(rows, width), o.amd_scratchEmbeddingBp(rows, vocabulary, width), o.amd_scratchTokenLogProbs(rows, 5003, 6),
                 o.amd_scratchClipByGlobalNorm(self.total)]
        self.scratch = [(dev.empty(n), n) for n in sizes] if scratch else [(None, 0)] * 4

    def fresh(self):
        """new inputs in the same buffers"""
        rs, ops = self.rs, self.dev.ops

        def put(v, values, dtype):
            a = np.ascontiguousarray(values, dtype=dtype)
            ops.memcpy(v.ptr, a.ctypes.data, a.nbytes, 1, None)

        T, C = STORAGE[self.S], COMPUTE[self.S]
        put(self.table, rs.randn(self.vocabulary, self.width), T)
        put(self.dz, rs.randn(self.rows, self.width), T)
        put(self.logits, rs.randn(self.rows, 5003) * 3, T)
        put(self.tokens, np.minimum(rs.randint(-1, self.vocabulary, self.rows), rs.randint(0, self.vocabulary, self.rows)), np.int64)
        put(self.next, rs.randint(-1, 5003, self.rows), np.int64)
        put(self.gain, 1 + rs.randn(self.width) / 8, T)
        put(self.bias, rs.randn(self.width), T)
        put(self.a, rs.randn(self.rows), C)

    def run(self):
        o, S = self.dev.ops, self.S
        call = lambda name: getattr(o, "amd_exec" + name + S)  # noqa: E731
        ex = lambda **k: extra(self.dev, stream=self.stream, **k)  # noqa: E731
        w = [(m and m.ptr, n) for m, n in self.scratch]
        call("Embedding")(ex(x=self.table, z=self.x), self.table.ptr, self.table.info_ptr, self.tokens.ptr, self.rows, self.x.ptr, self.x.info_ptr, 2.0)
        call("LayerNorm")(ex(x=self.x, z=self.z), self.x.ptr, self.x.info_ptr, self.gain.ptr, self.bias.ptr, self.z.ptr, self.z.info_ptr, self.mean.ptr,
                          self.inv.ptr, EPS)
        call("LayerNormBp")(ex(x=self.x, y=self.dz, z=self.dx), self.x.ptr, self.x.info_ptr, self.gain.ptr, self.mean.ptr, self.inv.ptr, self.dz.ptr,
                            self.dz.info_ptr, self.dx.ptr, self.dx.info_ptr, self.dg.ptr, self.db.ptr, *w[0])
        call("EmbeddingBp")(ex(x=self.dx, z=self.dtable), self.dx.ptr, self.dx.info_ptr, self.tokens.ptr, self.rows, self.dtable.ptr,
                            self.dtable.info_ptr, 2.0, 0, *w[1])
        call("TokenLogProbs")(ex(x=self.logits), self.logits.ptr, self.logits.info_ptr, self.next.ptr, self.lp.ptr, self.ls.ptr, self.h.ptr, 6, self.top.ptr,
                              self.top_lp.ptr, *w[2])
        call("TokenLogProbsBp")(ex(x=self.logits, z=self.dlogits), self.logits.ptr, self.logits.info_ptr, self.next.ptr, self.ls.ptr, self.h.ptr,
                                self.a.ptr, None, self.dlogits.ptr, self.dlogits.info_ptr)
        call("ClipByGlobalNorm")(ex(), self.tables.ptr, self.tables.ptr + 16, self.offsets.ptr, 2, self.total, 1.0, self.norm.ptr, *w[3])

    def results(self):
        return [v.get(False) if isinstance(v, View) else v.get() for v in (
            self.x, self.z, self.dx, self.dtable, self.dlogits, self.clipped[0], self.clipped[1], self.mean, self.inv, self.dg, self.db, self.lp, self.ls,
            self.h, self.top, self.top_lp, self.norm)]


def same(a, b):
    return all(np.array_equal(u, v, equal_nan=True) for u, v in zip(a, b))


def test_calls_in_captured_graphs(dev):
    """Two graphs captured on one stream, with scratch of their own, replayed in turn and at the same time on two streams, with
    new inputs, eager calls and synchronizations in between: the bits of the eager calls every time.  Without scratch a call is
    refused while the stream is captured, and the capture goes on."""
    hip = ctypes.CDLL("libamdhip64.so")
    ops = dev.ops
    calls = [Calls(dev, dev.stream, S, seed=k) for k, S in enumerate(("Float", "Half"))]
    eager = [Calls(dev, dev.stream, S, seed=k, scratch=False) for k, S in enumerate(("Float", "Half"))]
    stream, other = ctypes.c_void_p(dev.stream), ctypes.c_void_p(ops.createStream())
    executables, graphs = [], []
    for c in calls:
        graph, executable = ctypes.c_void_p(), ctypes.c_void_p()
        assert hip.hipStreamBeginCapture(stream, 1) == 0  # 1: thread-local capture mode
        try:
            c.run()
            held, c.scratch = c.scratch, [(None, 0)] * 4
            with pytest.raises(Nd4jError, match="scratch"):
                c.run()
            c.scratch = held
            ops.amd_scratchClipByGlobalNorm(1)  # (a call that succeeds: members like memcpy leave the last error as it was)
        finally:
            status = hip.hipStreamEndCapture(stream, ctypes.byref(graph))
        assert status == 0 and graph.value
        assert hip.hipGraphInstantiate(ctypes.byref(executable), graph, None, None, ctypes.c_size_t(0)) == 0
        graphs.append(graph)
        executables.append(executable)
    try:
        for replay in range(4):
            for c, e in zip(calls, eager):
                c.fresh()
                e.fresh()
            dev.sync()
            assert hip.hipGraphLaunch(executables[0], stream) == 0
            assert hip.hipGraphLaunch(executables[1], other if replay % 2 else stream) == 0
            for e in eager:
                e.run()
            dev.sync()
            assert hip.hipStreamSynchronize(other) == 0
            for c, e in zip(calls, eager):
                assert same(c.results(), e.results()), replay
    finally:
        for e, g in zip(executables, graphs):
            hip.hipGraphExecDestroy(e)
            hip.hipGraphDestroy(g)


def test_a_captured_call_needs_host_copies(dev):
    """without one the shapeInfo would be read back, which ends a capture: refused, and the capture goes on"""
    hip = ctypes.CDLL("libamdhip64.so")
    ops, stream, graph = dev.ops, ctypes.c_void_p(dev.stream), ctypes.c_void_p()
    rs = np.random.RandomState(2)
    x = rs.randn(6, 40).astype(np.float32)
    X, Z = View(dev, 6, 40, "dense", np.float32, x), View(dev, 6, 40, "dense", np.float32)
    full, bare = (ctypes.c_void_p * 20)(), (ctypes.c_void_p * 20)()
    full[0], full[1], full[8] = X.info.ctypes.data, dev.stream, Z.info.ctypes.data
    bare[1] = dev.stream
    infos = dev.upload(X.info), dev.upload(Z.info)
    args = (X.ptr, infos[0].ptr, None, None, Z.ptr, infos[1].ptr, None, None, 1e-5)
    dev.sync()
    assert hip.hipStreamBeginCapture(stream, 1) == 0  # 1: thread-local capture mode
    try:
        with pytest.raises(Nd4jError, match="host copy"):
            ops.amd_execLayerNormFloat(bare, *args)
        ops.amd_execLayerNormFloat(full, *args)
    finally:
        status = hip.hipStreamEndCapture(stream, ctypes.byref(graph))
    assert status == 0 and graph.value
    hip.hipGraphDestroy(graph)
    ops.amd_execLayerNormFloat(bare, *args)  # outside of a capture it is read back
    dev.sync()
    want = (x - x.mean(1, keepdims=True)) / np.sqrt(x.var(1, keepdims=True) + 1e-5)
    assert np.abs(Z.get() - want).max() < 1e-5  # (values below 4, a dozen roundings of 2^-24 of them)
    for v in (X, Z) + infos:
        v.free()


def test_calls_from_threads_on_streams_of_their_own(dev):
    """four threads, a stream and the library's scratch each: the results of one thread alone; then the streams are released"""
    ops = dev.ops
    streams = [ops.createStream() for _ in range(4)]
    calls = [Calls(dev, s, "Float", rows=37 + 200 * k, seed=k, scratch=False) for k, s in enumerate(streams)]
    want = []
    for c in calls:
        c.fresh()
        c.run()
        ops.streamSynchronize(c.stream)
        want.append(c.results())
    failures = []

    def work(c):
        try:
            for _ in range(20):
                c.run()
            ops.streamSynchronize(c.stream)
        except Exception as e:  # reported below, by the thread that asserts
            failures.append(e)

    threads = [threading.Thread(target=work, args=(c,)) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures
    for c, w in zip(calls, want):
        assert same(c.results(), w)
        ops.amd_releaseStream(c.stream)
        c.run()
        ops.streamSynchronize(c.stream)
        assert same(c.results(), w)
        ops.amd_releaseStream(c.stream)


def test_offsets_beyond_32_bits(dev):
    """three rows of halves 2^31 + 40 elements apart, more than 4 GiB: every operator reads and writes the right ones"""
    ops, n, pitch = dev.ops, 300, (1 << 31) + 40
    rs = np.random.RandomState(0)
    big, out = dev.empty(2 * (2 * pitch + n)), dev.empty(2 * (2 * pitch + n))
    info = harness.shape_info([3, n], strides=[pitch, 1])
    plain = harness.shape_info([3, n])
    x = rs.randn(3, n).astype(np.float16)

    def put(buf, values):
        for r in range(3):
            row = np.ascontiguousarray(values[r])
            ops.memcpy(buf.ptr + 2 * r * pitch, row.ctypes.data, row.nbytes, 1, None)

    def get(buf):
        dev.sync()
        rows = np.zeros((3, n), np.float16)
        for r in range(3):
            ops.memcpy(rows[r:].ctypes.data, buf.ptr + 2 * r * pitch, 2 * n, 2, None)
        return rows

    class At(object):
        def __init__(self, i):
            self.info = i

    far, near = At(info), At(plain)
    small, result = dev.upload(x), dev.upload(np.zeros((3, n), np.float16))
    mean, inv, ls, lp = (Vec(dev, np.zeros(3), np.float32) for _ in range(4))
    tokens, top, top_lp = Vec(dev, [2, 0, 2], np.int64), Vec(dev, np.zeros(6), np.int64), Vec(dev, np.zeros(6), np.float32)
    dg, db = Vec(dev, np.zeros(n), np.float16), Vec(dev, np.zeros(n), np.float16)
    I, J = info.ctypes.data, plain.ctypes.data

    def both(call):
        """the call on the far rows and on dense ones"""
        put(big, x)
        put(out, np.zeros((3, n), np.float16))
        call(far, big.ptr, I, far, out.ptr, I)
        first = get(out), [v.get() for v in (mean, inv, ls, lp, top, dg, db)]
        ops.memset(result.ptr, 0, 6 * n, 0, None)
        call(near, small.ptr, J, near, result.ptr, J)
        second = result.download(np.float16).reshape(3, n), [v.get() for v in (mean, inv, ls, lp, top, dg, db)]
        assert np.array_equal(first[0], second[0])
        for a, b in zip(first[1], second[1]):
            assert np.array_equal(a, b)

    both(lambda a, p, i, b, q, j: ops.amd_execLayerNormHalf(extra(dev, x=a, z=b), p, i, None, None, q, j, mean.ptr, inv.ptr, EPS))
    both(lambda a, p, i, b, q, j: ops.amd_execLayerNormBpHalf(extra(dev, x=a, y=a, z=b), p, i, None, mean.ptr, inv.ptr, p, i, q, j, dg.ptr, db.ptr, None, 0))
    both(lambda a, p, i, b, q, j: ops.amd_execEmbeddingHalf(extra(dev, x=a, z=b), p, i, tokens.ptr, 3, q, j, 1.0))
    both(lambda a, p, i, b, q, j: ops.amd_execEmbeddingBpHalf(extra(dev, x=a, z=b), p, i, tokens.ptr, 3, q, j, 1.0, 0, None, 0))
    both(lambda a, p, i, b, q, j: ops.amd_execTokenLogProbsHalf(extra(dev, x=a), p, i, tokens.ptr, lp.ptr, ls.ptr, None, 2, top.ptr, top_lp.ptr, None, 0))
    both(lambda a, p, i, b, q, j: ops.amd_execTokenLogProbsBpHalf(extra(dev, x=a, z=b), p, i, tokens.ptr, ls.ptr, None, lp.ptr, None, q, j))
    for v in (big, out, small, result):
        v.free()


def test_clipping_more_than_2_31_elements(dev):
    """two tensors of halves, 2^31 + 5000 elements in all, zero but for a few"""
    ops = dev.ops
    lengths = [1001, (1 << 31) + 3999]
    total = sum(lengths)
    big = dev.empty(2 * (total + 8))
    ops.memset(big.ptr, 0, 2 * (total + 8), 0, None)
    places = [0, 1000, 1001, 1 << 31, total - 1]
    three = np.array([3.0], np.float16)
    for p in places:
        ops.memcpy(big.ptr + 2 * p, three.ctypes.data, 2, 1, None)
    tables = dev.upload(np.array([big.ptr, big.ptr + 2 * lengths[0]], dtype=np.int64))
    offsets, norm = Vec(dev, [0, lengths[0], total], np.int64), Vec(dev, [0.0], np.float32)
    ops.amd_execClipByGlobalNormHalf(extra(dev), tables.ptr, tables.ptr, offsets.ptr, 2, total, 1.0, norm.ptr, None, 0)
    assert abs(norm.get()[0] - np.sqrt(45.0)) < 1e-6
    for p in places:
        value = np.zeros(1, np.float16)
        ops.memcpy(value.ctypes.data, big.ptr + 2 * p, 2, 2, None)
        assert value[0] == np.float16(np.float32(3.0) * np.float32(1 / np.sqrt(45.0)))
    big.free()
