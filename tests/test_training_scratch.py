"""The library's own scratch of the operators around a language model's matrix products: blocks that grow while work is queued,
several threads on streams of their own and on one stream; and scratch of the callers', of the sizes that they are told."""
import ctypes
import threading

import numpy as np
import pytest

from libnd4j_amd import harness
from test_training_ops import bp_inputs
from test_training_path import Calls, same
from training_views import COMPUTE, STORAGE, SUFFIXES, Vec, View, extra

pytestmark = pytest.mark.gpu

SIZES = ((5, 100), (37, 300), (230, 900), (600, 2400), (100, 5003))  # rows and width, with scratch from less than 1 MiB to 20


@pytest.fixture(scope="module")
def dev():
    return harness.Device()


def prepared(dev, stream, sizes, seed):
    """calls without scratch of their own on `stream`, and what they give with it, one after the other"""
    calls, want = [], []
    for k, (rows, width) in enumerate(sizes):
        ours, theirs = Calls(dev, dev.stream, "Float", rows, width, 300, seed + k), Calls(dev, stream, "Float", rows, width, 300, seed + k, False)
        ours.fresh()
        theirs.fresh()
        ours.run()
        dev.sync()
        want.append(ours.results())
        calls.append(theirs)
    return calls, want


def at_once(works):
    failures = []

    def guarded(work):
        try:
            work()
        except Exception as e:  # reported below, by the thread that asserts
            failures.append(e)

    threads = [threading.Thread(target=guarded, args=(w,)) for w in works]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures


def test_blocks_that_grow_behind_queued_work(dev):
    stream = dev.ops.createStream()
    calls, want = prepared(dev, stream, SIZES, 0)
    for _ in range(2):
        for c in calls + calls[::-1]:
            c.run()
        dev.ops.streamSynchronize(stream)
        for c, w in zip(calls, want):
            assert same(c.results(), w)
        dev.ops.amd_releaseStream(stream)


def test_threads_whose_blocks_grow(dev):
    streams = [dev.ops.createStream() for _ in range(4)]
    held = [prepared(dev, s, SIZES[k % 2:], 10 * k) for k, s in enumerate(streams)]

    def work(calls, stream):
        for _ in range(5):
            for c in calls:
                c.run()
        dev.ops.streamSynchronize(stream)

    at_once([lambda c=c, s=s: work(c, s) for (c, _), s in zip(held, streams)])
    for (calls, want), s in zip(held, streams):
        for c, w in zip(calls, want):
            assert same(c.results(), w)
        dev.ops.amd_releaseStream(s)


@pytest.mark.parametrize("plain", (False, True))
def test_threads_on_one_stream(dev, plain):
    """a call's launches are not mixed with another thread's that use the same block; plain: the stream of null"""
    stream = None if plain else dev.ops.createStream()
    held = [prepared(dev, stream if stream is not None else 0, SIZES[:4][::1 - 2 * (k % 2)], 10 * k) for k in range(4)]
    wait = dev.ops.streamSynchronize

    def work(calls):
        for _ in range(10):
            for c in calls:
                c.run()
        wait(stream)

    at_once([lambda c=c: work(c) for c, _ in held])
    for calls, want in held:
        for c, w in zip(calls, want):
            assert same(c.results(), w)
    dev.ops.amd_releaseStream(stream)


def test_threads_on_the_stream_of_every_thread(dev):
    """hipStreamPerThread, 2: one handle, and a stream and a block of its own for each thread"""
    held = [prepared(dev, 2, SIZES[:4][::1 - 2 * (k % 2)], 10 * k) for k in range(4)]

    def work(calls):
        for _ in range(10):
            for c in calls:
                c.run()
        dev.ops.streamSynchronize(2)
        dev.ops.amd_releaseStream(2)

    at_once([lambda c=c: work(c) for c, _ in held])
    for calls, want in held:
        for c, w in zip(calls, want):
            assert same(c.results(), w)


def test_a_block_grows_without_a_wait(dev):
    """The stream waits for a function of the host's; a call on it that needs a larger block returns all the same, and so does a
    call on another stream.  (The function ends by itself after 20 seconds.)"""
    hip = ctypes.CDLL("libamdhip64.so")
    stream, other = dev.ops.createStream(), dev.ops.createStream()
    (small, large), (want, more) = prepared(dev, stream, (SIZES[0], SIZES[3]), 3)
    (beside,), _ = prepared(dev, other, SIZES[2:3], 5)
    small.run()
    dev.ops.streamSynchronize(stream)
    go, returned = threading.Event(), threading.Event()
    waiting = ctypes.CFUNCTYPE(None, ctypes.c_void_p)(lambda _: go.wait(20) and None)

    def work():
        small.run()
        large.run()
        beside.run()
        returned.set()

    try:
        assert hip.hipLaunchHostFunc(ctypes.c_void_p(stream), waiting, None) == 0
        thread = threading.Thread(target=work)
        thread.start()
        in_time = returned.wait(10)
    finally:
        go.set()
    thread.join()
    dev.ops.streamSynchronize(stream)
    dev.ops.streamSynchronize(other)
    assert in_time
    assert same(small.results(), want) and same(large.results(), more)
    for s in (stream, other):
        dev.ops.amd_releaseStream(s)


@pytest.mark.parametrize("mode", (0, 1, 2))  # global, thread-local, relaxed
def test_eager_calls_beside_a_capture(dev, mode):
    """a stream that is not captured gets its block, and larger ones, and is released, while another one is captured; the graph
    replays as it should"""
    hip = ctypes.CDLL("libamdhip64.so")
    stream, other = dev.ops.createStream(), dev.ops.createStream()
    captured, twin = Calls(dev, stream, "Float", 37, 300, 300, 7), Calls(dev, stream, "Float", 37, 300, 300, 7)
    beside, want = prepared(dev, other, SIZES[:4], 20)
    for c in (captured, twin):
        c.fresh()
    dev.sync()
    graph, executable = ctypes.c_void_p(), ctypes.c_void_p()
    assert hip.hipStreamBeginCapture(ctypes.c_void_p(stream), mode) == 0
    try:
        for c in beside:
            c.run()
        dev.ops.amd_releaseStream(other)
        for c in beside:
            c.run()
        captured.run()
    finally:
        status = hip.hipStreamEndCapture(ctypes.c_void_p(stream), ctypes.byref(graph))
    assert status == 0 and graph.value
    dev.ops.streamSynchronize(other)
    for c, w in zip(beside, want):
        assert same(c.results(), w)
    assert hip.hipGraphInstantiate(ctypes.byref(executable), graph, None, None, ctypes.c_size_t(0)) == 0
    for _ in range(3):
        assert hip.hipGraphLaunch(executable, ctypes.c_void_p(stream)) == 0
        twin.run()
        dev.ops.streamSynchronize(stream)
        assert same(captured.results(), twin.results())
        for c in (captured, twin):
            c.fresh()
        dev.sync()
    hip.hipGraphExecDestroy(executable)
    hip.hipGraphDestroy(graph)
    for s in (stream, other):
        dev.ops.amd_releaseStream(s)


@pytest.mark.parametrize("mode", (0, 1, 2))
def test_shapes_read_back_beside_a_capture(dev, mode):
    """a call without host copies of its shapeInfo, on a stream that is not captured, while another one is"""
    hip = ctypes.CDLL("libamdhip64.so")
    stream, other = dev.ops.createStream(), dev.ops.createStream()
    x = np.random.RandomState(0).randn(6, 40).astype(np.float32)
    X, Z, Y = (View(dev, 6, 40, "dense", np.float32, x) for _ in range(3))
    infos = dev.upload(X.info), dev.upload(Z.info)
    bare = (ctypes.c_void_p * 20)()
    bare[1] = other
    graph = ctypes.c_void_p()
    dev.sync()
    assert hip.hipStreamBeginCapture(ctypes.c_void_p(stream), mode) == 0
    try:
        dev.ops.amd_execLayerNormFloat(bare, X.ptr, infos[0].ptr, None, None, Z.ptr, infos[1].ptr, None, None, 1e-5)
        dev.ops.amd_execLayerNormFloat(extra(dev, x=X, z=Y, stream=stream), X.ptr, None, None, None, Y.ptr, None, None, None, 1e-5)
    finally:
        status = hip.hipStreamEndCapture(ctypes.c_void_p(stream), ctypes.byref(graph))
    assert status == 0 and graph.value
    hip.hipGraphDestroy(graph)
    dev.ops.streamSynchronize(other)
    assert np.array_equal(Y.get(), x)  # (captured, and never launched)
    dev.ops.amd_execLayerNormFloat(extra(dev, x=X, z=Y), X.ptr, None, None, None, Y.ptr, None, None, None, 1e-5)
    assert np.array_equal(Z.get(), Y.get())


BP_SIZES = ((1, 1), (1, 5003), (3, 40), (511, 64), (513, 65), (700, 512), (700, 513), (3000, 1024), (300, 4097), (300, 4098), (260, 8195), (260, 8196),
            (257, 16391), (257, 16392), (100, 70001))


@pytest.mark.parametrize("S", SUFFIXES)
@pytest.mark.parametrize("rows,n", BP_SIZES)
def test_scratch_of_the_size_that_is_asked_for(dev, S, rows, n):
    """what a call is told to bring is enough, and nothing behind it is written"""
    ops, T, C = dev.ops, STORAGE[S], COMPUTE[S]
    rs = np.random.RandomState(rows + n)
    x, gain, mean, inv, dz = bp_inputs(S, rows, n, rows + n)
    tokens = rs.randint(-1, 50, rows)

    def guarded(size):
        return size, dev.upload(np.full(size + 4096, 0x5a, np.uint8))

    def whole(size, buf):
        assert (buf.download(np.uint8)[size:] == 0x5a).all()
        buf.free()

    for layout in ("dense", "inner2", "forder"):
        X, DZ, DX = View(dev, rows, n, layout, T, x), View(dev, rows, n, layout, T, dz), View(dev, rows, n, layout, T)
        M, I, DG, DB = Vec(dev, mean, C), Vec(dev, inv, C), Vec(dev, np.zeros(n), T), Vec(dev, np.zeros(n), T)
        size, buf = guarded(ops.amd_scratchLayerNormBp(rows, n))
        getattr(ops, "amd_execLayerNormBp" + S)(extra(dev, x=X, y=DZ, z=DX), X.ptr, X.info_ptr, None, M.ptr, I.ptr, DZ.ptr, DZ.info_ptr, DX.ptr, DX.info_ptr,
                                                DG.ptr, DB.ptr, buf.ptr, size)
        whole(size, buf)
        W, K = View(dev, 50, n, layout, T), Vec(dev, tokens, np.int64)
        size, buf = guarded(ops.amd_scratchEmbeddingBp(rows, 50, n))
        getattr(ops, "amd_execEmbeddingBp" + S)(extra(dev, x=DZ, z=W), DZ.ptr, DZ.info_ptr, K.ptr, rows, W.ptr, W.info_ptr, 1.0, 0, buf.ptr, size)
        whole(size, buf)
        k = min(n, 64)
        top, top_lp, lp = Vec(dev, np.zeros(rows * k), np.int64), Vec(dev, np.zeros(rows * k), C), Vec(dev, np.zeros(rows), C)
        size, buf = guarded(ops.amd_scratchTokenLogProbs(rows, n, k))
        getattr(ops, "amd_execTokenLogProbs" + S)(extra(dev, x=X), X.ptr, X.info_ptr, K.ptr, lp.ptr, None, None, k, top.ptr, top_lp.ptr, buf.ptr if size else None, size)
        whole(size, buf)
        for v in (X, DZ, DX, M, I, DG, DB, W, K, top, top_lp, lp):
            v.free()


@pytest.mark.parametrize("S", SUFFIXES)
@pytest.mark.parametrize("count", (1, 60))
def test_scratch_of_clipping_of_the_size_that_is_asked_for(dev, S, count):
    ops, total = dev.ops, 20000003
    flat = dev.empty(total * STORAGE[S]().itemsize)
    ops.memset(flat.ptr, 0, total * STORAGE[S]().itemsize, 0, None)
    ends = np.linspace(0, total, count + 1).astype(np.int64)
    tables, offsets = dev.upload(flat.ptr + ends[:-1] * STORAGE[S]().itemsize), Vec(dev, ends, np.int64)
    norm = Vec(dev, [1.0], COMPUTE[S])
    size = ops.amd_scratchClipByGlobalNorm(total)
    buf = dev.upload(np.full(size + 4096, 0x5a, np.uint8))
    getattr(ops, "amd_execClipByGlobalNorm" + S)(extra(dev), tables.ptr, tables.ptr, offsets.ptr, count, total, 1.0, norm.ptr, buf.ptr, size)
    assert (buf.download(np.uint8)[size:] == 0x5a).all() and norm.get()[0] == 0
    for v in (flat, tables, offsets, norm, buf):
        v.free()
