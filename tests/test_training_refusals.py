"""What the operators around a language model's matrix products refuse, before anything is enqueued: no GPU needed."""
import ctypes

import numpy as np
import pytest

from libnd4j_amd import harness
from libnd4j_amd.native import Nd4jError, NativeOps

SUFFIXES = ("Float", "Half", "Double")
P = 1 << 20  # an address that is never looked at


@pytest.fixture(scope="module")
def ops():
    return NativeOps()


def info(*shape, **kw):
    return harness.shape_info(list(shape), **kw)


def extra(x=None, y=None, z=None):
    e = (ctypes.c_void_p * 20)()
    for slot, v in ((0, x), (7, y), (8, z)):
        if v is not None:
            e[slot] = v.ctypes.data
    e._keep = (x, y, z)
    return e


A, B, EMPTY = info(4, 8), info(4, 9), info(4, 0)
SPLIT = info(2, 2, 8, strides=[100, 8, 1])
LONG = info(1, 1 << 31)


@pytest.mark.parametrize("S", SUFFIXES)
@pytest.mark.parametrize("why,x,z,args", [
    ("differ in shape", A, B, {}), ("without elements", EMPTY, EMPTY, {}), ("do not merge", SPLIT, SPLIT, {}), ("2\\^31", LONG, LONG, {}),
    ("epsilon", A, A, {"eps": -1.0}), ("epsilon", A, A, {"eps": float("nan")}), ("x is null", A, A, {"x": None}), ("z is null", A, A, {"z": None}),
    ("not aligned", A, A, {"x": P + 1}), ("not aligned", A, A, {"gain": P + 1}), ("not aligned", A, A, {"mean": P + 2})])
def test_layer_norm(ops, S, why, x, z, args):
    with pytest.raises(Nd4jError, match=why):
        getattr(ops, "amd_execLayerNorm" + S)(extra(x=x, z=z), args.get("x", P), x.ctypes.data, args.get("gain", P), P, args.get("z", P),
                                              z.ctypes.data, args.get("mean", P), P, args.get("eps", 1e-5))


@pytest.mark.parametrize("S", SUFFIXES)
@pytest.mark.parametrize("why,args", [
    ("differ in shape", {"dzi": B}), ("differ in shape", {"dxi": B}), ("no gradient", {"dx": None, "dg": None, "db": None}),
    ("mean is null", {"mean": None}), ("invStd is null", {"inv": None}), ("dz is null", {"dz": None}), ("not aligned", {"dg": P + 1}),
    ("scratch holds", {"w": P, "wb": 8}), ("scratch holds", {"w": P, "wb": -1}), ("not aligned to 16", {"w": P + 8, "wb": 1 << 30})])
def test_layer_norm_bp(ops, S, why, args):
    g = lambda key, other=P: args.get(key, other)  # noqa: E731
    with pytest.raises(Nd4jError, match=why):
        getattr(ops, "amd_execLayerNormBp" + S)(extra(A, g("dzi", A), g("dxi", A)), P, A.ctypes.data, P, g("mean"), g("inv"), g("dz"), A.ctypes.data,
                                                g("dx"), A.ctypes.data, g("dg"), g("db"), g("w", None), g("wb", 0))


@pytest.mark.parametrize("S", SUFFIXES)
@pytest.mark.parametrize("why,args", [
    ("negative number", {"n": -1}), ("not a row of the table's length", {"n": 5}), ("not a row of the table's length", {"zi": B}),
    ("table is null", {"t": None}), ("tokens is null", {"k": None}), ("z is null", {"z": None}), ("not aligned", {"k": P + 4})])
def test_embedding(ops, S, why, args):
    g = lambda key, other=P: args.get(key, other)  # noqa: E731
    with pytest.raises(Nd4jError, match=why):
        getattr(ops, "amd_execEmbedding" + S)(extra(x=info(50, 8), z=g("zi", A)), g("t"), None, g("k"), g("n", 4), g("z"), None, 1.0)


@pytest.mark.parametrize("S", SUFFIXES)
@pytest.mark.parametrize("why,args", [
    ("negative number", {"n": -1}), ("not a row of the table's length", {"n": 5}), ("not a row of the table's length", {"dzi": B}),
    ("dTable is null", {"t": None}), ("tokens is null", {"k": None}), ("dz is null", {"dz": None}), ("2\\^31 - 2\\^20 tokens", {"n": 1 << 31, "dzi": info(1 << 31, 8)}),
    ("2\\^31 - 2\\^20 tokens", {"ti": info(1 << 31, 8)}), ("too many elements", {"n": 1 << 30, "dzi": info(1 << 30, 1 << 20), "ti": info(50, 1 << 20)}),
    ("scratch holds", {"w": P, "wb": 8}), ("not aligned to 16", {"w": P + 8, "wb": 1 << 40})])
def test_embedding_bp(ops, S, why, args):
    g = lambda key, other=P: args.get(key, other)  # noqa: E731
    with pytest.raises(Nd4jError, match=why):
        getattr(ops, "amd_execEmbeddingBp" + S)(extra(x=g("dzi", A), z=g("ti", info(50, 8))), g("dz"), None, g("k"), g("n", 4), g("t"), None, 1.0, 0,
                                                g("w", None), g("wb", 0))


@pytest.mark.parametrize("S", SUFFIXES)
@pytest.mark.parametrize("why,args", [
    ("between 0 and 64", {"n": -1}), ("between 0 and 64", {"n": 65, "xi": info(4, 100)}), ("more alternatives", {"n": 9}), ("x is null", {"x": None}),
    ("tokens is null", {"t": None}), ("topTokens is null", {"top": None}), ("no result", {"lp": None, "ls": None, "h": None, "n": 0}),
    ("not aligned", {"ls": P + 2}), ("not aligned", {"top": P + 4}), ("without elements", {"xi": EMPTY})])
def test_token_log_probs(ops, S, why, args):
    g = lambda key, other=P: args.get(key, other)  # noqa: E731
    with pytest.raises(Nd4jError, match=why):
        getattr(ops, "amd_execTokenLogProbs" + S)(extra(x=g("xi", A)), g("x"), None, g("t"), g("lp"), g("ls"), g("h"), g("n", 3), g("top"), P, None, 0)


@pytest.mark.parametrize("S", SUFFIXES)
@pytest.mark.parametrize("why,args", [
    ("differ in shape", {"dxi": B}), ("neither", {"a": None, "b": None}), ("logSum is null", {"ls": None}), ("dx is null", {"dx": None}),
    ("tokens is null", {"t": None}), ("entropy is null", {"h": None}), ("not aligned", {"a": P + 2})])
def test_token_log_probs_bp(ops, S, why, args):
    g = lambda key, other=P: args.get(key, other)  # noqa: E731
    with pytest.raises(Nd4jError, match=why):
        getattr(ops, "amd_execTokenLogProbsBp" + S)(extra(x=A, z=g("dxi", A)), P, None, g("t"), g("ls"), g("h"), g("a"), g("b"), g("dx"), None)


@pytest.mark.parametrize("S", SUFFIXES)
@pytest.mark.parametrize("why,args", [
    ("negative number", {"n": -1}), ("negative number", {"total": -1}), ("greater than 0", {"most": 0.0}), ("greater than 0", {"most": float("nan")}),
    ("no result", {"dz": None, "norm": None}), ("elements without", {"n": 0}), ("table of tensors is null", {"dx": None}),
    ("offsets is null", {"o": None}), ("scratch holds", {"w": P, "wb": 8}), ("not aligned", {"norm": P + 2})])
def test_clip_by_global_norm(ops, S, why, args):
    g = lambda key, other=P: args.get(key, other)  # noqa: E731
    with pytest.raises(Nd4jError, match=why):
        getattr(ops, "amd_execClipByGlobalNorm" + S)(extra(), g("dx"), g("dz"), g("o"), g("n", 3), g("total", 100), g("most", 1.0), g("norm"),
                                                     g("w", None), g("wb", 0))


@pytest.mark.parametrize("S", SUFFIXES)
@pytest.mark.parametrize("strides", [[0, 1], [8, 0], [0, 0], [1, 1], [7, 1], [2, 4], [-2, 6], [1, 3]])
def test_results_whose_elements_share_places(ops, S, strides):
    shared, whole = info(4, 8, strides=strides), info(4, 8)
    with pytest.raises(Nd4jError, match="share places"):
        getattr(ops, "amd_execLayerNorm" + S)(extra(x=whole, z=shared), P, None, P, P, P, None, P, P, 1e-5)
    with pytest.raises(Nd4jError, match="share places"):
        getattr(ops, "amd_execLayerNormBp" + S)(extra(whole, whole, shared), P, None, P, P, P, P, None, P, None, P, P, None, 0)
    with pytest.raises(Nd4jError, match="share places"):
        getattr(ops, "amd_execEmbedding" + S)(extra(x=whole, z=shared), P, None, P, 4, P, None, 1.0)
    with pytest.raises(Nd4jError, match="share places"):
        getattr(ops, "amd_execEmbeddingBp" + S)(extra(x=whole, z=shared), P, None, P, 4, P, None, 1.0, 0, None, 0)
    with pytest.raises(Nd4jError, match="share places"):
        getattr(ops, "amd_execTokenLogProbsBp" + S)(extra(x=whole, z=shared), P, None, P, P, P, P, P, P, None)


@pytest.mark.parametrize("S", SUFFIXES)
@pytest.mark.parametrize("strides", [[8, 1], [1, 4], [9, 1], [-8, 1], [8, -1], [1, 5], [16, 2], [3, 4]])
def test_results_whose_elements_do_not(ops, S, strides):
    """refused for another reason, which is looked at later"""
    with pytest.raises(Nd4jError, match="x is null"):
        getattr(ops, "amd_execLayerNorm" + S)(extra(x=info(4, 8), z=info(4, 8, strides=strides)), None, None, P, P, P, None, P, P, 1e-5)


def test_scratch_sizes(ops):
    assert ops.amd_scratchLayerNormBp(0, 1) > 0
    assert ops.amd_scratchLayerNormBp(16384, 1024) < 1 << 26
    assert ops.amd_scratchEmbeddingBp(16384, 32000, 768) < 1 << 26
    assert ops.amd_scratchTokenLogProbs(4096, 32000, 5) >= 0
    assert ops.amd_scratchClipByGlobalNorm(0) > 0
    for call, args in ((ops.amd_scratchLayerNormBp, (-1, 5)), (ops.amd_scratchLayerNormBp, (5, 0)), (ops.amd_scratchEmbeddingBp, (1 << 31, 5, 5)),
                       (ops.amd_scratchEmbeddingBp, (5, -1, 5)), (ops.amd_scratchTokenLogProbs, (5, 5, 65)), (ops.amd_scratchClipByGlobalNorm, (-1,))):
        with pytest.raises(Nd4jError):
            call(*args)


def test_empty_calls_do_nothing(ops):
    """no rows, no tokens: nothing to compute, and nothing is enqueued (there is no GPU here to enqueue it on)"""
    none = info(0, 8)
    for S in SUFFIXES:
        getattr(ops, "amd_execLayerNorm" + S)(extra(x=none, z=none), None, None, None, None, None, None, None, None, 1e-5)
        getattr(ops, "amd_execLayerNormBp" + S)(extra(none, none, none), None, None, None, None, None, None, None, P, None, None, None, None, 0)
        getattr(ops, "amd_execEmbedding" + S)(extra(x=A), None, None, None, 0, None, None, 1.0)
        getattr(ops, "amd_execEmbeddingBp" + S)(extra(x=none, z=A), None, None, None, 0, P, None, 1.0, 1, None, 0)
        getattr(ops, "amd_execTokenLogProbs" + S)(extra(x=none), None, None, None, None, None, None, 2, None, None, None, 0)
        getattr(ops, "amd_execTokenLogProbsBp" + S)(extra(x=none, z=none), None, None, None, None, None, P, None, None, None)
    assert np.array_equal(A, info(4, 8))
