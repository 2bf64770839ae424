"""The operators around a language model's matrix products over views that run backwards or repeat elements, over vectors and scratch
that begin anywhere they may, against 64-bit results."""
import numpy as np
import pytest

from libnd4j_amd import harness
from test_training_ops import (bp_inputs, check_token_probs, embedding_bp_oracle, layer_norm_bp_oracle, layer_norm_oracle, token_probs_bp_oracle,
                               token_probs_oracle)
from training_views import COMPUTE, STORAGE, SUFFIXES, Vec, close, extra

pytestmark = pytest.mark.gpu

READ = {"rows backwards": (-1, 1, 0), "elements backwards": (1, -1, 0), "both backwards": (-1, -1, 3), "one row": (0, 1, 0), "one column": (1, 0, 0),
        "one element": (0, 0, 0), "f backwards": ("f", -1, 0)}
WRITTEN = ("rows backwards", "elements backwards", "both backwards", "f backwards")


@pytest.fixture(scope="module")
def dev():
    return harness.Device()


class Strided(object):
    """Rows in a buffer by strides of any sign: row and element as multiples of those of a matrix with `pad` elements between rows"""

    def __init__(self, dev, kind, rows, length, dtype, values=None):
        self.dev, self.dtype, self.rows, self.length = dev, np.dtype(dtype), rows, length
        row, el, pad = READ[kind]
        if row == "f":
            row, el = -1, -rows
        else:
            row *= length + pad
        size = abs(row) * max(rows - 1, 0) + abs(el) * (length - 1) + 1
        self.start = 5 + (abs(row) * (rows - 1) if row < 0 else 0) + (abs(el) * (length - 1) if el < 0 else 0)
        self.strides = (row, el)
        self.host = np.full(size + 10, 77, dtype=self.dtype)
        if values is not None:
            self.at(self.host)[...] = values
        self.info = harness.shape_info([rows, length], strides=[row, el], order="c")
        self.buf = dev.upload(self.host)
        self.ptr = self.buf.ptr + self.start * self.dtype.itemsize

    def at(self, host):
        return np.lib.stride_tricks.as_strided(host[self.start:], shape=(self.rows, self.length), strides=[s * self.dtype.itemsize for s in self.strides])

    def values(self):
        return self.at(self.host).copy()

    def get(self):
        now = self.buf.download(self.dtype, self.host.size)
        got, around = self.at(now).copy(), self.host.copy()
        self.at(now)[...] = 0
        self.at(around)[...] = 0
        assert np.array_equal(now, around), "elements outside the view were written"
        return got


class Off(object):
    """A dense vector one element behind a 16-byte boundary"""

    def __init__(self, dev, values, dtype):
        self.v = Vec(dev, np.concatenate([np.full(1, 77), np.asarray(values).reshape(-1)]), dtype)
        self.ptr = self.v.ptr + np.dtype(dtype).itemsize

    def get(self):
        whole = self.v.get()
        assert whole[0] == 77
        return whole[1:]


def scratch(dev, size):
    buf = dev.empty(size + 16)
    return buf.ptr + 16, size


@pytest.mark.parametrize("S", SUFFIXES)
@pytest.mark.parametrize("kx", sorted(READ))
@pytest.mark.parametrize("kz", WRITTEN)
def test_layer_norm(dev, S, kx, kz):
    T, C = STORAGE[S], COMPUTE[S]
    rs = np.random.RandomState(1)
    for rows, n in ((5, 33), (66, 300), (3, 2050)):
        X, Z = Strided(dev, kx, rows, n, T, rs.randn(rows, n)), Strided(dev, kz, rows, n, T)
        gain, bias = (1 + rs.randn(n) / 8).astype(T), (rs.randn(n) / 8).astype(T)
        G, B, M, I = Off(dev, gain, T), Off(dev, bias, T), Off(dev, np.zeros(rows), C), Off(dev, np.zeros(rows), C)
        getattr(dev.ops, "amd_execLayerNorm" + S)(extra(dev, x=X, z=Z), X.ptr, None, G.ptr, B.ptr, Z.ptr, None, M.ptr, I.ptr, 1e-3)
        want, want_mean, want_inv, tol, tol_mean, tol_inv = layer_norm_oracle(X.values(), gain, bias, 1e-3, S)
        close(Z.get(), want, tol)
        close(M.get(), want_mean, tol_mean)
        close(I.get(), want_inv, tol_inv)


@pytest.mark.parametrize("S", SUFFIXES)
@pytest.mark.parametrize("kx", sorted(READ))
@pytest.mark.parametrize("kdz,kdx", [("rows backwards", "elements backwards"), ("one row", "rows backwards"), ("both backwards", "both backwards"),
                                     ("f backwards", "f backwards"), ("one column", "rows backwards")])
def test_layer_norm_bp(dev, S, kx, kdz, kdx):
    T, C = STORAGE[S], COMPUTE[S]
    for rows, n in ((5, 33), (66, 300), (3, 2050)):
        x, gain, _, _, dz = bp_inputs(S, rows, n, 4)
        X, DZ, DX = Strided(dev, kx, rows, n, T, x), Strided(dev, kdz, rows, n, T, dz), Strided(dev, kdx, rows, n, T)
        x, dz = X.values(), DZ.values()
        mean, inv = x.astype(np.float64).mean(1).astype(C), (1 / np.sqrt(x.astype(np.float64).var(1) + 1e-2)).astype(C)
        G, M, I, DG, DB = Off(dev, gain, T), Off(dev, mean, C), Off(dev, inv, C), Off(dev, np.zeros(n), T), Off(dev, np.zeros(n), T)
        getattr(dev.ops, "amd_execLayerNormBp" + S)(extra(dev, x=X, y=DZ, z=DX), X.ptr, None, G.ptr, M.ptr, I.ptr, DZ.ptr, None, DX.ptr, None, DG.ptr,
                                                    DB.ptr, *scratch(dev, dev.ops.amd_scratchLayerNormBp(rows, n)))
        want = layer_norm_bp_oracle(x, gain, mean, inv, dz, S)
        for k, got in enumerate((DX.get(), DG.get(), DB.get())):
            close(got, want[k], want[3 + k], ("dx", "dGain", "dBias")[k])


@pytest.mark.parametrize("S", SUFFIXES)
@pytest.mark.parametrize("kt", sorted(READ))
@pytest.mark.parametrize("kz", WRITTEN)
def test_embedding(dev, S, kt, kz):
    T, C = STORAGE[S], COMPUTE[S]
    rs = np.random.RandomState(2)
    for count, n in ((40, 33), (130, 515)):
        W, Z = Strided(dev, kt, 20, n, T, rs.randn(20, n)), Strided(dev, kz, count, n, T)
        tokens = rs.randint(-2, 23, count)
        K = Off(dev, tokens, np.int64)
        getattr(dev.ops, "amd_execEmbedding" + S)(extra(dev, x=W, z=Z), W.ptr, None, K.ptr, count, Z.ptr, None, 1.7)
        want = (W.values().astype(C)[np.clip(tokens, 0, 19)] * C(1.7)).astype(T)
        want[tokens < 0] = 0
        want[tokens >= 20] = np.nan
        assert np.array_equal(Z.get(), want, equal_nan=True)


@pytest.mark.parametrize("S", SUFFIXES)
@pytest.mark.parametrize("kdz", sorted(READ))
@pytest.mark.parametrize("kt", WRITTEN)
@pytest.mark.parametrize("add", (False, True))
def test_embedding_bp(dev, S, kdz, kt, add):
    T = STORAGE[S]
    rs = np.random.RandomState(3)
    for count, n in ((40, 33), (300, 130)):
        into = rs.randn(20, n).astype(T)
        DZ, W = Strided(dev, kdz, count, n, T, rs.randn(count, n)), Strided(dev, kt, 20, n, T, into)
        tokens = rs.randint(-2, 15, count)
        K = Off(dev, tokens, np.int64)
        getattr(dev.ops, "amd_execEmbeddingBp" + S)(extra(dev, x=DZ, z=W), DZ.ptr, None, K.ptr, count, W.ptr, None, 0.5, 1 if add else 0,
                                                    *scratch(dev, dev.ops.amd_scratchEmbeddingBp(count, 20, n)))
        want, tol = embedding_bp_oracle(DZ.values(), tokens, 20, 0.5, into if add else None, S)
        close(W.get(), want, tol)


@pytest.mark.parametrize("S", SUFFIXES)
@pytest.mark.parametrize("kx", sorted(READ))
@pytest.mark.parametrize("kdx", WRITTEN)
def test_token_log_probs_and_gradient(dev, S, kx, kdx):
    T, C = STORAGE[S], COMPUTE[S]
    rs = np.random.RandomState(4)
    for rows, n, k in ((5, 33, 5), (70, 300, 3), (2, 5003, 17)):
        X, DX = Strided(dev, kx, rows, n, T, rs.randn(rows, n) * 3), Strided(dev, kdx, rows, n, T)
        x, tokens = X.values(), rs.randint(0, n, rows)
        tokens[0] = -1
        K = Off(dev, tokens, np.int64)
        lp, ls, h, a, b = (Off(dev, rs.randn(rows) / 4, C) for _ in range(5))
        top, top_lp = Off(dev, np.zeros(rows * k), np.int64), Off(dev, np.zeros(rows * k), C)
        av, bv = a.get().copy(), b.get().copy()
        size = dev.ops.amd_scratchTokenLogProbs(rows, n, k)
        getattr(dev.ops, "amd_execTokenLogProbs" + S)(extra(dev, x=X), X.ptr, None, K.ptr, lp.ptr, ls.ptr, h.ptr, k, top.ptr, top_lp.ptr,
                                                      *(scratch(dev, size) if size else (None, 0)))
        got = {"lp": lp.get(), "ls": ls.get(), "h": h.get(), "top": top.get().reshape(rows, k), "top_lp": top_lp.get().reshape(rows, k)}
        check_token_probs(got, token_probs_oracle(x, tokens, k, S))
        getattr(dev.ops, "amd_execTokenLogProbsBp" + S)(extra(dev, x=X, z=DX), X.ptr, None, K.ptr, ls.ptr, h.ptr, a.ptr, b.ptr, DX.ptr, None)
        want, tol = token_probs_bp_oracle(x, tokens, ls.get(), h.get(), av, bv, S)
        close(DX.get(), want, tol)
