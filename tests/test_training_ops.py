"""The operators around a language model's matrix products - layer norm, embedding, log probabilities of tokens, clipping
by the global norm, forward and backward - against their formulas in 64 bits, over types, lengths, layouts and masks.

Tolerances count roundings.  u is half a step of the compute type.  A sum of n terms that at least 64 lanes share (or 16
lanes with at most 32 terms each) takes at most n / 64 + 32 roundings a term, written N(n); any order of n terms takes at
most n.  A stored result adds one rounding to its own type (`unit`, and `smallest` where it is subnormal)."""
import numpy as np
import pytest

from libnd4j_amd import harness
from training_views import COMPUTE, LAYOUTS, STORAGE, SUFFIXES, Vec, View, close, extra, smallest, unit

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return harness.Device()


def N(n):
    return n / 64.0 + 32.0


def stored(value, S):
    return unit(STORAGE[S]) * np.abs(value) + smallest(STORAGE[S])


# ---- layer norm --------------------------------------------------------------------------------------------------------

def layer_norm_oracle(x, gain, bias, eps, S):
    x = x.astype(np.float64)
    n = x.shape[1]
    u = unit(COMPUTE[S])
    mean = x.mean(1, keepdims=True)
    d = x - mean
    s = 1.0 / np.sqrt((d * d).mean(1, keepdims=True) + eps)
    h = d * s
    g = np.ones(n) if gain is None else gain.astype(np.float64)
    b = np.zeros(n) if bias is None else bias.astype(np.float64)
    z = h * g + b
    d_mean = N(n) * u * np.abs(x).mean(1, keepdims=True) + u * np.abs(mean)
    d_h = s * (d_mean + u * np.abs(d)) + np.abs(h) * (N(n) + 8) * u + s * s * d_mean * d_mean * np.abs(h)
    tol_z = np.abs(g) * d_h + 4 * u * (np.abs(h * g) + np.abs(b))
    tol_s = s * ((N(n) + 8) * u + s * s * d_mean * d_mean)
    return z, mean[:, 0], s[:, 0], tol_z + stored(z, S), d_mean[:, 0], tol_s[:, 0]


def run_layer_norm(dev, S, x, gain, bias, eps, lx="dense", lz="dense", stats=True, inplace=False):
    T, C = STORAGE[S], COMPUTE[S]
    rows, n = x.shape
    X = View(dev, rows, n, lx, T, x)
    Z = X if inplace else View(dev, rows, n, lz, T)
    G, B = (None if v is None else Vec(dev, v, T) for v in (gain, bias))
    M, I = (Vec(dev, np.zeros(rows), C) if stats else None for _ in range(2))
    getattr(dev.ops, "amd_execLayerNorm" + S)(extra(dev, x=X, z=Z), X.ptr, X.info_ptr, G and G.ptr, B and B.ptr, Z.ptr, Z.info_ptr,
                                              M and M.ptr, I and I.ptr, eps)
    out = Z.get(), M and M.get(), I and I.get()
    for v in (X, Z, G, B, M, I):
        if v is not None:
            v.free()
    return out


LENGTHS = (1, 2, 3, 7, 8, 16, 31, 64, 65, 100, 128, 255, 256, 257, 511, 512, 768, 1000, 1023, 1024, 1025, 2047, 2048, 2049, 4095, 4096, 4097,
           5003, 8191, 8192, 8193, 16384, 16385, 32768, 32769, 70001)


@pytest.mark.parametrize("S", SUFFIXES)
@pytest.mark.parametrize("n", LENGTHS)
def test_layer_norm_lengths(dev, S, n):
    rs = np.random.RandomState(n)
    for rows in (1, 5) if n > 300 else (1, 4, 131):
        x = (rs.randn(rows, n) * 3 + 1).astype(STORAGE[S])
        gain, bias = (1 + rs.randn(n) / 8).astype(STORAGE[S]), (rs.randn(n) / 8).astype(STORAGE[S])
        z, mean, inv = run_layer_norm(dev, S, x, gain, bias, 1e-5)
        want, want_mean, want_inv, tol, tol_mean, tol_inv = layer_norm_oracle(x, gain, bias, 1e-5, S)
        close(z, want, tol, "z")
        close(mean, want_mean, tol_mean, "mean")
        close(inv, want_inv, tol_inv, "invStd")


@pytest.mark.parametrize("S", SUFFIXES)
@pytest.mark.parametrize("lx", LAYOUTS)
@pytest.mark.parametrize("lz", ("dense", "pitch3", "forder", "inner2"))
def test_layer_norm_layouts(dev, S, lx, lz):
    rs = np.random.RandomState(3)
    for rows, n in ((6, 40), (70, 129), (2, 1030)):
        x = rs.randn(rows, n).astype(STORAGE[S])
        gain = (1 + rs.randn(n) / 8).astype(STORAGE[S])
        z, mean, inv = run_layer_norm(dev, S, x, gain, None, 1e-3, lx, lz)
        want, _, _, tol, _, _ = layer_norm_oracle(x, gain, None, 1e-3, S)
        close(z, want, tol, "z")


@pytest.mark.parametrize("S", SUFFIXES)
def test_layer_norm_of_extremes(dev, S):
    """constant rows, rows far from zero, large values, no gain and bias, no statistics, in place, many rows"""
    rs = np.random.RandomState(4)
    n = 384
    big = 1e4 if S == "Half" else 1e15
    x = np.stack([np.zeros(n), np.full(n, 7.25), rs.randn(n) + 500, rs.randn(n) * big, rs.randn(n) * 1e-3]).astype(STORAGE[S])
    z, mean, inv = run_layer_norm(dev, S, x, None, None, 1e-5)
    want, want_mean, want_inv, tol, tol_mean, tol_inv = layer_norm_oracle(x, None, None, 1e-5, S)
    close(z, want, tol, "z")
    close(mean, want_mean, tol_mean, "mean")
    close(inv, want_inv, tol_inv, "invStd")
    same, _, _ = run_layer_norm(dev, S, x, None, None, 1e-5, stats=False, inplace=True)
    assert np.array_equal(same, z)
    for rows, n in ((20011, 24), (5000, 300)):
        x = rs.randn(rows, n).astype(STORAGE[S])
        z, _, _ = run_layer_norm(dev, S, x, None, None, 1e-5)
        want, _, _, tol, _, _ = layer_norm_oracle(x, None, None, 1e-5, S)
        close(z, want, tol, "z")


def test_layer_norm_of_nan_and_infinity(dev):
    x = np.random.RandomState(1).randn(5, 300).astype(np.float32)
    x[1, 7] = np.nan
    x[3, 299] = np.inf
    z, _, _ = run_layer_norm(dev, "Float", x, None, None, 1e-5)
    assert np.isnan(z[1]).all() and np.isnan(z[3]).all()
    assert np.isfinite(z[[0, 2, 4]]).all()


def layer_norm_bp_oracle(x, gain, mean, inv, dz, S):
    x, dz = x.astype(np.float64), dz.astype(np.float64)
    rows, n = x.shape
    u = unit(COMPUTE[S])
    s = inv.astype(np.float64)[:, None]
    h = (x - mean.astype(np.float64)[:, None]) * s
    g = np.ones(n) if gain is None else gain.astype(np.float64)
    a = dz * g
    c1, c2 = a.mean(1, keepdims=True), (a * h).mean(1, keepdims=True)
    dx = s * (a - c1 - h * c2)
    d_h = 3 * u * np.abs(h)
    d_c1 = (N(n) + 2) * u * np.abs(a).mean(1, keepdims=True)
    d_c2 = (N(n) + 6) * u * np.abs(a * h).mean(1, keepdims=True)
    tol_dx = s * (d_c1 + np.abs(h) * d_c2 + np.abs(c2) * d_h + 6 * u * (np.abs(a) + np.abs(c1) + np.abs(h * c2)))
    d_gain, d_bias = (dz * h).sum(0), dz.sum(0)
    tol_gain = (rows + 6) * u * np.abs(dz * h).sum(0)
    tol_bias = (rows + 2) * u * np.abs(dz).sum(0)
    return dx, d_gain, d_bias, tol_dx + stored(dx, S), tol_gain + stored(d_gain, S), tol_bias + stored(d_bias, S)


def run_layer_norm_bp(dev, S, x, gain, mean, inv, dz, lx="dense", ldz="dense", ldx="dense", wants=("dx", "dGain", "dBias"), inplace=None,
                      scratch=None):
    T, C = STORAGE[S], COMPUTE[S]
    rows, n = x.shape
    X, DZ = View(dev, rows, n, lx, T, x), View(dev, rows, n, ldz, T, dz)
    DX = {"dz": DZ, "x": X, None: None}[inplace] or View(dev, rows, n, ldx, T)
    G = None if gain is None else Vec(dev, gain, T)
    M, I = Vec(dev, mean, C), Vec(dev, inv, C)
    DG, DB = Vec(dev, np.full(n, 9.0), T), Vec(dev, np.full(n, 9.0), T)
    bytes_ = dev.ops.amd_scratchLayerNormBp(rows, n) if scratch else 0
    W = dev.empty(bytes_) if scratch else None
    getattr(dev.ops, "amd_execLayerNormBp" + S)(
        extra(dev, x=X, y=DZ, z=DX), X.ptr, X.info_ptr, G and G.ptr, M.ptr, I.ptr, DZ.ptr, DZ.info_ptr, DX.ptr if "dx" in wants else None,
        DX.info_ptr, DG.ptr if "dGain" in wants else None, DB.ptr if "dBias" in wants else None, W and W.ptr, bytes_)
    out = DX.get(), DG.get(), DB.get()
    for v in (X, DZ, DX, G, M, I, DG, DB, W):
        if v is not None:
            v.free()
    return out


def bp_inputs(S, rows, n, seed):
    rs = np.random.RandomState(seed)
    T, C = STORAGE[S], COMPUTE[S]
    x = (rs.randn(rows, n) * 2 + 0.5).astype(T)
    gain = (1 + rs.randn(n) / 8).astype(T)
    mean = x.astype(np.float64).mean(1).astype(C)
    inv = (1 / np.sqrt(x.astype(np.float64).var(1) + 1e-5)).astype(C)
    return x, gain, mean, inv, (rs.randn(rows, n) / 4).astype(T)


@pytest.mark.parametrize("S", SUFFIXES)
@pytest.mark.parametrize("n", LENGTHS)
def test_layer_norm_bp_lengths(dev, S, n):
    for rows in (1, 37) if n > 300 else (1, 4, 1031):
        args = bp_inputs(S, rows, n, n + rows)
        got = run_layer_norm_bp(dev, S, *args)
        want = layer_norm_bp_oracle(*args, S)
        for k, name in enumerate(("dx", "dGain", "dBias")):
            close(got[k], want[k], want[3 + k], "%s of [%d, %d]" % (name, rows, n))


@pytest.mark.parametrize("S", SUFFIXES)
@pytest.mark.parametrize("lx,ldz,ldx", [("pitch8", "dense", "pitch3"), ("pitch3", "offset1", "dense"), ("rank3", "pitch8", "rank3"),
                                        ("forder", "forder", "forder"), ("inner2", "dense", "forder"), ("dense", "forder", "inner2"),
                                        ("offset1", "pitch3", "offset1")])
def test_layer_norm_bp_layouts(dev, S, lx, ldz, ldx):
    for rows, n in ((6, 40), (130, 129), (2, 1030), (8, 4500)):
        args = bp_inputs(S, rows, n, 5)
        got = run_layer_norm_bp(dev, S, *args, lx=lx, ldz=ldz, ldx=ldx, scratch=True)
        want = layer_norm_bp_oracle(*args, S)
        for k, name in enumerate(("dx", "dGain", "dBias")):
            close(got[k], want[k], want[3 + k], name)


@pytest.mark.parametrize("S", SUFFIXES)
@pytest.mark.parametrize("rows,n", [(300, 257), (70, 5003), (4, 40000)])
def test_layer_norm_bp_parts_and_in_place(dev, S, rows, n):
    args = bp_inputs(S, rows, n, 8)
    whole = run_layer_norm_bp(dev, S, *args)
    for wants in (("dx",), ("dGain",), ("dBias",), ("dx", "dBias"), ("dGain", "dBias")):
        got = run_layer_norm_bp(dev, S, *args, wants=wants)
        for k, name in enumerate(("dx", "dGain", "dBias")):
            if name in wants:
                assert np.array_equal(got[k], whole[k]), (wants, name)
            else:
                assert (got[k] == (View.SENTINEL if k == 0 else 9.0)).all(), (wants, name)
    for where in ("dz", "x"):
        got = run_layer_norm_bp(dev, S, *args, inplace=where)
        for k in range(3):
            assert np.array_equal(got[k], whole[k]), (where, k)
    x, _, mean, inv, dz = args
    got = run_layer_norm_bp(dev, S, x, None, mean, inv, dz)
    want = layer_norm_bp_oracle(x, None, mean, inv, dz, S)
    for k in range(3):
        close(got[k], want[k], want[3 + k])


@pytest.mark.parametrize("S", SUFFIXES)
@pytest.mark.parametrize("n", (40, 300, 5003))
def test_layer_norm_bp_of_nan_infinity_and_overflow(dev, S, n):
    """a row's NaN and infinities stay in the row, and come out as the formula has them; so does what passes the type's range"""
    x, gain, mean, inv, dz = bp_inputs(S, 9, n, 3)
    dz[1, 5] = np.nan
    dz[2, n - 1] = np.inf
    x[3, 7] = np.nan
    inv[4] = 0
    inv[5] = np.nan
    inv[6] = 1e6  # beyond a half's range in every element of dx, and far inside a float's
    x[7, 0] = -np.inf
    for g in (gain, None):
        got = run_layer_norm_bp(dev, S, x, g, mean, inv, dz, wants=("dx",))[0]
        with np.errstate(all="ignore"):
            want, _, _, tol, _, _ = layer_norm_bp_oracle(x, g, mean, inv, dz, S)
            rounded = want.astype(STORAGE[S])
        assert np.array_equal(np.isnan(got), np.isnan(rounded))
        if S == "Half":
            assert (got[np.isnan(got)].view(np.uint16) == 0x7fff).all()
        far = np.isinf(rounded) & np.isinf(got)
        assert np.array_equal(got[far], rounded[far])
        near = ~far & ~np.isnan(rounded)
        near[6] &= S != "Half"  # (the row that the half rounds to infinity but near zeros of dx)
        assert not np.isinf(got[near]).any()
        close(got[near], want[near], tol[near])
        assert np.isnan(got[1]).all() and not got[4].any() and np.isfinite(got[[0, 8]]).all()
        assert np.isinf(got[6]).any() == (S == "Half")


def test_layer_norm_bp_without_rows(dev):
    x = np.zeros((0, 33), np.float32)
    got = run_layer_norm_bp(dev, "Float", x, None, np.zeros(0), np.zeros(0), x)
    assert not got[1].any() and not got[2].any()


def test_layer_norm_gradient_against_differences(dev):
    """double: the loss sum(z w) changes with x, gain and bias as the backward call says (central differences: an error of
    order h^2 and one of order eps / h, both below 1e-7 for h = 1e-4 and values of order 1)"""
    rs = np.random.RandomState(11)
    rows, n, eps, h = 3, 17, 1e-5, 1e-4
    x, gain, bias, w = rs.randn(rows, n), 1 + rs.randn(n) / 8, rs.randn(n), rs.randn(rows, n)

    def loss(x, gain, bias):
        return float((run_layer_norm(dev, "Double", x, gain, bias, eps)[0] * w).sum())

    _, mean, inv = run_layer_norm(dev, "Double", x, gain, bias, eps)
    dx, d_gain, d_bias = run_layer_norm_bp(dev, "Double", x, gain, mean, inv, w)
    for k in range(0, n, 5):
        for what, grad in (("x", dx[1, k]), ("gain", d_gain[k]), ("bias", d_bias[k])):
            up, down = [[v.copy() for v in (x, gain, bias)] for _ in range(2)]
            i = ("x", "gain", "bias").index(what)
            at = (1, k) if i == 0 else k
            up[i][at] += h
            down[i][at] -= h
            assert abs((loss(*up) - loss(*down)) / (2 * h) - grad) < 1e-6, (what, k)


# ---- embedding ---------------------------------------------------------------------------------------------------------

def run_embedding(dev, S, table, tokens, scale, lt="dense", lz="dense"):
    T = STORAGE[S]
    v, n = table.shape
    W, K = View(dev, v, n, lt, T, table), Vec(dev, tokens, np.int64)
    Z = View(dev, len(tokens), n, lz, T)
    getattr(dev.ops, "amd_execEmbedding" + S)(extra(dev, x=W, z=Z), W.ptr, W.info_ptr, K.ptr, len(tokens), Z.ptr, Z.info_ptr, scale)
    out = Z.get()
    for o in (W, K, Z):
        o.free()
    return out


@pytest.mark.parametrize("S", SUFFIXES)
@pytest.mark.parametrize("n", (1, 2, 7, 8, 9, 64, 65, 100, 512, 1023, 2048, 5003))
def test_embedding(dev, S, n):
    rs = np.random.RandomState(n)
    T, C = STORAGE[S], COMPUTE[S]
    for count, lt, lz in ((1, "dense", "dense"), (257, "dense", "pitch3"), (300, "pitch8", "rank3"), (64, "forder", "dense"),
                          (33, "offset1", "forder"), (30, "inner2", "offset1"), (2100, "pitch3", "dense")):
        table = rs.randn(91, n).astype(T)
        tokens = rs.randint(0, 91, count)
        tokens[::7] = -1
        tokens[1::11] = 91
        tokens[2::13] = 1 << 40
        tokens[3::17] = -(1 << 40)
        got = run_embedding(dev, S, table, tokens, 1.7, lt, lz)
        want = (table.astype(C)[np.clip(tokens, 0, 90)] * C(1.7)).astype(T)  # one product, one rounding: the same bits
        want[tokens < 0] = 0
        want[tokens >= 91] = np.nan
        assert np.array_equal(got, want, equal_nan=True)


def run_embedding_bp(dev, S, dz, tokens, vocabulary, scale, into=None, ldz="dense", lt="dense", scratch=False):
    T = STORAGE[S]
    count, n = dz.shape
    DZ, K = View(dev, count, n, ldz, T, dz), Vec(dev, tokens, np.int64)
    W = View(dev, vocabulary, n, lt, T, np.full((vocabulary, n), 5.0) if into is None else into)
    bytes_ = dev.ops.amd_scratchEmbeddingBp(count, vocabulary, n) if scratch else 0
    M = dev.empty(bytes_) if scratch else None
    getattr(dev.ops, "amd_execEmbeddingBp" + S)(extra(dev, x=DZ, z=W), DZ.ptr, DZ.info_ptr, K.ptr, count, W.ptr, W.info_ptr, scale,
                                                0 if into is None else 1, M and M.ptr, bytes_)
    out = W.get()
    for o in (DZ, K, W, M):
        if o is not None:
            o.free()
    return out


def embedding_bp_oracle(dz, tokens, vocabulary, scale, into, S):
    u = unit(COMPUTE[S])
    live = (tokens >= 0) & (tokens < vocabulary)
    want, size = (np.zeros((vocabulary, dz.shape[1])) for _ in range(2))
    np.add.at(want, tokens[live], dz.astype(np.float64)[live] * scale)
    np.add.at(size, tokens[live], np.abs(dz.astype(np.float64)[live] * scale))
    count = np.bincount(tokens[live], minlength=vocabulary)[:, None]
    tol = (count + 4) * u * size
    if into is not None:
        want += into.astype(np.float64)
        tol = np.where(count > 0, tol + u * np.abs(want), 0)
    return want, np.where(count > 0, tol + stored(want, S), 0)


def skewed(rs, count, vocabulary, kind):
    if kind == "one":
        return np.full(count, vocabulary // 2)
    if kind == "spread":
        return rs.randint(0, vocabulary, count)
    if kind == "runs":
        return np.sort(rs.randint(0, max(1, vocabulary // 3), count))
    t = np.minimum((vocabulary + 1.0) ** rs.rand(count), vocabulary).astype(np.int64) - 1
    t[rs.rand(count) < 0.1] = -1
    t[rs.rand(count) < 0.05] = vocabulary
    return t


@pytest.mark.parametrize("S", SUFFIXES)
@pytest.mark.parametrize("kind", ("one", "spread", "runs", "text"))
@pytest.mark.parametrize("count,vocabulary,n", [(1, 1, 1), (1, 300, 65), (15, 7, 3), (16, 256, 8), (17, 257, 64), (255, 1000, 33), (1024, 70, 256),
                                                (1025, 65536, 5), (4096, 65537, 4), (5000, 300, 129), (20000, 5000, 7), (70000, 40, 12)])
def test_embedding_bp(dev, S, kind, count, vocabulary, n):
    rs = np.random.RandomState(count + n)
    tokens = skewed(rs, count, vocabulary, kind).astype(np.int64)
    dz = rs.randn(count, n).astype(STORAGE[S])
    got = run_embedding_bp(dev, S, dz, tokens, vocabulary, 0.5)
    want, tol = embedding_bp_oracle(dz, tokens, vocabulary, 0.5, None, S)
    close(got, want, tol, kind)
    again = run_embedding_bp(dev, S, dz, tokens, vocabulary, 0.5, scratch=True)
    assert np.array_equal(got, again)
    into = rs.randn(vocabulary, n).astype(STORAGE[S])
    got = run_embedding_bp(dev, S, dz, tokens, vocabulary, 0.5, into=into)
    want, tol = embedding_bp_oracle(dz, tokens, vocabulary, 0.5, into, S)
    close(got, want, tol, kind + ", added")


@pytest.mark.parametrize("S", SUFFIXES)
@pytest.mark.parametrize("ldz,lt", [("pitch3", "dense"), ("dense", "pitch8"), ("forder", "dense"), ("dense", "inner2"), ("rank3", "offset1"),
                                    ("inner2", "forder"), ("offset1", "pitch3")])
def test_embedding_bp_layouts(dev, S, ldz, lt):
    rs = np.random.RandomState(2)
    for count, n in ((200, 70), (90, 600)):
        tokens = skewed(rs, count, 53, "text").astype(np.int64)
        dz = rs.randn(count, n).astype(STORAGE[S])
        got = run_embedding_bp(dev, S, dz, tokens, 53, 2.0, ldz=ldz, lt=lt)
        want, tol = embedding_bp_oracle(dz, tokens, 53, 2.0, None, S)
        close(got, want, tol)


def test_embedding_bp_without_tokens(dev):
    dz = np.zeros((0, 9), np.float32)
    tokens = np.zeros(0, np.int64)
    assert not run_embedding_bp(dev, "Float", dz, tokens, 40, 1.0).any()
    into = np.random.RandomState(0).randn(40, 9).astype(np.float32)
    assert np.array_equal(run_embedding_bp(dev, "Float", dz, tokens, 40, 1.0, into=into), into)


# ---- log probabilities of tokens ---------------------------------------------------------------------------------------

def token_probs_oracle(x, tokens, k, S):
    xd = x.astype(np.float64)
    rows, n = xd.shape
    u = unit(COMPUTE[S])
    out = {key: np.zeros(rows) for key in ("lp", "ls", "h", "t_lp", "t_ls", "t_h")}
    top, top_lp, t_top = np.zeros((rows, k), np.int64), np.zeros((rows, k)), np.zeros((rows, k))
    with np.errstate(all="ignore"):
        for r in range(rows):
            v, t = xd[r], int(tokens[r])
            order = [i for i in np.argsort(-v, kind="stable") if not np.isnan(v[i])][:k]
            top[r] = order + [-1] * (k - len(order))
            bad = np.isnan(v).any() or np.isposinf(v).any()
            none = not bad and np.isneginf(v).all()
            if bad:
                ls = h = np.nan
                of = np.full(n, np.nan)
                size = log_size = spread = 0.0
                d = np.zeros(n)
            elif none:
                ls, h, of = -np.inf, 0.0, np.full(n, -np.inf)
                size = log_size = spread = 0.0
                d = np.zeros(n)
            else:
                m = v.max()
                d = v - m
                e = np.exp(d)
                p = e / e.sum()
                live = p > 0
                log_size = np.log(e.sum())
                ls, of = m + log_size, d - log_size
                weight = -(p[live] * d[live])
                h = log_size + weight.sum()
                # exp: 4 roundings and those of its argument; the sum: N(n) more; every term counts with its share
                size = u * (N(n) + 6 + 3 * weight.sum()) + 3 * u * log_size
                spread = u * (weight * (N(n) + 8 + 3 * np.abs(d[live]))).sum() + size * weight.sum()
            out["ls"][r], out["h"][r] = ls, h
            out["t_ls"][r] = size + 4 * u * abs(ls) if np.isfinite(ls) else 0
            out["t_h"][r] = size + spread + 4 * u * h if np.isfinite(h) else 0
            out["lp"][r] = 0.0 if t < 0 else (np.nan if t >= n else of[t])
            ends = np.abs(np.where(np.isfinite(of), of, 0)) + np.abs(np.where(np.isfinite(d), d, 0))
            out["t_lp"][r] = size + 4 * u * ends[t] if 0 <= t < n else 0
            top_lp[r] = [np.nan if i < 0 else of[i] for i in top[r]]
            t_top[r] = [size + 4 * u * ends[i] if i >= 0 else 0 for i in top[r]]
    out.update(top=top, top_lp=top_lp, t_top=t_top)
    return out


def run_token_probs(dev, S, x, tokens, k, layout="dense", scratch=False, wants=("lp", "ls", "h", "top", "top_lp")):
    C = COMPUTE[S]
    rows, n = x.shape
    X, K = View(dev, rows, n, layout, STORAGE[S], x), Vec(dev, tokens, np.int64)
    o = {key: Vec(dev, np.full(rows, 3.0), C) for key in ("lp", "ls", "h")}
    o["top"], o["top_lp"] = Vec(dev, np.full(rows * k, 3), np.int64), Vec(dev, np.full(rows * k, 3.0), C)
    bytes_ = dev.ops.amd_scratchTokenLogProbs(rows, n, k) if scratch else 0
    W = dev.empty(bytes_) if scratch else None
    at = {key: v.ptr if key in wants else None for key, v in o.items()}
    getattr(dev.ops, "amd_execTokenLogProbs" + S)(extra(dev, x=X), X.ptr, X.info_ptr, K.ptr if "lp" in wants else None, at["lp"], at["ls"], at["h"],
                                                  k, at["top"], at["top_lp"], W and W.ptr, bytes_)
    X.get()
    out = {key: v.get() for key, v in o.items()}
    out["top"], out["top_lp"] = out["top"].reshape(rows, k), out["top_lp"].reshape(rows, k)
    for v in [X, K, W] + list(o.values()):
        if v is not None:
            v.free()
    return out


def check_token_probs(got, want):
    close(got["ls"], want["ls"], want["t_ls"], "logSum")
    close(got["lp"], want["lp"], want["t_lp"], "logProbs")
    close(got["h"], want["h"], want["t_h"], "entropy")
    assert np.array_equal(got["top"], want["top"]), "topTokens"
    close(got["top_lp"], want["top_lp"], want["t_top"], "topLogProbs")


@pytest.mark.parametrize("S", SUFFIXES)
@pytest.mark.parametrize("n", (1, 2, 3, 9, 63, 64, 65, 257, 511, 1000, 2049, 4097, 8191, 16384, 32003, 50257, 131073))
def test_token_log_probs_lengths(dev, S, n):
    rs = np.random.RandomState(n)
    for rows, k in ((1, min(8, n)), (3, min(64, n)), (40 if n < 5000 else 6, min(5, n)), (2, 0)):
        x = (rs.randn(rows, n) * 4).astype(STORAGE[S])
        tokens = rs.randint(0, n, rows)
        tokens[1::5] = -1
        tokens[2::5] = n
        check_token_probs(run_token_probs(dev, S, x, tokens, k), token_probs_oracle(x, tokens, k, S))


@pytest.mark.parametrize("S", SUFFIXES)
@pytest.mark.parametrize("more", (1, 5, 81, 200, 512, 904, 1105, 2047))
def test_token_log_probs_at_a_rows_end(dev, S, more):
    """the last slice of a row with few elements in its waves, and fewer than the alternatives; the largest ones lie there"""
    rs = np.random.RandomState(more)
    n = 8192 + more
    for k in (8, 17, 33, 64):
        x = (rs.randn(3, n) * 4).astype(STORAGE[S])
        x[1, 8192:] += 16
        x[2] = np.round(x[2])
        x[2, :8192 - 7] = -np.inf
        tokens = rs.randint(0, n, 3)
        check_token_probs(run_token_probs(dev, S, x, tokens, k), token_probs_oracle(x, tokens, k, S))


@pytest.mark.parametrize("S", SUFFIXES)
@pytest.mark.parametrize("layout", LAYOUTS)
def test_token_log_probs_layouts(dev, S, layout):
    rs = np.random.RandomState(6)
    for rows, n, k in ((6, 50, 7), (70, 1031, 4), (2, 20011, 16)):
        x = (rs.randn(rows, n) * 4).astype(STORAGE[S])
        tokens = rs.randint(0, n, rows)
        check_token_probs(run_token_probs(dev, S, x, tokens, k, layout, scratch=True), token_probs_oracle(x, tokens, k, S))


@pytest.mark.parametrize("S", SUFFIXES)
@pytest.mark.parametrize("n,layout", [(70, "dense"), (70, "forder"), (70, "inner2"), (3001, "dense"), (3001, "forder"), (3001, "pitch3"),
                                      (40000, "dense")])
def test_token_log_probs_of_masked_and_equal_rows(dev, S, n, layout):
    """rows of equal values, of few values, ascending and descending rows, masks of -infinity and of the type's lowest value
    with nothing, one element, few and all but one left, the largest values, signed zeros, NaN and +infinity"""
    rs = np.random.RandomState(n)
    low, high = float(np.finfo(STORAGE[S]).min), float(np.finfo(STORAGE[S]).max)
    ramp = np.linspace(-6, 6, n)
    rows = [np.zeros(n), np.full(n, 2.5), rs.randint(-2, 3, n), ramp, -ramp, np.full(n, -np.inf), np.full(n, low), np.full(n, high)]
    for mask in (-np.inf, low):
        for left in (1, 3, n - 1):
            v = np.full(n, mask)
            v[rs.permutation(n)[:left]] = rs.randn(left)
            rows.append(v)
    v = rs.randn(n)
    v[:-5] = -np.inf  # the first slices of the row hold nothing
    rows.append(v)
    v = rs.randn(n)
    v[5:] = low
    rows.append(v)
    zeros = np.zeros(n)
    zeros[::2] = -0.0
    rows.append(zeros)
    for bad in (np.nan, np.inf):
        v = rs.randn(n)
        v[n // 2] = bad
        rows.append(v)
    rows.append(np.full(n, np.nan))
    v = np.full(n, np.nan)
    v[[3, n - 2]] = 1.0, 2.0
    rows.append(v)
    x = np.array(rows).astype(STORAGE[S])
    for tokens in (np.arange(len(rows)) % n, np.full(len(rows), -1), np.full(len(rows), n - 1)):
        for k in (5, 64):
            check_token_probs(run_token_probs(dev, S, x, tokens, k, layout), token_probs_oracle(x, tokens, k, S))
    # many rows at once: each of them is a block's (a wave's, where it is short) instead of being cut into slices
    many = np.tile(x, (1024 // len(rows) + 1, 1)) if n <= 3001 else x[:0]
    if len(many):
        tokens = np.arange(len(many)) % n
        got, few = run_token_probs(dev, S, many, tokens, 5, layout), token_probs_oracle(x, tokens[:len(rows)], 5, S)
        want = {key: np.tile(v, (len(many) // len(rows),) + (1,) * (v.ndim - 1)) for key, v in few.items()}
        for key in ("lp", "t_lp"):  # (the tokens differ from one copy of the rows to the next)
            want[key] = np.concatenate([token_probs_oracle(x, tokens[i:i + len(rows)], 0, S)[key] for i in range(0, len(many), len(rows))])
        check_token_probs(got, want)


def test_token_log_probs_parts(dev):
    rs = np.random.RandomState(9)
    x = rs.randn(5, 7000).astype(np.float32)
    tokens = rs.randint(0, 7000, 5)
    whole = run_token_probs(dev, "Float", x, tokens, 6)
    for wants, k in ((("lp",), 0), (("ls",), 0), (("h",), 0), (("top",), 6), (("lp", "top", "top_lp"), 6), (("ls", "h"), 0)):
        got = run_token_probs(dev, "Float", x, tokens, k, wants=wants)
        for key in ("lp", "ls", "h", "top", "top_lp"):
            if key in wants:
                close(got[key], whole[key], 1e-5 * (1 + np.abs(whole[key])) if got[key].dtype != np.int64 else 0, key)
            else:
                assert (got[key] == 3).all(), key


def run_token_probs_bp(dev, S, x, tokens, ls, h, a, b, lx="dense", ldx="dense", inplace=False):
    C = COMPUTE[S]
    rows, n = x.shape
    X, K = View(dev, rows, n, lx, STORAGE[S], x), Vec(dev, tokens, np.int64)
    DX = X if inplace else View(dev, rows, n, ldx, STORAGE[S])
    V = [None if v is None else Vec(dev, v, C) for v in (ls, h, a, b)]
    getattr(dev.ops, "amd_execTokenLogProbsBp" + S)(extra(dev, x=X, z=DX), X.ptr, X.info_ptr, K.ptr, *[v and v.ptr for v in V], DX.ptr, DX.info_ptr)
    out = DX.get()
    for v in [X, K, DX] + V:
        if v is not None:
            v.free()
    return out


def token_probs_bp_oracle(x, tokens, ls, h, a, b, S):
    xd = x.astype(np.float64)
    rows, n = xd.shape
    u = unit(COMPUTE[S])
    want, tol = np.zeros((rows, n)), np.zeros((rows, n))
    with np.errstate(all="ignore"):
        for r in range(rows):
            t = int(tokens[r]) if a is not None else -1
            if np.isneginf(ls[r]):
                continue
            lp = xd[r] - float(ls[r])
            p = np.exp(lp)
            av = 0.0 if t < 0 else (np.nan if t >= n else float(a[r]))
            want[r] = -av * p
            if 0 <= t < n:
                want[r, t] += av
            # p: 4 roundings and those of its argument (that is at most |x| + |logSum|)
            d_p = p * u * (5 + 2 * np.where(p > 0, np.abs(lp) + np.abs(float(ls[r])), 0))
            tol[r] = abs(av) * (d_p + 2 * u * (p + 1.0 * (np.arange(n) == t)))
            if b is not None:
                w = np.where(p > 0, lp + float(h[r]), 0.0)
                want[r] -= float(b[r]) * p * w
                tol[r] += abs(float(b[r])) * (d_p * np.abs(w) + p * u * (4 * np.abs(w) + 2 * np.where(p > 0, np.abs(lp), 0) + 2 * abs(float(h[r]))))
                tol[r] += 2 * u * np.abs(want[r])
    # (subnormal p: exp's own last place)
    tol = tol + 8 * smallest(COMPUTE[S]) * (1 + np.abs(xd).max(initial=0, where=np.isfinite(xd)))
    return want, tol + stored(want, S)


def probs_inputs(S, x, rs):
    o = token_probs_oracle(x, np.zeros(x.shape[0], np.int64), 0, S)
    C = COMPUTE[S]
    rows = x.shape[0]
    return o["ls"].astype(C), o["h"].astype(C), rs.randn(rows).astype(C), (rs.randn(rows) / 4).astype(C)


@pytest.mark.parametrize("S", SUFFIXES)
@pytest.mark.parametrize("n", (1, 2, 7, 64, 65, 1000, 2049, 8191, 50257))
def test_token_log_probs_bp(dev, S, n):
    rs = np.random.RandomState(n)
    for rows, lx, ldx in ((1, "dense", "dense"), (4, "pitch3", "pitch8"), (6, "rank3", "offset1"), (5, "forder", "inner2"), (7, "dense", "dense")):
        x = (rs.randn(rows, n) * 3).astype(STORAGE[S])
        tokens = rs.randint(0, n, rows)
        tokens[1::4] = -1
        tokens[2::4] = n
        ls, h, a, b = probs_inputs(S, x, rs)
        for aa, bb in ((a, None), (a, b), (None, b)):
            got = run_token_probs_bp(dev, S, x, tokens, ls, h, aa, bb, lx, ldx)
            want, tol = token_probs_bp_oracle(x, tokens, ls, h, aa, bb, S)
            close(got, want, tol)
        got = run_token_probs_bp(dev, S, x, tokens, ls, h, a, b, lx, inplace=True)
        want, tol = token_probs_bp_oracle(x, tokens, ls, h, a, b, S)
        close(got, want, tol, "in place")


@pytest.mark.parametrize("S", SUFFIXES)
def test_token_log_probs_bp_of_masked_rows(dev, S):
    rs = np.random.RandomState(3)
    n = 1500
    x = rs.randn(5, n)
    x[0] = -np.inf
    x[1, 10:] = -np.inf
    x[2, 10:] = float(np.finfo(STORAGE[S]).min)
    x[3] = float(np.finfo(STORAGE[S]).min)
    x = x.astype(STORAGE[S])
    tokens = np.array([4, 700, 3, 9, 8])  # the second row's token is masked
    ls, h, a, b = probs_inputs(S, x, rs)
    for bb in (None, b):
        got = run_token_probs_bp(dev, S, x, tokens, ls, h, a, bb)
        want, tol = token_probs_bp_oracle(x, tokens, ls, h, a, bb, S)
        close(got, want, tol)
        assert not got[0].any()


def test_token_log_probs_gradient_against_differences(dev):
    """double: the sum of a logProb + b entropy changes with x as the backward call says"""
    rs = np.random.RandomState(12)
    rows, n, h = 2, 40, 1e-4
    x, a, b = rs.randn(rows, n), rs.randn(rows), rs.randn(rows)
    tokens = np.array([3, 39])

    def loss(x):
        o = run_token_probs(dev, "Double", x, tokens, 0)
        return float((o["lp"] * a + o["h"] * b).sum())

    o = run_token_probs(dev, "Double", x, tokens, 0)
    dx = run_token_probs_bp(dev, "Double", x, tokens, o["ls"], o["h"], a, b)
    for r, c in ((0, 3), (0, 4), (1, 39), (1, 0)):
        up, down = x.copy(), x.copy()
        up[r, c] += h
        down[r, c] -= h
        assert abs((loss(up) - loss(down)) / (2 * h) - dx[r, c]) < 1e-6


# ---- clipping ----------------------------------------------------------------------------------------------------------

def run_clip(dev, S, tensors, most, apart=True, inplace=False, results=True, scratch=False):
    """tensors of their own (apart) or views into one vector, one element behind its start"""
    T, C = STORAGE[S], COMPUTE[S]
    lengths = [t.size for t in tensors]
    total = sum(lengths)
    n = len(tensors)
    if apart:
        held = [Vec(dev, t, T) for t in tensors]
        out = held if inplace else [Vec(dev, np.full(t.size, 5.0), T) for t in tensors]
        at = [[v.ptr for v in held], [v.ptr for v in out]]
    else:
        flat = np.concatenate([np.zeros(1)] + list(tensors))
        held = [Vec(dev, flat, T)]
        out = held if inplace else [Vec(dev, np.full(total + 1, 5.0), T)]
        starts = 1 + np.cumsum([0] + lengths)[:-1]
        at = [[v[0].ptr + int(s) * np.dtype(T).itemsize for s in starts] for v in (held, out)]
    tables = dev.upload(np.array(at + [[0] * n], dtype=np.int64))
    offsets = Vec(dev, np.cumsum([0] + lengths), np.int64)
    norm = Vec(dev, [3.0], C)
    bytes_ = dev.ops.amd_scratchClipByGlobalNorm(total) if scratch else 0
    W = dev.empty(bytes_) if scratch else None
    getattr(dev.ops, "amd_execClipByGlobalNorm" + S)(extra(dev), tables.ptr, (tables.ptr + 8 * n) if results else None, offsets.ptr, n, total, most,
                                                     norm.ptr, W and W.ptr, bytes_)
    got = [v.get() for v in out]
    if not apart:
        got = np.split(got[0][1:], np.cumsum(lengths)[:-1])
    value = norm.get()[0]
    for v in held + (out if out is not held else []) + [tables, offsets, norm, W]:
        if v is not None:
            v.free()
    return got, value


def check_clip(got, value, tensors, most, S):
    norm = np.sqrt(sum((t.astype(np.float64) ** 2).sum() for t in tensors))
    u = unit(COMPUTE[S])
    assert abs(float(value) - norm) <= 2 * u * norm + 1e-12 * norm
    factor = most / norm if norm > most else 1.0
    for g, t in zip(got, tensors):
        want = t.astype(np.float64) * factor
        close(g, want, (3 * u * np.abs(want) + 1e-12 * np.abs(want) + stored(want, S)) if factor != 1.0 else 0.0)


@pytest.mark.parametrize("S", SUFFIXES)
@pytest.mark.parametrize("apart", (True, False))
@pytest.mark.parametrize("lengths", [[1], [5], [0, 3, 0, 0, 9, 0], [1] * 70, [16384], [1000003], [3, 100, 65537, 1, 8, 0, 5000], list(range(200)),
                                     [4096] * 9 + [1] * 600 + [30000]])
def test_clip_by_global_norm(dev, S, apart, lengths):
    rs = np.random.RandomState(len(lengths))
    tensors = [(rs.randn(k) / 8).astype(STORAGE[S]) for k in lengths]
    for most in (0.25, 1e6):
        got, value = run_clip(dev, S, tensors, most, apart)
        check_clip(got, value, tensors, most, S)
        same, _ = run_clip(dev, S, tensors, most, apart, inplace=True, scratch=True)
        for a, b in zip(got, same):
            assert np.array_equal(a, b)
    got, value = run_clip(dev, S, tensors, 0.0, apart, results=False)
    check_clip(tensors, value, tensors, 1e30, S)
    assert all((g == 5.0).all() for g in got)


@pytest.mark.parametrize("S", SUFFIXES)
def test_clip_of_many_tensors(dev, S):
    rs = np.random.RandomState(1)
    lengths = rs.randint(0, 40, 3000)
    lengths[rs.randint(0, 3000, 20)] = rs.randint(1000, 50000, 20)
    tensors = np.split((rs.randn(int(lengths.sum())) / 8).astype(STORAGE[S]), np.cumsum(lengths)[:-1])
    got, value = run_clip(dev, S, tensors, 1.0, apart=False)
    check_clip(got, value, tensors, 1.0, S)


@pytest.mark.parametrize("S", SUFFIXES)
@pytest.mark.parametrize("apart", (True, False))
def test_clip_of_large_tensors(dev, S, apart):
    """beyond 25 MB, where the tiles are larger: ends of tensors inside them, and a last tile that is not whole"""
    rs = np.random.RandomState(4)
    n = 30000000 // STORAGE[S]().itemsize
    lengths = [n // 2 + 1, 7, 0, 16384, n // 4 + 3, 3, n // 4 + 101]
    whole = (rs.randint(-64, 65, sum(lengths)) / 64).astype(STORAGE[S])
    tensors = np.split(whole, np.cumsum(lengths)[:-1])
    got, value = run_clip(dev, S, tensors, 1.0, apart)
    check_clip(got, value, tensors, 1.0, S)
    same, _ = run_clip(dev, S, tensors, 1.0, apart, inplace=True)
    assert all(np.array_equal(a, b) for a, b in zip(same, got))
    got, value = run_clip(dev, S, tensors, 0.0, apart, results=False)
    check_clip(tensors, value, tensors, 1e30, S)


@pytest.mark.parametrize("S", SUFFIXES)
def test_clip_of_extremes(dev, S):
    """no tensors; all zero; squares beyond the type's range; NaN and infinities, which change nothing but the norm"""
    got, value = run_clip(dev, S, [np.zeros(0)], 1.0)
    assert value == 0 and got[0].size == 0
    tensors = [np.zeros(1000, STORAGE[S])]
    got, value = run_clip(dev, S, tensors, 1.0)
    assert value == 0 and not got[0].any()
    big = {"Half": 6e4, "Float": 1e30, "Double": 1e150}[S]
    tensors = [np.full(500, big).astype(STORAGE[S]), np.full(77, -big).astype(STORAGE[S])]
    got, value = run_clip(dev, S, tensors, 1.0)
    check_clip(got, value, tensors, 1.0, S)
    for bad in (np.nan, np.inf, -np.inf):
        t = np.ones(5000, STORAGE[S])
        t[4321] = bad
        got, value = run_clip(dev, S, [t], 1.0)
        assert np.array_equal(got[0], t, equal_nan=True)
        assert np.isnan(value) if np.isnan(bad) else np.isposinf(value)
