"""The operators around a language model's matrix products at sizes where a block comes round again - rows of a second and later
turn, several tiles to a span, several rounds of a sort - against 64-bit results."""
import numpy as np
import pytest

from libnd4j_amd import harness
from test_training_ops import (bp_inputs, check_token_probs, embedding_bp_oracle, layer_norm_bp_oracle, layer_norm_oracle, run_embedding_bp,
                               run_layer_norm, run_layer_norm_bp, run_token_probs, skewed, token_probs_oracle)
from training_views import STORAGE, SUFFIXES, close

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return harness.Device()


@pytest.mark.parametrize("S,rows,n", [("Half", 12003, 1024), ("Half", 7001, 5003), ("Half", 70001, 100), ("Half", 40003, 250), ("Half", 5001, 16384),
                                      ("Float", 15001, 2048), ("Float", 9001, 4097), ("Float", 120001, 60), ("Float", 3001, 16384),
                                      ("Double", 9001, 1000), ("Double", 2501, 8190)])
def test_layer_norm_turns(dev, S, rows, n):
    rs = np.random.RandomState(n)
    x = (rs.randn(rows, n).astype(np.float32) * 3 + 1).astype(STORAGE[S])
    gain, bias = (1 + rs.randn(n) / 8).astype(STORAGE[S]), (rs.randn(n) / 8).astype(STORAGE[S])
    z, mean, inv = run_layer_norm(dev, S, x, gain, bias, 1e-5)
    for r in range(0, rows, 2048):  # (a stretch at a time: the 64-bit arrays take memory)
        to = slice(r, r + 2048)
        want, want_mean, want_inv, tol, tol_mean, tol_inv = layer_norm_oracle(x[to], gain, bias, 1e-5, S)
        close(z[to], want, tol, "z from row %d" % r)
        close(mean[to], want_mean, tol_mean, "mean")
        close(inv[to], want_inv, tol_inv, "invStd")
    same, _, _ = run_layer_norm(dev, S, x, gain, bias, 1e-5, inplace=True)
    assert np.array_equal(same, z)


@pytest.mark.parametrize("S,rows,n", [("Float", 9001, 1024), ("Float", 40001, 100), ("Float", 20001, 300), ("Float", 1500, 7001), ("Half", 2003, 5003),
                                      ("Half", 40001, 100), ("Half", 9001, 1000), ("Half", 1001, 16000), ("Double", 3001, 4095), ("Double", 9001, 120)])
def test_layer_norm_bp_turns(dev, S, rows, n):
    args = bp_inputs(S, rows, n, n + rows)
    got = run_layer_norm_bp(dev, S, *args)
    want = layer_norm_bp_oracle(*args, S)
    for k, name in enumerate(("dx", "dGain", "dBias")):
        close(got[k], want[k], want[3 + k], "%s of [%d, %d]" % (name, rows, n))
    for where in ("dz", "x"):
        same = run_layer_norm_bp(dev, S, *args, inplace=where)
        for k in range(3):
            assert np.array_equal(same[k], got[k]), (where, k)
    parts = run_layer_norm_bp(dev, S, *args, wants=("dGain", "dBias"))
    assert np.array_equal(parts[1], got[1]) and np.array_equal(parts[2], got[2])


@pytest.mark.parametrize("S,rows,n", [("Float", 200, 50257), ("Half", 300, 50257), ("Double", 1100, 40000), ("Half", 1030, 140001), ("Float", 70, 131073)])
@pytest.mark.parametrize("k", (0, 5, 64))
def test_token_log_probs_turns(dev, S, rows, n, k):
    """slices of several tiles, and spans of several tiles: a sample of the rows, with rows of few values among them"""
    rs = np.random.RandomState(n + k)
    x = (np.random.default_rng(n + k).standard_normal((rows, n), dtype=np.float32) * 4).astype(STORAGE[S])
    x[1::9] = np.round(x[1::9])
    x[2, :n - 40] = -np.inf
    x[3, 40:] = -np.inf
    tokens = rs.randint(0, n, rows)
    got = run_token_probs(dev, S, x, tokens, k)
    sample = np.unique(np.concatenate([np.arange(12), rs.randint(0, rows, 12), [rows - 1]]))
    check_token_probs({key: v[sample] for key, v in got.items()}, token_probs_oracle(x[sample], tokens[sample], k, S))


@pytest.mark.parametrize("S", SUFFIXES)
def test_token_log_probs_of_more_rows_than_blocks(dev, S):
    """a wave for a row, and more rows than the launch has blocks: 2^20 + 77 of 5 elements"""
    rs = np.random.RandomState(1)
    rows, n, k = (1 << 20) + 77, 5, 3
    x = rs.randint(-9, 10, (rows, n)).astype(STORAGE[S])
    tokens = rs.randint(0, n, rows)
    got = run_token_probs(dev, S, x, tokens, k)
    sample = np.concatenate([np.arange(0, rows, 9973), np.arange((1 << 20) - 5, rows)])
    check_token_probs({key: v[sample] for key, v in got.items()}, token_probs_oracle(x[sample], tokens[sample], k, S))


@pytest.mark.parametrize("S", SUFFIXES)
@pytest.mark.parametrize("kind", ("spread", "text", "one"))
@pytest.mark.parametrize("count,vocabulary,n", [(300001, 65537, 3), (600000, 300, 8), (262145, 100000, 1)])
def test_embedding_bp_turns(dev, S, kind, count, vocabulary, n):
    """more tokens than the sort has threads, and the longest chunks"""
    rs = np.random.RandomState(count)
    tokens = skewed(rs, count, vocabulary, kind).astype(np.int64)
    dz = rs.randn(count, n).astype(STORAGE[S])
    want, tol = embedding_bp_oracle(dz, tokens, vocabulary, 0.5, None, S)
    close(run_embedding_bp(dev, S, dz, tokens, vocabulary, 0.5), want, tol, kind)
    into = rs.randn(vocabulary, n).astype(STORAGE[S])
    want, tol = embedding_bp_oracle(dz, tokens, vocabulary, 0.5, into, S)
    close(run_embedding_bp(dev, S, dz, tokens, vocabulary, 0.5, into=into, scratch=True), want, tol, kind + ", added")


@pytest.mark.parametrize("S", ("Float", "Half"))
@pytest.mark.parametrize("count", (1, 300, 4095, 4096, 4097))
@pytest.mark.parametrize("vocabulary", ((1 << 20) - 1, 1 << 20, (1 << 20) + 1, 1 << 24))
def test_embedding_bp_of_large_vocabularies(dev, S, count, vocabulary):
    """around 2^20 rows, where a token and its position no longer share a 32-bit word"""
    rs = np.random.RandomState(count)
    tokens = rs.randint(0, vocabulary, count)
    tokens[::3] = vocabulary - 1
    tokens[1::5] = vocabulary
    tokens[2::7] = -1
    tokens[3::11] = 0
    dz = rs.randn(count, 1).astype(STORAGE[S])
    want, tol = embedding_bp_oracle(dz, tokens, vocabulary, 2.0, None, S)
    close(run_embedding_bp(dev, S, dz, tokens, vocabulary, 2.0), want, tol)
