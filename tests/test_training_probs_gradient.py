"""The gradient of log probabilities of tokens: unlikely tokens, and padding over rows that hold anything."""
import numpy as np
import pytest

from libnd4j_amd import harness
from test_training_ops import run_token_probs, run_token_probs_bp, stored, token_probs_bp_oracle
from training_views import COMPUTE, STORAGE, SUFFIXES, close, smallest, unit

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return harness.Device()


@pytest.mark.parametrize("S", SUFFIXES)
@pytest.mark.parametrize("lx,ldx", [("dense", "dense"), ("pitch3", "offset1"), ("forder", "forder"), ("inner2", "dense")])
@pytest.mark.parametrize("n", (40, 3000, 9001))
def test_unlikely_tokens(dev, S, lx, ldx, n):
    """x and logSum are multiples of 2^-6, so that x - logSum is exact, down to log probabilities of -100 (a float's exp is
    subnormal from -87.3 on).  exp takes 4 roundings, the product one more, the comparison as many of its own in double; a subnormal
    one is off by a place of its own, twice for the two products."""
    rs = np.random.RandomState(n)
    C, u = COMPUTE[S], unit(COMPUTE[S])
    lp = -rs.randint(0, 100 * 64 + 1, (5, n)) / 64.0
    if S == "Half":
        lp = np.round(lp * 8) / 8  # (11 bits)
    ls = np.array([0.0, 1.0, -2.0, 16.0, 0.5])
    x = (lp + ls[:, None]).astype(STORAGE[S])
    lp = x.astype(np.float64) - ls[:, None]
    tokens = rs.randint(0, n, 5)
    a = np.array([1.0, -0.75, 3.0, 1e-3, 64.0])
    got = run_token_probs_bp(dev, S, x, tokens, ls.astype(C), None, a.astype(C), None, lx, ldx)
    a = a.astype(C).astype(np.float64)
    p = np.exp(lp)
    want = -a[:, None] * p
    want[np.arange(5), tokens] += a
    tol = (5 * u + 5 * 2.0 ** -53) * np.abs(a)[:, None] * p + 2 * smallest(C) * (1 + np.abs(a)[:, None])
    tol[np.arange(5), tokens] += 2 * u * np.abs(a)
    close(got, want, tol + stored(want, S))


@pytest.mark.parametrize("S", SUFFIXES)
@pytest.mark.parametrize("lx,ldx", [("dense", "dense"), ("pitch3", "offset1"), ("forder", "forder"), ("inner2", "dense")])
@pytest.mark.parametrize("n", (40, 3000, 9001))
def test_padding_has_no_gradient_whatever_the_row_holds(dev, S, lx, ldx, n):
    """a negative token: the row's log probability is 0 by definition, and zeros come back for rows of NaN and infinities too"""
    rs = np.random.RandomState(n)
    C = COMPUTE[S]
    x = rs.randn(7, n).astype(STORAGE[S])
    x[0] = np.nan
    x[1, n // 2] = np.nan
    x[2, 3] = np.inf
    x[3] = np.inf
    x[4] = -np.inf
    tokens = np.array([-1, -5, -1, -1, -1, -1, n // 3])
    out = run_token_probs(dev, S, x, tokens, 0)
    assert not out["lp"][:6].any()
    a = rs.randn(7).astype(C)
    a[1], a[2] = np.nan, np.inf  # (nor does what stands in a padded place count)
    for inplace in (False, True):
        got = run_token_probs_bp(dev, S, x, tokens, out["ls"], None, a, None, lx, ldx, inplace)
        assert not got[:6].any()
        want, tol = token_probs_bp_oracle(x[6:], tokens[6:], out["ls"][6:], None, a[6:], None, S)
        close(got[6:], want, tol)
    # with entropies the row's NaN are those of the entropy's gradient, and a row of numbers has that alone
    b = (rs.randn(7) / 4).astype(C)
    got = run_token_probs_bp(dev, S, x, tokens, out["ls"], out["h"], a, b, lx, ldx)
    want, tol = token_probs_bp_oracle(x[5:], tokens[5:], out["ls"][5:], out["h"][5:], a[5:], b[5:], S)
    close(got[5:], want, tol)
    assert not got[4].any() and np.isnan(got[1]).all()
