"""Layer norm of rows whose values (nearly) agree: what is left after the mean is small, and it is all that counts.

Rows here have a mean that a float holds exactly, and partial sums that are exact in any order (whole multiples of the values'
last place, fewer than 2^24 of them).  So the mean is exact, and so is what is left of a value after it: a constant row is the
bias and nothing else, and its gain has no gradient."""
import numpy as np
import pytest

from libnd4j_amd import harness
from test_training_ops import N, layer_norm_bp_oracle, run_layer_norm, run_layer_norm_bp, stored
from training_views import COMPUTE, STORAGE, SUFFIXES, close, unit

pytestmark = pytest.mark.gpu

VALUES = (0.0, 7.25, 100.0, -333.25, 1000.0, -2000.0, 30000.0, 60000.0)
LENGTHS = (1, 3, 100, 128, 300, 768, 1000, 1023, 2048, 5003, 8191)
EPS = 1e-5


@pytest.fixture(scope="module")
def dev():
    return harness.Device()


def affine(S, n, seed=0):
    rs = np.random.RandomState(seed)
    return (1 + rs.randn(n) / 8).astype(STORAGE[S]), (rs.randn(n) / 8).astype(STORAGE[S])


@pytest.mark.parametrize("S", SUFFIXES)
@pytest.mark.parametrize("layout", ("dense", "pitch3", "offset1", "forder", "inner2"))
def test_a_constant_row_is_the_bias(dev, S, layout):
    for n in LENGTHS if layout in ("dense", "pitch3") else (100, 1023):
        x = np.repeat(np.array(VALUES), n).reshape(len(VALUES), n).astype(STORAGE[S])
        gain, bias = affine(S, n)
        for g, b in ((gain, bias), (gain, None), (None, bias), (None, None)):
            z, mean, _ = run_layer_norm(dev, S, x, g, b, EPS, layout, layout)
            assert np.array_equal(mean, np.array(VALUES)), n
            assert np.array_equal(z, np.broadcast_to(np.zeros(n, z.dtype) if b is None else b, z.shape)), (n, layout)


@pytest.mark.parametrize("S", SUFFIXES)
@pytest.mark.parametrize("layout", ("dense", "pitch3", "offset1", "forder", "inner2"))
def test_a_constant_row_has_no_gradient_of_the_gain(dev, S, layout):
    for n in LENGTHS if layout in ("dense", "pitch3") else (100, 1023):
        x = np.repeat(np.array(VALUES), n).reshape(len(VALUES), n).astype(STORAGE[S])
        gain, _ = affine(S, n)
        dz = np.random.RandomState(n).randn(*x.shape).astype(STORAGE[S])
        inv = np.full(len(VALUES), 1 / np.sqrt(EPS)).astype(COMPUTE[S])
        mean = np.array(VALUES).astype(COMPUTE[S])
        for g in (gain, None):
            got = run_layer_norm_bp(dev, S, x, g, mean, inv, dz, layout, layout, layout)
            want = layer_norm_bp_oracle(x, g, mean, inv, dz, S)
            assert not got[1].any(), (n, layout)
            for k, name in enumerate(("dx", "dGain", "dBias")):
                close(got[k], want[k], want[3 + k], "%s of rows of %d" % (name, n))


def nearly_constant(n, centre, step):
    """As many elements a step above the centre as below it, and the others (at least one) on it."""
    x = np.full(n, float(centre))
    x[1:n // 3] += step
    x[n // 3:2 * (n // 3) - 1] -= step
    return x


ROWS = ((1000.0, 0.5), (2000.0, 1.0), (-333.25, 0.25), (60000.0, 32.0))


@pytest.mark.parametrize("S", SUFFIXES)
@pytest.mark.parametrize("layout", ("dense", "pitch3", "forder"))
def test_nearly_constant_rows(dev, S, layout):
    """The variance is a sum of equal exact squares: exact, divided by n and added to epsilon and so on, five roundings to the
    deviation's inverse (the root halves those before it); a product with it, with the gain, a sum with the bias: 8 roundings, and
    as many of the comparison's own."""
    u = unit(COMPUTE[S])
    for n in (9, 100, 768, 1000, 1023, 2048, 5003, 8191):
        x = np.stack([nearly_constant(n, c, q) for c, q in ROWS]).astype(STORAGE[S])
        gain, bias = affine(S, n)
        z, mean, _ = run_layer_norm(dev, S, x, gain, bias, EPS, layout, layout)
        assert np.array_equal(mean, np.array([c for c, _ in ROWS]))
        d = x.astype(np.float64) - mean.astype(np.float64)[:, None]
        h = d / np.sqrt((d * d).mean(1, keepdims=True) + EPS)
        want = h * gain.astype(np.float64) + bias.astype(np.float64)
        close(z, want, 16 * u * (np.abs(h * gain.astype(np.float64)) + np.abs(bias.astype(np.float64))) + stored(want, S), "rows of %d" % n)
        bare, _, _ = run_layer_norm(dev, S, x, None, None, EPS, layout, layout)
        close(bare, h, 16 * u * np.abs(h) + stored(h, S), "rows of %d" % n)


@pytest.mark.parametrize("S", SUFFIXES)
def test_one_element_that_differs(dev, S):
    """8191 elements of 2000 and one of 2001: the mean, 2000 + 2^-13, has 24 bits, the elements less the mean are exact, and the
    variance is a sum of positive terms, each of which takes N(n) roundings"""
    n, u = 8192, unit(COMPUTE[S])
    x = np.full((2, n), 2000.0).astype(STORAGE[S])
    x[:, 17] = 2001
    z, mean, inv = run_layer_norm(dev, S, x, None, None, EPS)
    assert (mean.astype(np.float64) == 2000 + 2.0 ** -13).all()
    d = x.astype(np.float64) - (2000 + 2.0 ** -13)
    h = d / np.sqrt((d * d).mean(1, keepdims=True) + EPS)
    close(z, h, (N(n) + 8) * u * np.abs(h) + stored(h, S))
    dz = np.random.RandomState(0).randn(2, n).astype(STORAGE[S])
    got, want = run_layer_norm_bp(dev, S, x, None, mean, inv, dz), layer_norm_bp_oracle(x, None, mean, inv, dz, S)
    for k, name in enumerate(("dx", "dGain", "dBias")):
        close(got[k], want[k], want[3 + k], name)
