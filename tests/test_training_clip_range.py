"""Clipping by the global norm at the ends of the types' ranges."""
import numpy as np
import pytest

from libnd4j_amd import harness
from test_training_ops import run_clip, stored
from training_views import COMPUTE, STORAGE, Vec, close, extra, unit

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return harness.Device()


def wide(tensors):
    """The norm in extended precision, whose exponents reach far beyond a double's."""
    return np.sqrt(sum((t.astype(np.longdouble) ** 2).sum() for t in tensors))


def check(dev, S, tensors, most, **how):
    """Squares, and sums of at most 2000 of them in double: at most 2001 + 2 roundings of 2^-53, which the root halves, and one
    to the norm's type; the factor and the product one of the compute type each, the product in two steps two."""
    C, u = COMPUTE[S], unit(COMPUTE[S])
    slack = 1002 * 2.0 ** -53
    norm = wide(tensors)
    got, value = run_clip(dev, S, tensors, most, **how)
    top = np.longdouble(np.finfo(C).max)
    if norm > top * (1 + 4 * u):
        assert np.isposinf(value)
        for g, t in zip(got, tensors):
            assert np.array_equal(g, t)  # a norm of infinity changes nothing
        return
    assert np.isfinite(value)
    assert abs(np.longdouble(value) - norm) <= (u + slack) * norm + float(np.finfo(C).smallest_subnormal)
    factor = np.longdouble(most) / norm if norm > most else np.longdouble(1)
    for g, t in zip(got, tensors):
        want = (t.astype(np.longdouble) * factor).astype(np.float64)
        close(g, want, ((4 * u + slack) * np.abs(want) + 2 * stored(want, S)) if factor != 1 else 0.0)


@pytest.mark.parametrize("apart", (True, False))
def test_floats_whose_norm_no_float_holds(dev, apart):
    for values in ([3e38] * 4, [3.4e38, 1e38], [3e38, 0.0, -3e38], [2e38] * 1500):
        check(dev, "Float", [np.array(values, np.float32), np.ones(77, np.float32)], 1.0, apart=apart)
        check(dev, "Float", [np.array(values, np.float32)], 1.0, apart=apart, inplace=True)
    for values in ([3.4e38], [2e38, -2e38], [1e38] * 11):  # these are held
        check(dev, "Float", [np.array(values, np.float32), np.ones(77, np.float32)], 1.0, apart=apart)


@pytest.mark.parametrize("S", ("Float", "Double"))
@pytest.mark.parametrize("n", (3, 700))
def test_factors_below_the_normal_range(dev, S, n):
    """large gradients and a small bound: the factor has few bits in the type, or none, and the product all"""
    rs = np.random.RandomState(n)
    big, small = (1e37, (1e-2, 1e-4, 1e-9)) if S == "Float" else (1e306, (1e-3, 1e-8, 1e-20))
    tensors = [(rs.randn(n) * big / 8).astype(STORAGE[S]), rs.randn(n).astype(STORAGE[S])]
    for most in small:
        check(dev, S, tensors, most)
        check(dev, S, tensors, most, inplace=True)


@pytest.mark.parametrize("apart", (True, False))
def test_doubles_whose_squares_no_double_holds(dev, apart):
    rs = np.random.RandomState(2)
    rows = rs.randn(600)
    for scale in (1e200, 1e153, 1e155, 1e306, 1e-153, 1e-155, 1e-163, 1e-200, 1e-300, 1e-310):
        check(dev, "Double", [rows * scale, -rows[:5] * scale], 1.0, apart=apart)
        check(dev, "Double", [rows * scale, rows[:77] * 1e-3], 0.5, apart=apart)
        check(dev, "Double", [rows * scale, rows[:77] * 1e-170, rows[:9] * 1e150], scale / 4, apart=apart)
    check(dev, "Double", [np.array([1.7e308])], 1.0, apart=apart)
    check(dev, "Double", [np.array([1.7e308, 1e308])], 1.0, apart=apart)  # the norm is beyond the range
    check(dev, "Double", [np.array([5e-324, 0.0, -5e-324])], 1.0, apart=apart)
    for bad in (np.nan, np.inf):
        t = np.array([1e200, bad, 1e-200, 1.0])
        got, value = run_clip(dev, "Double", [t], 1.0, apart)
        assert np.array_equal(got[0], t, equal_nan=True)
        assert np.isnan(value) if np.isnan(bad) else np.isposinf(value)
