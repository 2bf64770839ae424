"""Strided device arrays and 64-bit oracles for the tests of the operators around a language model's matrix products."""
import numpy as np

from libnd4j_amd import harness

SUFFIXES = ("Float", "Half", "Double")
STORAGE = {"Float": np.float32, "Half": np.float16, "Double": np.float64}
COMPUTE = {"Float": np.float32, "Half": np.float32, "Double": np.float64}


def unit(dtype):
    """A rounding to this type is off by at most this, relative to the value."""
    return float(np.finfo(dtype).eps) / 2


def smallest(dtype):
    """... or by at most this where the value is subnormal."""
    return float(np.finfo(dtype).smallest_subnormal) / 2


LAYOUTS = ("dense", "pitch8", "pitch3", "offset1", "forder", "inner2", "rank3")


class View(object):
    """Rows of numbers somewhere in a larger buffer whose other elements hold a sentinel."""

    SENTINEL = 77.0

    def __init__(self, dev, rows, length, layout, dtype, values=None):
        self.dev, self.dtype, self.layout = dev, np.dtype(dtype), layout
        lead, start = 0, 0
        strides = [length, 1]
        shape = [rows, length]
        if layout == "pitch8":
            strides = [length + 8, 1]
        elif layout == "pitch3":
            strides = [length + 3, 1]
        elif layout == "offset1":
            start = 1
        elif layout == "forder":
            strides = [1, rows]
        elif layout == "inner2":
            strides = [2 * length + 1, 2]
        elif layout == "rank3" and rows % 2 == 0:
            shape = [2, rows // 2, length]
            strides = [rows // 2 * (length + 5), length + 5, 1]
        self.start = start
        span = start + 1 + sum((n - 1) * s for n, s in zip(shape, strides)) + 16
        if rows == 0:
            span = start + 16
        self.host = np.full(span, self.SENTINEL, dtype=self.dtype)
        self.info = harness.shape_info(shape, strides=strides, order="f" if layout == "forder" else "c")
        self.shape, self.strides = shape, strides
        self.rows, self.length = rows, length
        if values is not None:
            self._at(self.host)[...] = np.asarray(values, dtype=self.dtype).reshape(shape)
        self.buf = dev.upload(self.host)

    def _at(self, host):
        item = self.dtype.itemsize
        return np.lib.stride_tricks.as_strided(host[self.start:], shape=self.shape, strides=[s * item for s in self.strides])

    @property
    def ptr(self):
        return self.buf.ptr + self.start * self.dtype.itemsize

    @property
    def info_ptr(self):
        return self.info.ctypes.data

    def get(self, check=True):
        """The view's values; everything around them has to be what it was."""
        now = self.buf.download(self.dtype, self.host.size)
        values = self._at(now).copy().reshape(self.rows, self.length)
        if check:
            self._at(now)[...] = 0
            around = self.host.copy()
            self._at(around)[...] = 0
            assert np.array_equal(now, around), "elements outside the view were written"
        return values

    def free(self):
        self.buf.free()


class Vec(object):
    """A dense device vector with a few sentinel elements behind it."""

    def __init__(self, dev, values, dtype):
        self.n = int(np.size(values))
        self.dtype = np.dtype(dtype)
        self.host = np.concatenate([np.asarray(values, dtype=self.dtype).reshape(-1), np.full(4, 77, dtype=self.dtype)])
        self.buf = dev.upload(self.host)

    @property
    def ptr(self):
        return self.buf.ptr

    def get(self):
        now = self.buf.download(self.dtype, self.n + 4)
        assert np.array_equal(now[self.n:], self.host[self.n:]), "elements behind the vector were written"
        return now[:self.n]

    def free(self):
        self.buf.free()


def extra(dev, x=None, y=None, z=None, stream=None):
    import ctypes
    e = (ctypes.c_void_p * 20)()
    e[1] = dev.stream if stream is None else stream
    for slot, v in ((0, x), (7, y), (8, z)):
        if v is not None:
            e[slot] = v.info.ctypes.data
    return e


def close(got, want, tolerance, what=""):
    """got within tolerance of want, element by element; infinities and NaN in the same places."""
    got, want = np.asarray(got, dtype=np.float64), np.asarray(want, dtype=np.float64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), what + ": NaN in other places"
    assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)]), what + ": other infinities"
    tolerance = np.broadcast_to(np.asarray(tolerance, dtype=np.float64), want.shape)
    off = np.where(fine, np.abs(np.where(fine, got, 0) - np.where(fine, want, 0)), 0.0)
    bad = off > tolerance
    if bad.any():
        at = tuple(int(i) for i in np.argwhere(bad)[0])
        raise AssertionError("%s: %d of %d off, first at %s: %r, wanted %r, tolerance %r" % (
            what, int(bad.sum()), bad.size, at, float(got[at]), float(want[at]), float(tolerance[at])))
