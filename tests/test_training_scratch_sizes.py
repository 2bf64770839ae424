"""How much scratch the operators around a language model's matrix products ask for: no GPU needed."""
import pytest

from libnd4j_amd.native import NativeOps


@pytest.fixture(scope="module")
def ops():
    return NativeOps()


def test_layer_norm_gradients_of_long_rows(ops):
    """Rows beyond what a block holds in registers go by the kernel of the columns, in at most 2048 / (length / 64) ranges of rows:
    two sums of a double for each column and range."""
    for length in (16400, 20000, 70001, 1 << 20, 1 << 24):
        ranges = max(1, -(-2048 // -(-length // 64)))
        for rows in (1, 100, 4096, 1 << 20):
            assert ops.amd_scratchLayerNormBp(rows, length) <= 2 * 8 * ranges * (length + 8), (rows, length)


def test_layer_norm_gradients_of_ordinary_rows(ops):
    """256 blocks' sums, of doubles as the widest"""
    assert ops.amd_scratchLayerNormBp(16384, 1024) <= 2 * 8 * 256 * 1024
    assert ops.amd_scratchLayerNormBp(4097, 5003) <= 2 * 4 * 256 * 5008  # (doubles of that length are not held in registers)
