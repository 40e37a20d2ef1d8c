"""Sizes at the ends of the int8 calls' 32-bit indexes: refused before anything is launched."""

import pytest

from qgemv_roofline_b200 import _lib

FAKE = 0x10000  # 16-byte aligned, never read


def quantize(rows, K, ldx=None):
    return _lib.lib().qgemv_int8_quantize(FAKE, 0, ldx or K, rows, K, FAKE, K, FAKE, None)


@pytest.mark.parametrize("K", [(1 << 31) - 17, (1 << 31) - 255, (1 << 31) - 511, 1 << 31, 1 << 40])
def test_rows_whose_index_would_pass_32_bits(K):
    """k_quant_rows counts a row's columns in steps of 256 in 32 bits."""
    assert quantize(1, K) == 5 and quantize(2, K) == 5
    assert "K" in _lib.last_error()
