"""The 8-bit K/V format at the ends of what bf16 holds: the oracle by hand, and over every large bf16."""

import numpy as np
import pytest

from oracle import bf16, lowbit


def _block(*bits):
    x = np.zeros((1, 1, 64))
    x[0, 0, : len(bits)] = bf16.bits_to_f32(np.array(bits, np.uint16))
    return x


def test_largest_values_by_hand():
    # e4m3, scale 2^120: codes 240 and 256 stand for 1.875 2^127 and 2^128; halfway is 1.9375 2^127, 0x7f78
    v, byte = lowbit.kv8_values(_block(0x7F7F, 0x7F78, 0x7F77, 0xFF78, 0x7F00), "e4m3")
    top = 1.875 * 2.0**127
    assert byte.tolist() == [[247]] and v[0, 0, :5].tolist() == [top, top, top, -top, 2.0**127]
    # int8, scale 2^122: codes 63 and 64 stand for 1.96875 2^127 and 2^128; halfway is 1.984375 2^127, 0x7f7e
    v, byte = lowbit.kv8_values(_block(0x7F7F, 0x7F7E, 0x7F7D, 0xFF7F, 0x7F00), "int8")
    top = 1.96875 * 2.0**127
    assert byte.tolist() == [[249]] and v[0, 0, :5].tolist() == [top, top, top, -top, 2.0**127]
    # one bit less as the largest and the scale is 2^121, where the last code is 127
    v, byte = lowbit.kv8_values(_block(0x7F7E), "int8")
    assert byte.tolist() == [[248]] and v[0, 0, 0] == 1.984375 * 2.0**127


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_every_value_is_a_finite_bf16(fmt):
    for top in range(0x7E00, 0x7F80):
        x = _block(*range(top, top - 64, -1))
        v, _ = lowbit.kv8_values(x, fmt)
        assert np.abs(v).max() < 2.0**128
        assert (bf16.round_f32(v.astype(np.float32)) == v).all()
