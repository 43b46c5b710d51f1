"""The int4 weight oracle: codes within half a step, the least scale that
reaches, constant groups, and the packing."""

import numpy as np
import pytest

from conftest import fp16_exact
from oracle import int4


@pytest.mark.parametrize("group", [32, 64, 128])
def test_weights_come_back_within_half_a_step(group):
    rng = np.random.default_rng(group)
    w = fp16_exact(rng.standard_normal((7, 3 * group)) * np.exp(rng.normal(0, 3, (7, 1))))
    w[2, :group] = w[2, 0]
    codes, scales, zeros = int4.quantise(w, group)
    got = int4.weight64(codes, scales, zeros, group)
    step = np.repeat(scales.astype(np.float64), group, axis=1)
    # Half a step, and the fp32 quotient's rounding (2^-24 of at most 15 steps, twice).
    assert (np.abs(got - w) <= step * (0.5 + 2.0**-19)).all()
    assert codes.max() == 15 and codes.min() == 0
    assert scales[2, 0] == 0 and (codes[2, :group] == 0).all()
    g = w.reshape(7, 3, group).astype(np.float64)
    reach = g.max(2) - g.min(2)
    assert (15 * scales.astype(np.float64) >= reach).all()
    below = np.nextafter(scales, np.float16(0)).astype(np.float64)
    assert ((15 * below < reach) | (scales == 0)).all()


def test_the_first_of_two_codes_is_in_the_low_bits():
    codes = np.arange(16, dtype=np.uint8).reshape(2, 8)
    assert int4.packed(codes).tolist() == [[0x10, 0x32, 0x54, 0x76], [0x98, 0xBA, 0xDC, 0xFE]]
