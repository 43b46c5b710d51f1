"""What a server keeps once for every prompt's window attention: no sizes ask for
more partials than 65,536 rows' parts (512 workgroups of 128 rows, or 256 of 32,
are the most that a launch with parts has), head_dim + 2 floats each."""

import itertools

import pytest


@pytest.mark.parametrize("heads,kv", [(14, 2), (12, 2), (32, 8), (4, 4), (6, 2), (40, 1), (64, 64),
                                      (2048, 1)])
@pytest.mark.parametrize("hd", [64, 128])
def test_partials_are_bounded(heads, kv, hd):
    from microinfer import _microinfer as m
    need = m.device.attention_window_partials.__wrapped__
    most = 0
    for seq_q, past, window, sinks in itertools.product(
            (1, 2, 3, 16, 33, 100, 129, 300, 500, 680, 1000, 1365, 2047, 2726, 4000, 5461, 8191, 16384,
             40000), (0, 60, 3000, 14336, 300000), (0, 1, 64, 1024, 4096, 100000), (0, 4, 5000)):
        most = max(most, need(seq_q, seq_q + past, heads, kv, hd, window, sinks))
    assert 0 < most <= 65536 * (hd + 2)
