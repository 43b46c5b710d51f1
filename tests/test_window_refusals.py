"""What window attention refuses: no device call is made."""

import pytest

from test_int4_refusals import On


def args(**change):
    a = dict(q=On(3 * 4 * 64), k=On(5 * 2 * 64, 0x20000), v=On(5 * 2 * 64, 0x30000),
             out=On(3 * 4 * 64, 0x40000), seq_q=3, seq_k=5, heads=4, kv_heads=2, head_dim=64,
             window=2, sinks=1)
    a.update(change)
    return a


@pytest.mark.parametrize("change,word", [
    (dict(seq_q=-1), "negative"),
    (dict(seq_q=6), "exceeds seq_k"),
    (dict(window=-1), "negative"),
    (dict(sinks=-1), "negative"),
    (dict(k_stride=-128), "negative"),
    (dict(q=On(767)), "q holds 767"),
    (dict(k=On(639, 0x20000)), "k holds 639"),
    (dict(v=On(639, 0x30000)), "v holds 639"),
    (dict(out=On(767, 0x40000)), "out holds 767"),
    (dict(q=On(10**6), q_stride=248), "strides"),
    (dict(k=On(10**6, 0x20000), k_stride=64), "strides"),
    (dict(k=On(10**6, 0x20000), k_stride=132), "aligned"),
    (dict(k_stride=136), "k holds 640"),
    (dict(q=On(768, 0x10008)), "aligned"),
    (dict(partials=On(100, 0x50008, 4)), "aligned"),
    (dict(out=On(768)), "over its queries"),
    (dict(out=On(768, 0x20000)), "keys or values"),
    (dict(out=On(768, 0x30000)), "keys or values"),
    (dict(head_dim=32), "head_dim 64 or 128"),
    (dict(kv_heads=3, k=On(10**6, 0x20000), v=On(10**6, 0x30000)), "whole number"),
    (dict(seq_k=0x7fffff01, k=On(1 << 50, 0x20000), v=On(1 << 50, 0x30000)), "exceeds window"),
])
def test_attention_window_refuses(change, word):
    from microinfer import _microinfer as m
    with pytest.raises(ValueError, match=word):
        m.device.attention_window(**args(**change))


def test_partials_that_are_too_few_are_refused_and_nothing_to_do_is_done():
    from microinfer import _microinfer as m
    need = m.device.attention_window_partials(1, 4096, 4, 2, 64)
    assert need > 0
    with pytest.raises(ValueError, match="partials need"):
        m.device.attention_window(**args(seq_q=1, seq_k=4096, window=0, k=On(1 << 20, 0x200000),
                                         v=On(1 << 20, 0x600000), partials=On(need - 1, 0x50000, 4)))
    m.device.attention_window(**args(seq_q=0))
    m.device.attention_window(**args(seq_q=0, seq_k=0))
    assert m.device.attention_window_partials(0, 0, 4, 2, 64) == 0
    assert m.device.attention_window_partials(4096, 4096, 32, 8, 64) == 0
