"""The serving operators refuse to write over what other workgroups still read:
any overlap, not equal addresses alone. No device call is made."""

import pytest

import test_batch_refusals as batch
import test_int4_refusals as int4
import test_window_refusals as window
from test_int4_refusals import On

# q 3 x 256 halves at 0x10000, k and v 5 x 128 at 0x20000 and 0x30000.
Q, K, V, ROW = 0x10000, 0x20000, 0x30000, 512


@pytest.mark.parametrize("change,word", [
    (dict(out=On(768, Q + 2 * ROW)), "over its queries"),       # its first row on q's last
    (dict(out=On(768, Q - 3 * ROW + 16)), "over its queries"),  # its last bytes on q's first
    (dict(out=On(768, K + 1280 - 16)), "keys or values"),
    (dict(out=On(768, V - 3 * ROW + 16)), "keys or values"),
])
def test_window_attention_refuses_any_overlap(change, word):
    from microinfer import _microinfer as m
    with pytest.raises(ValueError, match=word):
        m.device.attention_window(**window.args(**change))


def test_window_attention_refuses_rows_of_the_fused_buffer_it_reads():
    """q, k and v in rows of 512 halves (heads 4, kv 2, head_dim 64): an out that starts among the
    rows meets keys; partials too."""
    from microinfer import _microinfer as m
    d = m.device
    rows, width = 40, 512

    def call(at, partials=None):
        d.attention_window(On(rows * width, Q), On(rows * width - 256, Q + 512),
                           On(rows * width - 384, Q + 768), On(rows * 256, at), rows, rows, 4, 2, 64,
                           0, 0, q_stride=width, k_stride=width, v_stride=width, partials=partials)

    end = Q + 2 * rows * width
    for at in (Q + 1024, Q + 1024 * (rows - 1) + 512, end - 16, Q - rows * 512 + 16):
        with pytest.raises(ValueError, match="cannot write over"):
            call(at)
    floats = d.attention_window_partials(1, 4096, 4, 2, 64)
    keys = dict(seq_q=1, seq_k=4096, window=0, k=On(1 << 20, 0x200000), v=On(1 << 20, 0x600000))
    for at in (0x200000, 0x600000 + (1 << 20) - 64, Q, 0x40000):
        with pytest.raises(ValueError, match="cannot write over|partials"):
            d.attention_window(**window.args(**keys, partials=On(floats, at, 4)))


@pytest.mark.parametrize("change", [
    dict(out=On(512, 0x10010)), dict(out=On(512, 0x10000 - 1024 + 16)),
    dict(out=On(512, 0x50000), lengths=On(2, 0x503f8, 4)),
    dict(out=On(512, 0x50000), pages=On(6, 0x50200, 8)),
    dict(out=On(512, 0x50000), tiers=On(6, 0x503ff, 1)),
    dict(mass=On(24, 0x20000 + 1020, 4), partials=On(1 << 20, 0x40000, 4)),
    dict(mass=On(24, 0x30000, 4), partials=On(24, 0x30050, 4)),
    dict(mass=On(24, 0x30000, 4), partials=On(24, 0x10000, 4)),
])
def test_batch_attention_refuses_any_overlap(change):
    from microinfer import _microinfer as m
    apart = dict(lengths=On(2, 0x90000, 4), pages=On(6, 0x91000, 8), tiers=On(6, 0x92000, 1))
    with pytest.raises(ValueError, match="write over"):
        m.device.attention_batch(**batch.args(**{**apart, **change}))


APART = dict(x=On(256, 0x10000), codes=On(512, 0x11000, 1), scales=On(8, 0x12000),
             zeros=On(8, 0x13000), bias=On(8, 0x14000), out=On(16, 0x20000))


@pytest.mark.parametrize("at", [0x10000 + 510, 0x10000 - 16, 0x11000 + 511, 0x12000 + 14, 0x13000 + 2,
                                0x14000 - 30])
def test_int4_projections_refuse_any_overlap(at):
    from microinfer import _microinfer as m
    with pytest.raises(ValueError, match="write over its input"):
        m.device.linear_int4(**int4.args(**{**APART, "out": On(16, at)}))
    if at < 0x14000 - 30:
        a = int4.args(**{**APART, "out": On(16, at & ~3, 4)})
        del a["bias"]
        with pytest.raises(ValueError, match="write over its input"):
            m.device.linear_int4_accumulate(**a)


@pytest.mark.parametrize("change", [
    dict(codes=On(512, 0x10800 - 16, 1)), dict(scales=On(8, 0x10400)), dict(zeros=On(8, 0x10000 - 2)),
    dict(scales=On(8, 0x11000 + 510)), dict(zeros=On(8, 0x12000 + 14)),
])
def test_quantise_int4_refuses_any_overlap(change):
    from microinfer import _microinfer as m
    q = dict(weight=On(8 * 128, 0x10000), codes=On(512, 0x11000, 1), scales=On(8, 0x12000),
             zeros=On(8, 0x13000), group=128, in_features=128, out_features=8)
    with pytest.raises(ValueError, match="write over"):
        m.device.quantise_int4(**{**q, **change})
