"""What the int4 projections refuse: no device call is made."""

import pytest


class On:
    """A stand-in for a device tensor: an address and a size."""

    def __init__(self, count, address=0x10000, item=2):
        self.address, self.numel, self.nbytes = address, count, item * count


def args(**change):
    a = dict(x=On(2 * 128), codes=On(8 * 64, item=1), scales=On(8), zeros=On(8), group=128,
             bias=On(8), out=On(16, 0x20000), rows=2, in_features=128, out_features=8)
    a.update(change)
    return a


@pytest.mark.parametrize("change,word", [
    (dict(group=16), "groups of 32, 64 or 128"),
    (dict(group=64, in_features=96), "whole groups"),
    (dict(out_features=-1), "negative"),
    (dict(rows=-1), "negative"),
    (dict(x=On(255)), "x holds 255"),
    (dict(codes=On(511, item=1)), "codes holds 511"),
    (dict(scales=On(7)), "scales holds 14"),
    (dict(zeros=On(7)), "zeros holds 14"),
    (dict(bias=On(7)), "bias holds 7"),
    (dict(out=On(15, 0x20000)), "out holds 15"),
    (dict(out=On(256)), "over its input"),
    (dict(x=On(256, 0x10008)), "16-byte aligned"),
    (dict(codes=On(512, 0x10008, item=1)), "16-byte aligned"),
])
def test_linear_int4_refuses(change, word):
    from microinfer import _microinfer as m
    with pytest.raises(ValueError, match=word):
        m.device.linear_int4(**args(**change))


@pytest.mark.parametrize("change,word", [
    (dict(in_features=0, x=On(0), codes=On(0), scales=On(0), zeros=On(0)), "at least one group"),
    (dict(rows=65535 * 64 + 1, x=On(1 << 40), out=On(1 << 40, 0x20000)), "rows"),
    (dict(in_features=(1 << 24) + 128, x=On(1 << 40), codes=On(1 << 40, item=1),
          scales=On(1 << 40), zeros=On(1 << 40)), "16777216 in_features"),
    (dict(out_features=(1 << 27) + 1, codes=On(1 << 40, item=1), scales=On(1 << 40),
          zeros=On(1 << 40), bias=None, out=On(1 << 40, 0x20000)), "134217728 out_features"),
])
def test_linear_int4_refuses_sizes(change, word):
    from microinfer import _microinfer as m
    with pytest.raises(ValueError, match=word):
        m.device.linear_int4(**args(**change))


def test_accumulate_and_quantise_refuse():
    from microinfer import _microinfer as m
    a = args()
    del a["bias"]
    a["out"] = On(15, item=4)
    with pytest.raises(ValueError, match="out needs 16 floats"):
        m.device.linear_int4_accumulate(**a)
    q = dict(weight=On(8 * 128), codes=On(512, item=1), scales=On(8), zeros=On(8), group=128,
             in_features=128, out_features=8)
    for change, word in ((dict(weight=On(1023)), "weight holds 1023"), (dict(group=0), "groups of"),
                         (dict(weight=On(1024, 0x10002)), "aligned"),
                         (dict(codes=On(511, item=1)), "codes holds 511")):
        with pytest.raises(ValueError, match=word):
            m.device.quantise_int4(**{**q, **change})


def test_nothing_to_do_is_done():
    from microinfer import _microinfer as m
    m.device.linear_int4(**args(rows=0))
    m.device.linear_int4(**args(out_features=0))
