"""Buffers of enough elements but too few bytes, which the serving operators
must refuse before any device call: tables of 64-bit addresses and 32-bit
lengths given in narrower elements, fp32 scratch and masses given as fp16."""

import pytest

import test_batch_refusals as batch
import test_window_refusals as window
from test_int4_refusals import On


@pytest.mark.parametrize("change,word", [
    (dict(pages=On(6, item=4)), "pages holds 3 entries of 8 bytes"),
    (dict(pages=On(6, item=2)), "pages holds 1 "),
    (dict(pages=On(6, item=1)), "pages holds 0 "),
    (dict(lengths=On(2, item=2)), "lengths holds 1 "),
    (dict(lengths=On(2, item=1)), "lengths holds 0 "),
    (dict(mass=On(24, 0x30000, 2), partials=On(1 << 20, 0x40000, 4)), "mass needs 24 floats"),
])
def test_attention_batch_refuses_narrow_tables(change, word):
    from microinfer import _microinfer as m
    with pytest.raises(ValueError, match=word):
        m.device.attention_batch(**batch.args(**change))


def test_partials_count_as_floats():
    """The floats asked for, in fp16 elements: half of the bytes."""
    from microinfer import _microinfer as m
    d = m.device
    need = d.attention_batch_partials(1, 1024, 4, 2, 64)
    long = batch.args(batch=1, max_pages=1024, pages=On(1024, item=8), tiers=On(1024, item=1))
    with pytest.raises(ValueError, match=f"partials need {need} floats; got {need // 2}"):
        d.attention_batch(**{**long, "partials": On(need, 0x40000, 2)})
    need = d.attention_window_partials(1, 4096, 4, 2, 64)
    keys = dict(seq_q=1, seq_k=4096, window=0, k=On(1 << 20, 0x200000), v=On(1 << 20, 0x600000))
    with pytest.raises(ValueError, match=f"partials need {need} floats; got {need // 2}"):
        d.attention_window(**window.args(**keys, partials=On(need, 0x50000, 2)))


def test_a_table_in_int32_words_holds_half_as_many_addresses():
    """DeviceIndex is the package's own integer array: its bytes are what counts."""
    from microinfer import _microinfer as m

    class Words(m.DeviceIndex):
        def __init__(self, count, address):  # no device here
            self.count, self._storage = count, type("At", (), dict(ptr=address))()

    with pytest.raises(ValueError, match="pages holds 5 entries of 8 bytes"):
        m.device.attention_batch(**batch.args(pages=Words(11, 0x10000)))
    assert Words(12, 0).nbytes == 48
    with pytest.raises(ValueError, match="tiers holds 4 entries"):
        m.device.attention_batch(**batch.args(pages=Words(12, 0x10000), tiers=Words(1, 0x30000)))


@pytest.mark.parametrize("change,word", [
    (dict(q=On(768, item=1)), "q holds 384"), (dict(k=On(640, 0x20000, 1)), "k holds 320"),
    (dict(v=On(640, 0x30000, 1)), "v holds 320"), (dict(out=On(768, 0x40000, 1)), "out holds 384"),
])
def test_attention_window_refuses_bytes_for_halves(change, word):
    from microinfer import _microinfer as m
    with pytest.raises(ValueError, match=word):
        m.device.attention_window(**window.args(**change))


def test_the_others_refuse_bytes_for_halves():
    import test_int4_refusals as int4
    from microinfer import _microinfer as m
    for name, count in (("q", 512), ("out", 512)):
        with pytest.raises(ValueError, match=f"{name} holds {count // 2}"):
            m.device.attention_batch(**batch.args(**{name: On(count, 0x20000, 1)}))
    for name, count in (("x", 256), ("bias", 8), ("out", 16)):
        with pytest.raises(ValueError, match=f"{name} holds {count // 2}"):
            m.device.linear_int4(**int4.args(**{name: On(count, 0x20000, 1)}))
    q = dict(weight=On(8 * 128, item=1), codes=On(512, item=1), scales=On(8), zeros=On(8), group=128,
             in_features=128, out_features=8)
    with pytest.raises(ValueError, match="weight holds 512"):
        m.device.quantise_int4(**q)
