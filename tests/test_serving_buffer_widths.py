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
