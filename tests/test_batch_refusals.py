"""What the batch's decode refuses: no device call is made."""

import pytest

from test_int4_refusals import On


def args(**change):
    a = dict(q=On(2 * 4 * 64), pages=On(6, item=8), tiers=On(6, item=1), lengths=On(2, item=4),
             out=On(2 * 4 * 64, 0x20000), batch=2, max_pages=3, heads=4, kv_heads=2, head_dim=64,
             window=0, sinks=0, mass=None, partials=None)
    a.update(change)
    return a


@pytest.mark.parametrize("change,word", [
    (dict(batch=-1), "negative"),
    (dict(max_pages=-1), "negative"),
    (dict(window=-1), "negative"),
    (dict(sinks=-2), "negative"),
    (dict(q=On(511)), "q holds 511"),
    (dict(out=On(511, 0x20000)), "out holds 511"),
    (dict(pages=On(5, item=8)), "pages holds 5"),
    (dict(tiers=On(5, item=1)), "tiers holds 5"),
    (dict(lengths=On(1, item=4)), "lengths holds 1"),
    (dict(mass=On(23, item=4)), "mass needs 24"),
    (dict(mass=On(24, item=4)), "masses need partials"),
    (dict(mass=On(24, item=4), partials=On(23, 0x30000, 4)), "partials need"),
    (dict(head_dim=32), "head_dim 64 or 128"),
    (dict(head_dim=128), "q holds 512"),
    (dict(kv_heads=3), "whole number of query heads"),
    (dict(kv_heads=0), "whole number of query heads"),
    (dict(heads=34, q=On(1 << 20), out=On(1 << 20, 0x200000)), "at most 16"),
    (dict(q=On(512, 0x10008)), "16-byte aligned"),
    (dict(out=On(512, 0x20004)), "16-byte aligned"),
    (dict(partials=On(1 << 20, 0x30004, 4)), "16-byte aligned"),
    (dict(out=On(512)), "over its queries"),
])
def test_attention_batch_refuses(change, word):
    from microinfer import _microinfer as m
    with pytest.raises(ValueError, match=word):
        m.device.attention_batch(**args(**change))


def test_sizes_past_the_launch_are_refused():
    from microinfer import _microinfer as m
    big = 1 << 40
    for change, word in ((dict(batch=65536), "65535"), (dict(max_pages=1 << 27), "pages a sequence")):
        a = args(q=On(big), pages=On(big, item=8), tiers=On(big, item=1), lengths=On(big, item=4),
                 out=On(big, 0x20000), **change)
        with pytest.raises(ValueError, match=word):
            m.device.attention_batch(**a)


def test_an_empty_batch_is_done_and_caches_must_match_their_positions():
    from microinfer import _microinfer as m
    m.device.attention_batch(**args(batch=0))
    m.device.attention_caches([], [], 0, On(0), On(0, 0x20000), 4, 2, 64)
    with pytest.raises(ValueError, match="1 caches and 2"):
        m.device.attention_caches([object()], [1, 2], 0, On(256), On(256, 0x20000), 4, 2, 64)


def test_partials_grow_with_what_is_asked():
    from microinfer import _microinfer as m
    need = m.device.attention_batch_partials
    assert need(4, 2, 4, 2, 64) == 0  # one run a sequence
    assert need(1, 1024, 12, 2, 128) > 0
    assert need(1, 1024, 12, 2, 128, mass=True) == need(1, 1024, 12, 2, 128) + 12 * 1024
    assert need(1, 1024, 12, 2, 128, window=64, sinks=4) < need(1, 1024, 12, 2, 128)
    with pytest.raises(ValueError):
        need(1, 1024, 12, 2, 96)


@pytest.mark.parametrize("heads,kv,hd", [(14, 2, 64), (12, 2, 128), (32, 8, 64), (6, 3, 64)])
def test_partials_for_the_longest_and_most_do_for_less(heads, kv, hd):
    """A buffer made for a serving run's largest step: no shorter or smaller one asks for more."""
    from microinfer import _microinfer as m
    need = m.device.attention_batch_partials
    for window in (0, 700):
        for batch in (1, 3, 8, 48, 300):
            by_pages = [need(batch, p, heads, kv, hd, window, 4) for p in range(0, 1200, 7)]
            assert by_pages == sorted(by_pages)
    for pages in (1, 2, 3, 40, 1000):
        by_batch = [need(b, pages, heads, kv, hd) for b in range(0, 400)]
        assert by_batch == sorted(by_batch)
