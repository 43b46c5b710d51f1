"""What a ragged batch's operators refuse, overlaps among it: no device call is made."""

import pytest

from test_int4_refusals import On


def device():
    from microinfer import _microinfer as m
    return m.device


# -- append ------------------------------------------------------------------------------

def append_args(**change):
    a = dict(q=On(6 * 256, 0x10000), k=On(6 * 128, 0x20000), v=On(6 * 128, 0x30000),
             q_out=On(6 * 256, 0x40000), k_out=On(6 * 128, 0x50000), pages=On(6, 0x60000, 8),
             tiers=On(6, 0x61000, 1), lengths=On(2, 0x62000, 4), offsets=On(3, 0x63000, 4), batch=2,
             max_pages=3, rows=6, rope=None, heads=4, kv_heads=2, head_dim=64)
    a.update(change)
    return a


@pytest.mark.parametrize("change,word", [
    (dict(batch=-1), "negative"), (dict(max_pages=-1), "negative"), (dict(rows=-1), "negative"),
    (dict(heads=-1), "negative"), (dict(q_stride=-8), "negative"), (dict(v_stride=-8), "negative"),
    (dict(q=On(6 * 256 - 1)), "q holds 1535"), (dict(k=On(767)), "k holds 767"),
    (dict(v=On(767)), "v holds 767"), (dict(q_out=On(1535, 0x40000)), "q_out holds 1535"),
    (dict(k_out=On(767, 0x50000)), "k_out holds 767"), (dict(v_out=On(767, 0x70000)), "v_out holds 767"),
    (dict(pages=On(5, item=8)), "pages holds 5"), (dict(tiers=On(5, item=1)), "tiers holds 5"),
    (dict(lengths=On(1, item=4)), "lengths holds 1"), (dict(offsets=On(2, item=4)), "offsets holds 2"),
    (dict(head_dim=63), "even head_dim"), (dict(heads=0), "query and KV heads"),
    (dict(kv_heads=0), "query and KV heads"), (dict(q_stride=255, q=On(9999)), "strides"),
    (dict(k_stride=120, k=On(9999, 0x20000)), "strides"), (dict(offsets=None), "one row"),
    (dict(q_out=On(1536, 0x10000 + 1536 * 2 - 2)), "over what it reads"),
    (dict(q_out=On(1536, 0x20010)), "over what it reads"),
    (dict(k_out=On(768, 0x30000 - 16)), "over what it reads"),
    (dict(k_out=On(768, 0x60010)), "over what it reads"),
    (dict(k_out=On(768, 0x61004)), "over what it reads"),
    (dict(v_out=On(768, 0x62004)), "over what it reads"),
    (dict(v_out=On(768, 0x63008)), "over what it reads"),
    (dict(k_out=On(768, 0x40010)), "over one another"),
    (dict(v_out=On(768, 0x50010)), "over one another"),
])
def test_append_batch_refuses(change, word):
    with pytest.raises(ValueError, match=word):
        device().append_batch(**append_args(**change))


def test_append_refuses_too_wide_rows_and_tables_that_cover_too_little():
    big = 1 << 40
    with pytest.raises(ValueError, match="channels"):
        device().append_batch(**append_args(heads=1 << 20, q=On(big), q_out=On(big, 1 << 50)))
    rope = device().RopeTable(64, 1e4)  # covers nothing yet
    with pytest.raises(ValueError, match="covers 0"):
        device().append_batch(**append_args(rope=rope))
    wide = device().RopeTable(128, 1e4)
    with pytest.raises(ValueError, match="turns 128"):
        device().append_batch(**append_args(rope=wide))


def test_append_caches_refuses_lists_that_do_not_match():
    a = append_args(v_out=None)
    for name in ("pages", "tiers", "lengths", "offsets", "batch", "max_pages", "rows"):
        del a[name]
    d = device()
    d.append_caches([], [], [], 0, **a)
    with pytest.raises(ValueError, match="1 caches, 2 starts"):
        d.append_caches([object()], [0, 1], [1], 0, **a)
    with pytest.raises(ValueError, match="negative"):
        d.append_caches([object()], [0], [-1], 0, **a)


def test_nothing_to_append_is_done():
    device().append_batch(**append_args(rows=0))
    device().append_batch(**append_args(batch=0, offsets=On(1, 0x63000, 4)))


# -- packed attention --------------------------------------------------------------------

def packed_args(**change):
    a = dict(q=On(3 * 256, 0x10000), k=On(5 * 128, 0x20000), v=On(5 * 128, 0x30000),
             out=On(768, 0x40000), offsets_q=On(3, 0x50000, 4), offsets_k=On(3, 0x51000, 4), batch=2,
             rows_q=3, rows_k=5, heads=4, kv_heads=2, head_dim=64)
    a.update(change)
    return a


@pytest.mark.parametrize("change,word", [
    (dict(batch=-1), "negative"), (dict(rows_q=-1), "negative"), (dict(rows_k=-1), "negative"),
    (dict(k_stride=-8), "negative"), (dict(q=On(767)), "q holds 767"), (dict(k=On(639)), "k holds 639"),
    (dict(v=On(639)), "v holds 639"), (dict(out=On(767, 0x40000)), "out holds 767"),
    (dict(offsets_q=On(2, item=4)), "offsets_q holds 2"),
    (dict(offsets_k=On(2, item=4)), "offsets_k holds 2"),
    (dict(head_dim=32), "head_dim 64 or 128"), (dict(kv_heads=3, k=On(9999), v=On(9999)), "whole number"),
    (dict(kv_heads=0), "whole number"), (dict(rows_k=0), "needs keys"),
    (dict(q=On(768, 0x10008)), "16-byte aligned"), (dict(out=On(768, 0x40002)), "16-byte aligned"),
    (dict(k=On(9999, 0x20000), k_stride=132), "16-byte aligned"),
    (dict(offsets_q=On(3, 0x50002, 4)), "4-byte"),
    (dict(k=On(9999, 0x20000), k_stride=120), "strides"),
    (dict(out=On(768, 0x10010)), "over its queries"), (dict(out=On(768, 0x20000 + 1264)), "keys"),
    (dict(out=On(768, 0x30000 - 16)), "values"), (dict(out=On(768, 0x50000 - 1536 + 16)), "offsets"),
    (dict(partials=On(1 << 20, 0x30004, 4)), "16-byte aligned"),
])
def test_attention_packed_refuses(change, word):
    with pytest.raises(ValueError, match=word):
        device().attention_packed(**packed_args(**change))


def test_partials_of_packed_attention():
    d = device()
    need = d.attention_packed_partials
    assert need(4, 0, 0, 4, 2, 64) == 0
    floats = need(1, 1, 4096, 4, 2, 64)
    assert floats > 0
    keys = dict(batch=1, rows_q=1, rows_k=4096, k=On(1 << 20, 0x200000), v=On(1 << 20, 0x600000))
    with pytest.raises(ValueError, match="partials need"):
        d.attention_packed(**packed_args(**keys, partials=On(floats - 1, 0x900000, 4)))
    for at in (0x200000, 0x40000, 0x10000, 0x50000):
        with pytest.raises(ValueError, match="write over|partials"):
            d.attention_packed(**packed_args(**keys, partials=On(floats, at, 4)))
    for heads, kv, hd in ((14, 2, 64), (12, 2, 128), (32, 8, 64), (40, 1, 64), (128, 8, 128)):
        for rows in list(range(1, 130)) + [200, 333, 500, 777, 1024, 1500, 2000, 3000, 5000, 9999]:
            for keys in (rows, rows + 1000, rows + 100000):
                for batch in (1, 5, 100):
                    assert need(batch, rows, keys, heads, kv, hd) <= 65536 * (hd + 2)


def test_no_queries_are_done():
    device().attention_packed(**packed_args(rows_q=0, rows_k=0))
    device().attention_packed(**packed_args(batch=0))


# -- 8 bits ------------------------------------------------------------------------------

def int8_args(**change):
    a = dict(x=On(3 * 64, 0x10000, 1), x_scales=On(3, 0x11000, 4), weight=On(8 * 64, 0x12000, 1),
             w_scales=On(8, 0x13000, 4), bias=On(8, 0x14000), out=On(24, 0x20000), rows=3,
             in_features=64, out_features=8)
    a.update(change)
    return a


@pytest.mark.parametrize("change,word", [
    (dict(rows=-1), "negative"), (dict(out_features=-1), "negative"), (dict(in_features=-16), "negative"),
    (dict(in_features=40), "whole sixteens"), (dict(x=On(191, item=1)), "x holds 191"),
    (dict(x_scales=On(2, item=4)), "x_scales needs 3"), (dict(weight=On(511, item=1)), "weight holds 511"),
    (dict(w_scales=On(7, item=4)), "w_scales needs 8"), (dict(bias=On(7)), "bias holds 7"),
    (dict(out=On(23, 0x20000)), "out holds 23"), (dict(in_features=0), "in_features"),
    (dict(in_features=1 << 17, x=On(1 << 30, 0x10000, 1), weight=On(1 << 30, 1 << 40, 1)), "131056"),
    (dict(rows=(1 << 21) + 1, x=On(1 << 40, 1 << 50, 1), x_scales=On(1 << 40, 1 << 54, 4),
          out=On(1 << 40, 1 << 58)), "2097152 rows"),
    (dict(x=On(192, 0x10008, 1)), "16-byte aligned"), (dict(weight=On(512, 0x12004, 1)), "16-byte aligned"),
    (dict(out=On(24, 0x20008)), "16-byte aligned"), (dict(out=On(24, 0x10000)), "write over"),
    (dict(out=On(24, 0x12000 + 496)), "write over"), (dict(out=On(24, 0x14000)), "write over"),
    (dict(out=On(24, 0x13010)), "write over"), (dict(out=On(24, 0x11000 - 32)), "write over"),
])
def test_linear_int8_refuses(change, word):
    with pytest.raises(ValueError, match=word):
        device().linear_int8(**int8_args(**change))


def test_int8_accumulate_and_quantise_refuse():
    d = device()
    a = int8_args(out=On(24, 0x20000, 4))
    del a["bias"]
    for change, word in ((dict(out=On(23, 0x20000, 4)), "out needs 24"),
                         (dict(residual=On(23, 0x30000, 4)), "residual needs 24"),
                         (dict(residual=On(24, 0x20010, 4)), "write over"),
                         (dict(residual=On(24, 0x30004, 4)), "16-byte aligned")):
        with pytest.raises(ValueError, match=word):
            d.linear_int8_accumulate(**{**a, **change})
    q = dict(x=On(3 * 64, 0x10000), codes=On(192, 0x20000, 1), scales=On(3, 0x30000, 4), rows=3,
             features=64)
    for change, word in ((dict(rows=-1), "negative"), (dict(stride=-8), "negative"),
                         (dict(features=8), "whole sixteens"), (dict(features=0), "have values"),
                         (dict(x=On(191)), "x holds 191"), (dict(codes=On(191, 0x20000, 1)), "codes holds"),
                         (dict(scales=On(2, 0x30000, 4)), "scales needs 3"),
                         (dict(stride=68, x=On(999, 0x10000)), "multiple of 8"),
                         (dict(stride=56, x=On(999, 0x10000)), "apart"),
                         (dict(x=On(192, 0x10008)), "16-byte aligned"),
                         (dict(codes=On(192, 0x10010, 1)), "write over"),
                         (dict(scales=On(3, 0x10000 + 380, 4)), "write over"),
                         (dict(scales=On(3, 0x20010, 4)), "write over")):
        with pytest.raises(ValueError, match=word):
            d.quantise_rows_int8(**{**q, **change})
    d.quantise_rows_int8(**{**q, "rows": 0})
    d.linear_int8(**int8_args(rows=0))
    d.linear_int8(**int8_args(out_features=0))


# -- sampling ----------------------------------------------------------------------------

SCRATCH = 1 << 16  # floats, more than three rows of 100 logits take


def sample_args(**change):
    a = dict(logits=On(300, 0x10000, 4), uniforms=On(3, 0x20000, 4), tokens=On(3, 0x30000, 4), rows=3,
             vocab=100, scratch=On(SCRATCH, 0x40000, 4))
    a.update(change)
    return a


@pytest.mark.parametrize("change,word", [
    (dict(rows=-1), "negative"), (dict(vocab=-1), "negative"), (dict(stride=-1), "negative"),
    (dict(logits=On(299, item=4)), "logits needs 300"), (dict(uniforms=On(2, item=4)), "uniforms needs 3"),
    (dict(tokens=On(2, item=4)), "tokens holds 2"), (dict(temperature=On(2, item=4)), "temperature holds"),
    (dict(top_k=On(2, item=4)), "top_k holds 2"), (dict(top_p=On(2, item=4)), "top_p holds 2"),
    (dict(min_p=On(2, item=4)), "min_p holds 2"), (dict(scratch=None), "scratch needs"),
    (dict(stride=99), "apart"),
    (dict(vocab=0), "a token at least"),
    (dict(vocab=(1 << 20) + 1, logits=On(1 << 30, item=4)), "1048576"),
    (dict(rows=65536, logits=On(1 << 30, item=4), uniforms=On(1 << 20, item=4),
          tokens=On(1 << 20, item=4)), "65535 rows"),
    (dict(scratch=On(SCRATCH, 0x40008, 4)), "aligned"), (dict(logits=On(300, 0x10002, 4)), "aligned"),
    (dict(top_k=On(3, 0x50002, 4)), "aligned"), (dict(tokens=On(3, 0x10000, 4)), "write over"),
    (dict(tokens=On(3, 0x20004, 4)), "write over"), (dict(top_p=On(3, 0x30008, 4)), "write over"),
    (dict(scratch=On(SCRATCH, 0x10000, 4)), "write over"), (dict(scratch=On(SCRATCH, 0x30000 - 16, 4)), "lies over"),
])
def test_sample_refuses(change, word):
    with pytest.raises(ValueError, match=word):
        device().sample_f32(**sample_args(**change))


def test_sampling_scratch_grows_and_no_rows_are_done():
    d = device()
    assert d.sample_scratch(0, 1000) == 0
    need = d.sample_scratch(3, 100)
    assert need < SCRATCH
    with pytest.raises(ValueError, match=f"scratch needs {need} floats; got {need - 1}"):
        d.sample_f32(**sample_args(scratch=On(need - 1, 0x40000, 4)))
    sizes = [d.sample_scratch(3, v) for v in range(0, 60000, 511)]
    assert sizes == sorted(sizes)
    assert d.sample_scratch(4, 9000) > d.sample_scratch(3, 9000)
    d.sample_f32(**sample_args(rows=0))
    with pytest.raises(ValueError, match="logits holds 299"):
        d.sample(**sample_args(logits=On(299, item=2)))


# -- scaled angles -----------------------------------------------------------------------

@pytest.mark.parametrize("scaling,word", [
    (dict(kind="dynamic", factor=2.0), "kind is one of"), (dict(factor=2.0), "kind is one of"),
    (dict(kind="linear"), "a linear scaling has"), (dict(kind="linear", factor=2.0, low=1.0), "has"),
    (dict(kind="linear", factor=0.5), "at least 1"), (dict(kind="linear", factor=float("nan")), "at least 1"),
    (dict(kind="llama3", factor=8.0, low=4.0, high=1.0, original=8192), "low < high"),
    (dict(kind="llama3", factor=8.0, low=1.0, high=4.0, original=0), "original context"),
    (dict(kind="yarn", factor=4.0, original=4096, fast=1.0, slow=2.0), "slow <= fast"),
    (dict(kind="yarn", factor=4.0, original=4096, magnitude=0.0), "magnitude must be positive"),
])
def test_rope_scalings_refuse(scaling, word):
    with pytest.raises(ValueError, match=word):
        device().RopeTable(64, 1e4, scaling)


def test_rope_tables_refuse():
    d = device()
    for hd, theta, word in ((7, 1e4, "positive and even"), (0, 1e4, "positive and even"),
                            (64, -1.0, "theta")):
        with pytest.raises(ValueError, match=word):
            d.RopeTable(hd, theta, dict(kind="linear", factor=2.0))
    with pytest.raises(ValueError, match="frequencies must be finite"):
        d.RopeTable(64, 1e-320, dict(kind="linear", factor=2.0))
