"""Several prompts' attention in one run of rows: lengths from nothing on, head
layouts, cached prefixes, queries with no key, rows of no sequence, strides,
splits, values that are not finite where a row does not see them; against float64.

Tolerance as attention_window's: the fp32 sums' bound, half a step of fp16 for
every weight (2^-11 of the sums of p |v|; 2^-20 more for the hardware's
exponential) and for the output (2^-11 of it, 2^-25 below fp16's normals)."""

import numpy as np
import pytest

from conftest import announce, fp16_exact
from oracle import ragged
from test_gpu_int4 import Bytes
from test_gpu_kv_pages import mi, put

pytestmark = pytest.mark.gpu


def inputs(rng, rows, keys, heads, kv, hd):
    q, k, v = (rng.standard_normal((n, h, hd)) for n, h in ((rows, heads), (keys, kv), (keys, kv)))
    k[..., :2] *= 10
    return fp16_exact(q), fp16_exact(k), fp16_exact(v)


def offsets(counts, before=0):
    return before + np.concatenate([[0], np.cumsum(counts)]).astype(np.int64)


def attend(q, k, v, oq, ok, split, same=False):
    d = mi().device
    rows, heads, hd = q.shape
    keys, kv, _ = k.shape
    y = Bytes(count=2 * q.size)
    y.numel = q.size
    parts, batch = None, len(oq) - 1
    if split:
        parts = d.empty_f32(max(1, d.attention_packed_partials(batch, rows, keys, heads, kv, hd)))
    d.attention_packed(put(q), put(k), put(v), y, d.DeviceIndex(oq),
                       None if same else d.DeviceIndex(ok), batch, rows, keys, heads, kv, hd,
                       partials=parts)
    return y.read().view(np.float16).reshape(q.shape)


def check(got, q, k, v, oq, ok, what):
    want, bound, terms = ragged.packed_attention(q, k, v, oq, ok)
    none = np.isnan(want).all((1, 2))
    assert (got[none].view(np.uint16) == 0xA5A5).all(), f"{what}: rows of no sequence"
    got, want, bound, terms = got[~none].astype(np.float64), want[~none], bound[~none], terms[~none]
    assert np.isfinite(got).all(), f"{what}: not finite"
    limit = bound + (2.0**-11 + 2.0**-20) * terms + 2.0**-11 * np.abs(want) + 2.0**-25
    err = np.abs(got - want) / limit
    assert err.size == 0 or err.max() <= 1.0, f"{what}: {err.max():.3g} of the limit at {np.unravel_index(err.argmax(), err.shape)}"


@pytest.mark.parametrize("heads,kv,hd", [(14, 2, 64), (12, 2, 128), (32, 8, 64), (4, 4, 128),
                                         (5, 5, 64), (16, 1, 128), (40, 1, 64), (33, 3, 64)])
def test_head_layouts(heads, kv, hd):
    rng = np.random.default_rng(heads + hd)
    for counts in ([1], [1, 1, 1], [3, 0, 70, 1, 33], [200], [0, 0, 64, 0], [31, 32, 33, 128, 5]):
        o = offsets(counts)
        q, k, v = inputs(rng, o[-1], o[-1], heads, kv, hd)
        for split in (False, True):
            announce("packed", heads, kv, hd, counts, split)
            check(attend(q, k, v, o, o, split, same=True), q, k, v, o, o, f"{heads}/{kv}x{hd} {counts}")


@pytest.mark.parametrize("hd", [64, 128])
def test_prefixes_and_rows_with_no_key(hd):
    rng = np.random.default_rng(hd)
    for new, keys in (([5, 40, 1], [5, 300, 777]), ([1, 1, 1, 1], [1, 1000, 33, 64]),
                      ([30, 10, 4], [20, 0, 4]), ([64], [2000]), ([3, 0, 2], [0, 50, 100])):
        oq, ok = offsets(new), offsets(keys)
        q, k, v = inputs(rng, oq[-1], ok[-1], 6, 2, hd)
        for split in (False, True):
            announce("prefixes", hd, new, keys, split)
            check(attend(q, k, v, oq, ok, split), q, k, v, oq, ok, f"{new} of {keys}")


@pytest.mark.parametrize("hd", [64, 128])
def test_rows_and_keys_of_no_sequence(hd):
    rng = np.random.default_rng(10 + hd)
    oq, ok = offsets([40, 0, 9], 7), offsets([60, 5, 9], 11)
    q, k, v = inputs(rng, oq[-1] + 30, ok[-1] + 40, 6, 2, hd)
    k[:11], v[:11], k[ok[-1]:], v[ok[-1]:] = np.nan, np.inf, -np.inf, np.nan
    for split in (False, True):
        announce("no sequence", hd, split)
        check(attend(q, k, v, oq, ok, split), q, k, v, oq, ok, f"behind the last {split}")


@pytest.mark.parametrize("heads,kv,hd,new,past", [
    (32, 8, 64, [700, 1, 300, 0, 77], [0, 0, 0, 0, 0]), (12, 2, 128, [1500, 257, 64], [0, 0, 0]),
    (14, 2, 64, [1301, 640], [99, 0]), (28, 4, 128, [700, 3, 200], [3, 900, 64]),
    (32, 8, 64, [300, 200, 100], [1200, 64, 1]), (32, 8, 64, [40] * 30, [11] * 30),
    (12, 2, 128, [65] * 20, [500] * 20), (14, 2, 64, [160], [2440]), (12, 2, 128, [300], [2600])])
def test_many_rows(heads, kv, hd, new, past):
    """The large tiles: sequences that begin and end inside them, ragged last tiles."""
    rng = np.random.default_rng(sum(new) + hd)
    oq, ok = offsets(new), offsets(np.add(new, past))
    q, k, v = inputs(rng, oq[-1], ok[-1], heads, kv, hd)
    for split in (False, True):
        announce("many", heads, kv, hd, new, past, split)
        check(attend(q, k, v, oq, ok, split), q, k, v, oq, ok, f"{heads}/{kv}x{hd} {new} {past}")


@pytest.mark.parametrize("hd,rows", [(64, 40), (128, 40), (64, 1400), (128, 900)])
def test_values_not_seen_may_be_anything(hd, rows):
    """Each sequence's last value is infinite or NaN in a channel: only its last row sees it."""
    rng = np.random.default_rng(rows + hd)
    counts = [rows // 2, 7, rows // 2 - 7]
    o = offsets(counts)
    q, k, v = inputs(rng, o[-1], o[-1], 6, 2, hd)
    clean = v.copy()
    for i, bad in enumerate((np.inf, np.nan, -np.inf)):
        v[o[i + 1] - 1, :, 3 + i] = bad
        clean[o[i + 1] - 1, :, 3 + i] = 0
    for split in (False, True):
        announce("not finite", hd, rows, split)
        got = attend(q, k, v, o, o, split)
        last = o[1:] - 1
        keep = np.setdiff1d(np.arange(o[-1]), last)
        want, bound, terms = ragged.packed_attention(q, k, clean, o, o)
        limit = bound + (2.0**-11 + 2.0**-20) * terms + 2.0**-11 * np.abs(want) + 2.0**-25
        assert (np.abs(got[keep].astype(np.float64) - want[keep]) <= limit[keep]).all()
        for i, r in enumerate(last):
            assert not np.isfinite(got[r, :, 3 + i].astype(np.float64)).any()
            others = np.delete(np.arange(hd), 3 + i)
            assert (np.abs(got[r][:, others].astype(np.float64) - want[r][:, others]) <=
                    limit[r][:, others]).all()


@pytest.mark.parametrize("hd", [64, 128])
def test_views_of_one_projection(hd):
    rng = np.random.default_rng(hd)
    d = mi().device
    heads, kv, counts = 6, 2, [100, 31, 260]
    o = offsets(counts)
    q, k, v = inputs(rng, o[-1], o[-1], heads, kv, hd)
    fused = np.concatenate([x.reshape(len(x), -1) for x in (q, k, v)], 1)
    base, width = put(fused), fused.shape[1]
    cut = [0, heads * hd, (heads + kv) * hd]
    views = [d.view(base, at, fused.size - at) for at in cut]
    out = Bytes(count=2 * q.size)
    out.numel = q.size
    index = d.DeviceIndex(o)
    announce("fused", hd)
    d.attention_packed(*views, out, index, None, 3, o[-1], o[-1], heads, kv, hd, width, width, width)
    check(out.read().view(np.float16).reshape(q.shape), q, k, v, o, o, "fused")


def test_scores_far_below_zero_and_large():
    rng = np.random.default_rng(3)
    o = offsets([50, 60])
    q, k, v = inputs(rng, 110, 110, 4, 2, 64)
    q[:] = fp16_exact(np.abs(q))
    for k_ in (-np.abs(k) * 50, np.abs(k) * 50):
        k_ = fp16_exact(k_)
        announce("scores")
        check(attend(q, k_, v, o, o, True), q, k_, v, o, o, "scores")


@pytest.mark.parametrize("batch", [4096, 4097, 6000])
def test_more_sequences_than_are_held(batch):
    rng = np.random.default_rng(batch)
    o = offsets(rng.integers(0, 2, batch))
    q, k, v = inputs(rng, o[-1], o[-1], 2, 1, 64)
    announce("sequences", batch)
    check(attend(q, k, v, o, o, False), q, k, v, o, o, "sequences")


@pytest.mark.parametrize("heads,kv,hd", [(14, 2, 64), (12, 2, 128)])
def test_a_captured_call_follows_its_offsets(heads, kv, hd):
    m = mi()
    d = m.device
    rng = np.random.default_rng(hd)
    rows, batch = 300, 4
    q, k, v = inputs(rng, rows, rows, heads, kv, hd)
    on, out = [put(x) for x in (q, k, v)], Bytes(count=2 * q.size)
    out.numel = q.size
    index = d.DeviceIndex(np.zeros(batch + 1))
    parts = d.empty_f32(max(1, d.attention_packed_partials(batch, rows, rows, heads, kv, hd)))
    stream = m.Stream()
    graph = m.Graph(stream)
    with graph.capture():
        d.attention_packed(*on, out, index, None, batch, rows, rows, heads, kv, hd, partials=parts)
    for i in range(4):
        o = offsets(rng.multinomial(rows - 10 * i, [0.25] * 4))
        m._h2d(index.address, o.astype(np.int32))
        m._h2d(out.address, np.full(out.count, 0xA5, np.uint8))
        announce("captured packed", i)
        graph.launch()
        stream.synchronize()
        check(out.read().view(np.float16).reshape(q.shape), q, k, v, o, o, f"replay {i}")
