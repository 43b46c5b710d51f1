"""A prompt's attention through a sliding window with sinks on the device:
lengths from one token on, windows and sinks that end inside and on a step's
edge, head layouts, strides, splits, values that are not finite where a query
does not see them; against float64.

Tolerance: the fp32 sums' bound, half a step of fp16 for every weight (2^-11
of the sums of p |v|; 2^-20 more for the hardware's exponential) and for the
output (2^-11 of it, 2^-25 below fp16's normals)."""

import numpy as np
import pytest

from conftest import announce, fp16_exact
from oracle import windows
from test_gpu_int4 import Bytes
from test_gpu_kv_pages import mi, put

pytestmark = pytest.mark.gpu


def inputs(rng, seq_q, seq_k, heads, kv, hd):
    q, k, v = (rng.standard_normal((n, h, hd)) for n, h in ((seq_q, heads), (seq_k, kv), (seq_k, kv)))
    k[..., :2] *= 10
    return fp16_exact(q), fp16_exact(k), fp16_exact(v)


def check(got, q, k, v, window, sinks, what):
    want, bound, terms = windows.window_attention(q, k, v, window, sinks)
    limit = bound + (2.0**-11 + 2.0**-20) * terms + 2.0**-11 * np.abs(want) + 2.0**-25
    assert np.isfinite(got).all(), f"{what}: not finite"
    err = np.abs(got - want) / limit
    assert err.max() <= 1.0, f"{what}: {err.max():.3g} of the limit at {np.unravel_index(err.argmax(), err.shape)}"


def attend(q, k, v, window, sinks, split):
    d = mi().device
    seq_q, heads, hd = q.shape
    seq_k, kv, _ = k.shape
    y = Bytes(count=2 * q.size)
    y.numel = q.size
    parts = None
    if split:
        parts = d.empty_f32(max(1, d.attention_window_partials(seq_q, seq_k, heads, kv, hd, window,
                                                               sinks)))
    d.attention_window(put(q), put(k), put(v), y, seq_q, seq_k, heads, kv, hd, window, sinks,
                       partials=parts)
    return y.read().view(np.float16).reshape(q.shape).astype(np.float64)


@pytest.mark.parametrize("heads,kv,hd", [(14, 2, 64), (12, 2, 128), (32, 8, 64), (4, 4, 128),
                                         (5, 5, 64), (16, 1, 128), (40, 1, 64), (33, 3, 64)])
def test_head_layouts(heads, kv, hd):
    rng = np.random.default_rng(heads + hd)
    for seq_q, seq_k in ((1, 1), (1, 77), (3, 64), (70, 70), (65, 200)):
        q, k, v = inputs(rng, seq_q, seq_k, heads, kv, hd)
        announce("window layout", heads, kv, hd, seq_q, seq_k)
        check(attend(q, k, v, 33, 4, False), q, k, v, 33, 4, f"{heads}/{kv}x{hd} {seq_q}:{seq_k}")


@pytest.mark.parametrize("window,sinks", [
    (0, 0), (0, 7), (1, 0), (1, 1), (2, 40), (31, 0), (32, 4), (33, 33), (64, 64), (65, 4),
    (100, 1000), (199, 1), (200, 1), (201, 1), (100000, 3)])
@pytest.mark.parametrize("hd", [64, 128])
def test_windows_and_sinks(window, sinks, hd):
    rng = np.random.default_rng(window + sinks + hd)
    for seq_q, seq_k in ((200, 200), (37, 330), (1, 1000)):
        q, k, v = inputs(rng, seq_q, seq_k, 6, 2, hd)
        for split in (False, True):
            announce("window", window, sinks, hd, seq_q, seq_k, split)
            check(attend(q, k, v, window, sinks, split), q, k, v, window, sinks,
                  f"window {window} sinks {sinks} {seq_q}:{seq_k}")


@pytest.mark.parametrize("heads,kv,hd,seq_q,seq_k,window,sinks", [
    (32, 8, 64, 700, 900, 300, 4), (32, 8, 64, 601, 601, 0, 0), (12, 2, 128, 1500, 1500, 257, 70),
    (14, 2, 64, 1301, 1400, 64, 0), (28, 4, 128, 700, 703, 1, 0), (32, 8, 64, 300, 1500, 0, 0),
    (32, 8, 64, 301, 1501, 1200, 130), (32, 8, 64, 530, 2500, 0, 0), (14, 2, 64, 160, 2600, 2400, 33)])
def test_many_rows(heads, kv, hd, seq_q, seq_k, window, sinks):
    """Prompts of the kernel's large tiles: ragged last tiles, waves with no rows."""
    rng = np.random.default_rng(seq_q)
    q, k, v = inputs(rng, seq_q, seq_k, heads, kv, hd)
    announce("window many", heads, kv, hd, seq_q, seq_k)
    check(attend(q, k, v, window, sinks, True), q, k, v, window, sinks, f"{seq_q}:{seq_k}")


@pytest.mark.parametrize("hd", [64, 128])
def test_few_rows_over_a_long_range(hd):
    rng = np.random.default_rng(hd)
    q, k, v = inputs(rng, 3, 20001, 4, 2, hd)
    d = mi().device
    assert d.attention_window_partials(3, 20001, 4, 2, hd) > 0
    for window in (0, 9000):
        for split in (False, True):
            announce("window long", hd, window, split)
            check(attend(q, k, v, window, 5, split), q, k, v, window, 5, f"long {window} {split}")


@pytest.mark.parametrize("scale", [80.0, 0.0, -40.0])
def test_scores_far_apart_alike_and_rising(scale):
    """Scores of hundreds, of zero, and keys whose scores rise along the range, so that every
    step's maximum passes the last."""
    rng = np.random.default_rng(4)
    q, k, v = inputs(rng, 40, 400, 4, 2, 64)
    if scale > 0:
        q = fp16_exact(q * scale)
    elif scale == 0:
        q = np.zeros_like(q)
    else:
        q[..., 0], k[..., 0] = 8.0, (np.arange(400) / 16.0)[:, None]
        q, k = fp16_exact(q), fp16_exact(k)
    announce("window scores", scale)
    check(attend(q, k, v, 0, 0, False), q, k, v, 0, 0, f"scores {scale}")
    check(attend(q, k, v, 300, 4, True), q, k, v, 300, 4, f"scores {scale} windowed")


@pytest.mark.parametrize("heads,kv,hd,seq", [(14, 2, 64, 300), (12, 2, 128, 1400), (32, 8, 64, 600)])
def test_rows_of_one_projection(heads, kv, hd, seq):
    """q, k and v as views of fused rows, and keys alone in a wider buffer."""
    m = mi()
    d = m.device
    rng = np.random.default_rng(seq)
    q, k, v = inputs(rng, seq, seq, heads, kv, hd)
    width = (heads + 2 * kv) * hd
    fused = put(np.concatenate([x.reshape(seq, -1) for x in (q, k, v)], 1))
    out = d.empty(q.size)
    views = [d.view(fused, at, seq * width - at) for at in (0, heads * hd, (heads + kv) * hd)]
    announce("window fused", heads, kv, hd, seq)
    d.attention_window(*views, out, seq, seq, heads, kv, hd, 100, 4, q_stride=width, k_stride=width,
                       v_stride=width)
    check(out.to_numpy().reshape(q.shape).astype(np.float64), q, k, v, 100, 4, "fused")
    wide = np.full((seq, kv * hd + 24), np.nan)
    wide[:, 8:8 + kv * hd] = k.reshape(seq, -1)
    kw = put(wide)
    d.attention_window(put(q), d.view(kw, 8, kw.numel - 8), put(v), out, seq, seq, heads, kv, hd, 0,
                       0, k_stride=kv * hd + 24)
    check(out.to_numpy().reshape(q.shape).astype(np.float64), q, k, v, 0, 0, "wide keys")


@pytest.mark.parametrize("heads,kv,hd,seq_q", [(6, 2, 64, 150), (6, 2, 128, 150), (32, 8, 64, 640),
                                               (32, 8, 128, 640)])
def test_what_a_query_does_not_see_may_be_anything(heads, kv, hd, seq_q):
    """Keys and values of NaN and infinity: before the windows, between the sinks and the windows
    of the later queries, after the first queries. Queries that see none of them are exact; those
    that do are not finite in that channel."""
    rng = np.random.default_rng(hd + seq_q)
    seq_k, window, sinks = seq_q + 50, 40, 3
    q, k, v = inputs(rng, seq_q, seq_k, heads, kv, hd)
    bad = [5, 20, 49, 50 + 64, 50 + 100, seq_k - 1]
    kb, vb = k.copy(), v.copy()
    for i, j in enumerate(bad):
        vb[j, :, i] = (np.nan, np.inf, -np.inf)[i % 3]
        if i % 2:
            kb[j] = np.nan
    seen = np.stack([windows.visible(50 + i, seq_k, window, sinks) for i in range(seq_q)])
    clean = ~seen[:, bad].any(1)
    assert clean.any() and not clean.all()
    want, bound, terms = windows.window_attention(q, k, v, window, sinks)
    limit = bound + (2.0**-11 + 2.0**-20) * terms + 2.0**-11 * np.abs(want) + 2.0**-25
    for split in (False, True):
        announce("window not finite", heads, kv, hd, seq_q, split)
        got = attend(q, kb, vb, window, sinks, split)
        assert np.isfinite(got[clean]).all()
        assert (np.abs(got - want) <= limit)[clean].all()
        for i, j in enumerate(bad):
            assert not np.isfinite(got[seen[:, j]][:, :, i]).any()


@pytest.mark.parametrize("hd", [64, 128])
def test_replayed_graphs_and_repeats_to_the_bit(hd):
    m = mi()
    d = m.device
    rng = np.random.default_rng(12)
    seq_q, seq_k, heads, kv = 5, 3000, 8, 2
    q, k, v = inputs(rng, seq_q, seq_k, heads, kv, hd)
    dq, dk, dv = d.empty(q.size), put(k), put(v)
    stream = m.Stream()
    graphs = []
    for window in (0, 1000):
        parts = d.empty_f32(d.attention_window_partials(seq_q, seq_k, heads, kv, hd, window, 4))
        out = d.empty(q.size)
        graph = m.Graph(stream)
        with graph.capture():
            d.attention_window(dq, dk, dv, out, seq_q, seq_k, heads, kv, hd, window, 4,
                               partials=parts)
        graphs.append((graph, out, window, parts))
    for i in range(4):
        q = fp16_exact(rng.standard_normal(q.shape))
        m._h2d(dq.address, q.astype(np.float16))
        for graph, out, window, _ in graphs:
            announce("window replay", i, window)
            graph.launch()
            stream.synchronize()
            got = out.to_numpy().reshape(q.shape)
            check(got.astype(np.float64), q, k, v, window, 4, f"replay {window}")
            np.testing.assert_array_equal(got, attend(q, k, v, window, 4, True).astype(np.float32))
