"""The choice of a token: every setting alone and together, ties, rows of one
logit and of a part's edges, infinities and NaN, uniforms at both ends, strides,
fp16 logits; the oracle's token, to the index.

A decision whose border lies within 1e-9 of the kept weights is not tested (the
histograms' weights are whole numbers of 2^-38 of the largest, of which a row of
2^18 may be off by 2^-21 at most, and by some 2^-30 in practice)."""

import numpy as np
import pytest

from conftest import announce
from oracle import ragged
from test_gpu_int4 import Bytes
from test_gpu_kv_pages import mi

pytestmark = pytest.mark.gpu


def on(x, dtype):
    return Bytes(np.frombuffer(np.ascontiguousarray(x, dtype).tobytes(), np.uint8))


def choose(logits, u, half=False, stride=0, **settings):
    d = mi().device
    rows, vocab = logits.shape
    wide = np.full((rows, stride or vocab), 1e4)
    wide[:, :vocab] = logits
    tokens, scratch = Bytes(count=4 * rows), d.empty_f32(d.sample_scratch(rows, vocab))
    logits_on = on(wide, np.float16 if half else np.float32)
    logits_on.numel = wide.size
    kinds = dict(temperature=np.float32, top_k=np.int32, top_p=np.float32, min_p=np.float32)
    given = {n: on(np.broadcast_to(v, rows), kinds[n]) for n, v in settings.items()}
    (d.sample if half else d.sample_f32)(logits_on, on(u, np.float32), tokens, rows, vocab,
                                         stride=stride, scratch=scratch, **given)
    return tokens.read().view(np.int32)


def check(logits, u, what, half=False, stride=0, **settings):
    logits = np.asarray(logits, np.float16 if half else np.float32)
    u = np.asarray(u, np.float32)
    announce("sample", what)
    got = choose(logits, u, half, stride, **settings)
    near = 0
    for i, row in enumerate(logits):
        mine = {n: float(np.broadcast_to(np.asarray(v, np.int32 if n == "top_k" else np.float32),
                                         len(logits))[i]) for n, v in settings.items()}
        if "top_k" in mine:
            mine["top_k"] = int(mine["top_k"])
        token, border = ragged.sample(row, float(u[i]), **mine)
        if border < 1e-9:
            near += 1
            continue
        assert got[i] == token, f"{what} row {i} {mine} u {u[i]}: {got[i]}, not {token}"
    # (Half of 50,000 equal weights, say, lies on a border by its numbers.)
    assert near <= max(1, len(logits) // 8)


def peaked(rng, rows, vocab):
    x = 2.0 * rng.standard_normal((rows, vocab))
    for r in x:
        r[rng.integers(0, vocab, 40)] += rng.exponential(4.0, 40)
    return x


@pytest.mark.parametrize("vocab", [1, 2, 63, 1000, 4095, 4096, 4097, 8192, 32000, 128256, 151936, 200003])
@pytest.mark.parametrize("half", [False, True])
def test_vocabularies(vocab, half):
    rng = np.random.default_rng(vocab)
    rows = 5
    x = peaked(rng, rows, vocab)
    u = rng.random(rows)
    stride = vocab + 5 if vocab < 5000 else 0
    check(x, u, f"{vocab} plain", half, stride)
    check(x, u, f"{vocab} all", half, stride, temperature=rng.uniform(0.3, 2, rows),
          top_k=rng.integers(1, 300, rows), top_p=rng.uniform(0.1, 1, rows),
          min_p=rng.uniform(0, 0.3, rows))


@pytest.mark.parametrize("settings", [
    dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=np.nan), dict(temperature=0.05),
    dict(temperature=1e-6), dict(temperature=30.0), dict(temperature=np.inf), dict(top_k=1), dict(top_k=2),
    dict(top_k=50), dict(top_k=5000), dict(top_k=10**9), dict(top_k=-3), dict(top_k=0), dict(top_p=0.0),
    dict(top_p=-1.0), dict(top_p=0.1), dict(top_p=0.9), dict(top_p=0.9999), dict(top_p=1.0),
    dict(top_p=2.0), dict(top_p=np.nan), dict(min_p=1.0), dict(min_p=7.0), dict(min_p=0.5),
    dict(min_p=0.05), dict(min_p=1e-8), dict(min_p=-1.0), dict(min_p=np.nan),
    dict(top_k=40, top_p=0.8), dict(top_k=3, top_p=0.99), dict(top_p=0.95, min_p=0.1),
    dict(temperature=5.0, top_k=3000, top_p=0.97, min_p=1e-3), dict(temperature=40.0, top_p=0.5),
    dict(temperature=40.0, top_k=60000), dict(temperature=40.0, min_p=0.9)])
def test_settings(settings):
    rng = np.random.default_rng(5)
    check(peaked(rng, 12, 30011), rng.random(12), settings, **settings)


@pytest.mark.parametrize("half", [False, True])
def test_ties(half):
    """Few different logits: borders inside runs of thousands of equal ones."""
    rng = np.random.default_rng(6)
    rows, vocab = 10, 50000
    x = rng.integers(0, 4, (rows, vocab)).astype(np.float64) / 2
    u = rng.random(rows)
    check(x, u, "ties k", half, top_k=rng.integers(1, vocab, rows))
    check(x, u, "ties p", half, top_p=rng.uniform(0, 1, rows))
    check(x, u, "ties both", half, top_k=rng.integers(1, vocab, rows), top_p=rng.uniform(0, 1, rows))
    check(x, u, "ties m", half, min_p=np.exp(-rng.integers(0, 4, rows) / 2) * 0.999)
    flat = np.zeros((4, vocab))
    check(flat, [0.0, 0.3, 0.7, 0.9999], "flat", half)
    check(flat, [0.0, 0.3, 0.7, 0.9999], "flat k", half, top_k=[1, 7, 20000, 49999])
    check(flat, [0.0, 0.3, 0.7, 0.9999], "flat p", half, top_p=[1e-9, 0.31, 0.5, 0.77])
    check(np.where(np.arange(vocab) % 2 == 0, 0.0, -0.0)[None], [0.6], "zeros of both signs", half, top_k=[777])


def test_many_close_logits():
    """More than a list of logits in a border's bucket, all different."""
    rng = np.random.default_rng(7)
    x = rng.uniform(0, 0.1, (6, 120000)).astype(np.float32)
    u = rng.random(6)
    check(x, u, "close k", top_k=rng.integers(1, 120000, 6))
    check(x, u, "close p", top_p=rng.uniform(0, 1, 6))
    check(x, u, "close m", min_p=rng.uniform(0.9, 1, 6))
    check(x, u, "close all", top_k=[100000] * 6, top_p=[0.7] * 6, min_p=[0.92] * 6)


def test_uniforms_at_the_ends():
    rng = np.random.default_rng(8)
    x = peaked(rng, 8, 9000)
    u = [0.0, -1.0, np.nan, 1.0, 5.0, np.nextafter(1, 0, dtype=np.float32), 1e-30, 0.5]
    want_u = [0.0, 0.0, 0.0, 1.0, 1.0, u[5], 1e-30, 0.5]
    got = choose(x.astype(np.float32), np.asarray(u, np.float32), top_k=20)
    for i in range(8):
        kept = np.sort(np.argsort(-x[i].astype(np.float32), kind="stable")[:20])
        if want_u[i] == 0.0:
            assert got[i] == kept[0]
        elif want_u[i] >= 1.0:
            assert got[i] == kept[-1]
        else:
            assert got[i] == ragged.sample(x[i].astype(np.float32), float(np.float32(want_u[i])), top_k=20)[0]


def test_infinities_and_nan():
    rng = np.random.default_rng(9)
    vocab = 9001
    x = peaked(rng, 9, vocab)
    x[0, :] = -np.inf                      # nothing to choose
    x[1, :] = np.nan
    x[2, :] = -np.inf
    x[2, 8000] = -5                        # one
    x[3, ::2] = np.nan
    x[4, rng.integers(0, vocab, 8000)] = -np.inf
    x[5, [17, 4099, 9000]] = np.inf        # share the weight
    x[6, :4096] = -np.inf                  # a whole part
    x[7, 4096:] = np.nan
    x[8, :] = -1e30
    u = rng.random(9)
    for s in ({}, dict(top_k=5), dict(top_p=0.6), dict(min_p=0.3), dict(temperature=0.0),
              dict(temperature=0.7, top_k=100, top_p=0.9, min_p=0.01)):
        check(x, u, f"not finite {s}", **s)


def test_extreme_scales():
    rng = np.random.default_rng(10)
    for size in (1e-30, 1e-6, 1e4, 1e12, 3e37):
        x = rng.standard_normal((6, 5000)) * size
        for s in ({}, dict(top_k=9, top_p=0.7), dict(min_p=0.2), dict(temperature=1e-3),
                  dict(temperature=float(np.float32(size)), top_p=0.9, min_p=0.05)):
            check(x, rng.random(6), f"size {size} {s}", **s)


def test_shares_follow_the_weights():
    """A row chosen from 4,000 evenly spaced uniforms: each token as often as it weighs."""
    rng = np.random.default_rng(11)
    row = peaked(rng, 1, 300).astype(np.float32)
    n = 4000
    got = choose(np.repeat(row, n, 0), (np.arange(n) + 0.5) / n, top_p=0.9)
    w = np.exp(row[0].astype(np.float64) - row.max())
    order = np.argsort(-w)
    keep = order[:np.searchsorted(np.cumsum(w[order]), 0.9 * w.sum()) + 1]
    want = np.zeros(300)
    want[keep] = w[keep] / w[keep].sum() * n
    # An interval of length L holds L evenly spaced points, one more or less.
    assert (np.abs(np.bincount(got, minlength=300) - want) <= 1 + 1e-6).all()


def test_a_captured_choice_follows_its_logits():
    m = mi()
    d = m.device
    rng = np.random.default_rng(12)
    rows, vocab = 3, 20000
    x, u, tokens = d.empty_f32(rows * vocab), d.empty_f32(rows), Bytes(count=4 * rows)
    scratch = d.empty_f32(d.sample_scratch(rows, vocab))
    t = on([0.7, 0.0, 1.3], np.float32)
    k = on([40, 0, 1000], np.int32)
    stream = m.Stream()
    graph = m.Graph(stream)
    with graph.capture():
        d.sample_f32(x, u, tokens, rows, vocab, t, k, scratch=scratch)
    for i in range(5):
        h, hu = peaked(rng, rows, vocab).astype(np.float32), rng.random(rows).astype(np.float32)
        m._h2d(x.address, h)
        m._h2d(u.address, hu)
        announce("captured sample", i)
        graph.launch()
        stream.synchronize()
        want = [ragged.sample(h[j], float(hu[j]), tt, kk)[0] for j, (tt, kk) in
                enumerate(((float(np.float32(0.7)), 40), (0.0, 0), (float(np.float32(1.3)), 1000)))]
        np.testing.assert_array_equal(tokens.read().view(np.int32), want)
