"""Rows in codes of 8 bits and their products: every kernel form, ragged rows and
outputs, inputs that end inside a step, biases, residuals in place and apart,
rows of zeros and of values that are not finite.

Codes and scales are the oracle's to the bit. A sum is exact; its scaling rounds
three times in fp32 (the sum, two products), the bias or residual once (2^-24 of
the result), the fp16 output half a step (2^-11, 2^-25 below its normals)."""

import numpy as np
import pytest

from conftest import announce, fp16_exact
from oracle import ragged
from test_gpu_int4 import Bytes, halves
from test_gpu_kv_pages import mi, put

pytestmark = pytest.mark.gpu


def floats(x):
    return Bytes(np.frombuffer(np.ascontiguousarray(x, np.float32).tobytes(), np.uint8))


def quantised(x, stride=0):
    """Codes and scales by the device; x (rows, features)."""
    rows, features = x.shape
    wide = np.full((rows, stride or features), np.nan)
    wide[:, :features] = x
    codes, scales = Bytes(count=rows * features), Bytes(count=4 * rows)
    mi().device.quantise_rows_int8(put(wide), codes, scales, rows, features, stride)
    return codes.read().view(np.int8).reshape(x.shape), scales.read().view(np.float32)


@pytest.mark.parametrize("features", [16, 64, 496, 512, 528, 896, 1024, 1040, 1536, 2048, 2064, 4864,
                                      8192, 8208, 8960, 16384, 16400, 20000])
def test_quantised_rows(features):
    rng = np.random.default_rng(features)
    for rows, stride in ((1, 0), (7, features + 8)):
        x = rng.standard_normal((rows, features)) * np.exp(rng.uniform(-8, 5, (rows, 1)))
        x[:, rng.random(features) < 0.02] *= 8
        x = fp16_exact(x)
        announce("rows", rows, features, stride)
        codes, scales = quantised(x, stride)
        want, scale = ragged.quantise_rows(x)
        np.testing.assert_array_equal(scales, scale)
        np.testing.assert_array_equal(codes, want)


def test_quantised_edges():
    """Zeros, one value, subnormals, the largest, halves between codes, infinities and NaN."""
    ties = np.zeros((1, 256))
    ties[0, :254] = (np.arange(254) - 126.5) / 127 * 127
    ties[0, 255] = 127
    rows = [np.zeros(256), np.full(256, -3.0), np.full(256, 2.0**-24), np.full(256, 65504.0),
            np.arange(256) * 2.0**-24, ties[0], np.linspace(-1, 1, 256)]
    for bad in (np.inf, -np.inf, np.nan):
        r = np.ones(256)
        r[200] = bad
        rows.append(r)
    x = np.asarray(rows, np.float16).astype(np.float32)
    announce("edges")
    codes, scales = quantised(x)
    want, scale = ragged.quantise_rows(x)
    np.testing.assert_array_equal(codes, want)
    np.testing.assert_array_equal(scales, scale)
    assert np.isnan(scales[-3:]).all() and scales[0] == 0


def codes_of(rng, rows, n, whole=False):
    c = rng.integers(-128, 128, (rows, n)).astype(np.int8)
    return c, np.exp(rng.uniform(-6, 0, rows)).astype(np.float32)


def multiply(x, xs, w, ws, bias=None, residual=None, in_place=False):
    d = mi().device
    rows, n, out = len(x), x.shape[1], len(w)
    at = Bytes(x.view(np.uint8)), floats(xs), Bytes(w.view(np.uint8)), floats(ws)
    if residual is None:
        y = Bytes(count=2 * rows * out)
        y.numel = rows * out
        d.linear_int8(*at, put(bias) if bias is not None else None, y, rows, n, out)
        return y.read().view(np.float16).reshape(rows, out).astype(np.float64)
    r = floats(residual)
    y = r if in_place else Bytes(count=4 * rows * out)
    d.linear_int8_accumulate(*at, y, rows, n, out, residual=None if in_place else r)
    return y.read().view(np.float32).reshape(rows, out).astype(np.float64)


def check(rng, rows, n, out, what):
    (x, xs), (w, ws) = codes_of(rng, rows, n), codes_of(rng, out, n)
    xs *= np.float32(1e-2 / np.sqrt(n))
    y, off = ragged.linear_int8(x, xs, w, ws)
    bias = fp16_exact(rng.standard_normal(out))
    for b in (None, bias):
        want = y if b is None else y + b
        got = multiply(x, xs, w, ws, b)
        limit = off + 2.0**-24 * np.abs(want) * 1.001 + 2.0**-11 * (np.abs(want) + off) + 2.0**-25
        assert (np.abs(got - want) <= limit).all(), f"{what}: {(np.abs(got - want) / limit).max()}"
    residual = rng.standard_normal((rows, out)).astype(np.float32)
    want = y + residual
    for in_place in (True, False):
        got = multiply(x, xs, w, ws, residual=residual, in_place=in_place)
        limit = off + 2.0**-24 * (np.abs(want) + off) + 2.0**-149
        assert (np.abs(got - want) <= limit).all(), f"{what} residual: {(np.abs(got - want) / limit).max()}"


@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 32, 33, 48, 64, 65, 100, 128])
def test_few_rows(rows):
    rng = np.random.default_rng(rows)
    for n, out in ((16, 1), (48, 17), (128, 16), (144, 33), (896, 128), (1536, 100), (2048, 257),
                   (8960, 48)):
        announce("few", rows, n, out)
        check(rng, rows, n, out, f"{rows} x {n} -> {out}")


@pytest.mark.parametrize("rows,n,out", [
    (512, 64, 4096), (513, 16, 4097), (1000, 80, 1100), (1027, 1536, 1031), (2048, 128, 2048),
    (1777, 192, 2049), (4100, 208, 1100), (300, 112, 8200), (129, 1024, 16384), (4096, 64, 4096)])
def test_many_rows(rows, n, out):
    rng = np.random.default_rng(rows + n)
    announce("many", rows, n, out)
    check(rng, rows, n, out, f"{rows} x {n} -> {out}")


@pytest.mark.parametrize("rows,n,out", [
    (16, 128, 8256), (24, 2048, 8192), (33, 16, 8200), (64, 80, 4097), (256, 192, 1024), (70, 1536, 3000),
    (65, 208, 16321), (60, 128, 20000), (640, 144, 4096), (700, 64, 15000), (1030, 128, 16500)])
def test_tiles_between(rows, n, out):
    """Between the choices of tiles: shared inputs whose last group has none, 64 rows of many outputs."""
    rng = np.random.default_rng(rows + n)
    announce("between", rows, n, out)
    check(rng, rows, n, out, f"{rows} x {n} -> {out}")


def test_sums_of_the_largest_codes():
    """-128 x -128 over the most inputs stays in 32 bits."""
    rng = np.random.default_rng(0)
    n = (1 << 17) - 16
    for rows in (2, 70):
        x, w = np.full((rows, n), -128, np.int8), np.full((40, n), -128, np.int8)
        w[3] = 127
        one = np.ones
        announce("largest", rows)
        y = multiply(x, one(rows, np.float32), w, one(40, np.float32),
                     residual=np.zeros((rows, 40), np.float32))
        np.testing.assert_array_equal(y, (x.astype(np.float64) @ w.T.astype(np.float64)).astype(np.float32))


def test_a_row_that_is_not_finite_spoils_its_own_outputs():
    rng = np.random.default_rng(1)
    x = fp16_exact(rng.standard_normal((5, 256)))
    x[2, 7] = np.inf
    w = fp16_exact(rng.standard_normal((48, 256)))
    (xc, xs), (wc, ws) = quantised(x), quantised(w)
    announce("not finite")
    y = multiply(xc, xs, wc, ws)
    assert np.isnan(y[2]).all() and np.isfinite(np.delete(y, 2, 0)).all()


def test_rows_through_a_quantised_weight():
    """From fp16 rows and weight to outputs: the error of the codes, half a step of each."""
    rng = np.random.default_rng(2)
    x, w = fp16_exact(rng.standard_normal((300, 1536))), fp16_exact(rng.standard_normal((512, 1536)) / 39)
    (xc, xs), (wc, ws) = quantised(x), quantised(w)
    announce("rows through")
    got = multiply(xc, xs, wc, ws)
    want = x.astype(np.float64) @ w.T
    # A code is off by half at most: |x| sw / 2 + |w| sx / 2 + sx sw / 4 an input.
    size = (np.abs(x).sum(1)[:, None] * ws / 2 + np.abs(w).sum(1) * xs[:, None] / 2 +
            1536 * np.outer(xs, ws) / 4) * 1.001
    assert (np.abs(got - want) <= size + 2.0**-11 * (np.abs(want) + size)).all()
    assert np.abs(got - want).mean() < 0.05 * np.abs(want).mean()


def test_a_captured_projection_follows_its_rows():
    m = mi()
    d = m.device
    rng = np.random.default_rng(3)
    rows, n, out = 40, 512, 300
    w, ws = quantised(fp16_exact(rng.standard_normal((out, n))))
    x, codes, scales = d.empty(rows * n), Bytes(count=rows * n), Bytes(count=4 * rows)
    wt, wst, y = Bytes(w.view(np.uint8)), floats(ws), Bytes(count=2 * rows * out)
    y.numel = rows * out
    stream = m.Stream()
    graph = m.Graph(stream)
    with graph.capture():
        d.quantise_rows_int8(x, codes, scales, rows, n)
        d.linear_int8(codes, scales, wt, wst, None, y, rows, n, out)
    for i in range(4):
        h = fp16_exact(rng.standard_normal((rows, n)))
        m._h2d(x.address, h.astype(np.float16))
        announce("captured int8", i)
        graph.launch()
        stream.synchronize()
        xc, xs = ragged.quantise_rows(h)
        want, off = ragged.linear_int8(xc, xs, w, ws)
        got = y.read().view(np.float16).reshape(rows, out).astype(np.float64)
        assert (np.abs(got - want) <= off + 2.0**-11 * (np.abs(want) + off) + 2.0**-25).all()
