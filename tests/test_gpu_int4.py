"""4-bit weights on the device: the quantiser to the bit, projections against
float64 at the sizes where the kernel's tiles, splits and phases end.

Tolerance: the fp32 sums' bound (oracle.int4.linear_bound) and, for fp16
outputs, half a step of fp16 (2^-11 of the value, 2^-25 below its normals)."""

import numpy as np
import pytest

from conftest import announce, fp16_exact
from oracle import int4
from test_gpu_kv_pages import mi, put

pytestmark = pytest.mark.gpu


class Bytes:
    """Device bytes with a sentinel past the end."""

    def __init__(self, host=None, count=0):
        m = mi()
        host = np.full(count, 0xA5, np.uint8) if host is None else np.asarray(host, np.uint8)
        self.count = self.nbytes = host.size
        self._storage = m._Storage(host.size + 64)
        m._h2d(self._storage.ptr, np.concatenate([host.reshape(-1), np.full(64, 0xA5, np.uint8)]))

    @property
    def address(self):
        return self._storage.ptr

    def read(self):
        raw = np.empty(self.count + 64, np.uint8)
        mi()._d2h(raw, self.address)
        assert (raw[self.count:] == 0xA5).all(), "written past the end"
        return raw[:self.count]


def halves(x):
    return np.frombuffer(np.ascontiguousarray(x, np.float16).tobytes(), np.uint8)


def weight(rng, out, n_in):
    w = rng.standard_normal((out, n_in)) * n_in**-0.5
    w[:, rng.random(n_in) < 0.02] *= 8  # outlier inputs
    return fp16_exact(w)


class Int4:
    """A weight's codes, scales and zeros on the device, from the oracle."""

    def __init__(self, w, group):
        self.group = group
        self.codes, self.scales, self.zeros = int4.quantise(w, group)
        self.on = (Bytes(int4.packed(self.codes)), Bytes(halves(self.scales)),
                   Bytes(halves(self.zeros)))
        self.w64 = int4.weight64(self.codes, self.scales, self.zeros, group)

    def bound(self, x):
        return int4.linear_bound(x, self.codes, self.scales, self.zeros, self.group)


def check_half(got, want, bound):
    limit = bound + 2.0**-11 * np.abs(want) + 2.0**-25
    assert (np.abs(got - want) <= limit).all(), np.max(np.abs(got - want) / limit)


@pytest.mark.parametrize("out,n_in,group", [
    (1, 32, 32), (3, 64, 64), (5, 128, 128), (7, 96, 32), (1, 192, 64), (33, 1536, 128),
    (257, 896, 32), (130, 896, 64), (1000, 4864, 128), (2, 8960, 128)])
def test_quantise_is_the_oracle_s(out, n_in, group):
    d = mi().device
    rng = np.random.default_rng(out + n_in + group)
    w = weight(rng, out, n_in)
    w[0, :group] = w[0, 0]            # a constant group
    w[out - 1, -group:] *= 2.0**-14   # subnormal steps
    w[out // 2, :2] = (65504.0, -65504.0) if group == 64 else w[out // 2, :2]
    w = fp16_exact(w)
    want = int4.quantise(w, group)
    groups = out * (n_in // group)
    codes, scales, zeros = Bytes(count=out * n_in // 2), Bytes(count=2 * groups), Bytes(count=2 * groups)
    announce("quantise", out, n_in, group)
    d.quantise_int4(put(w), codes, scales, zeros, group, n_in, out)
    np.testing.assert_array_equal(codes.read().reshape(out, -1), int4.packed(want[0]))
    np.testing.assert_array_equal(scales.read().view(np.float16).reshape(want[1].shape), want[1])
    np.testing.assert_array_equal(zeros.read().view(np.float16).reshape(want[2].shape), want[2])


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 15, 16, 17, 32, 33, 64, 65, 130])
@pytest.mark.parametrize("out,n_in,group", [
    (1, 32, 32), (17, 96, 32), (128, 896, 32), (40, 64, 64), (65, 192, 64), (130, 896, 64),
    (16, 128, 128), (50, 640, 128), (300, 1536, 128)])
def test_linear_against_float64(rows, out, n_in, group):
    d = mi().device
    rng = np.random.default_rng(rows + out + n_in)
    w = Int4(weight(rng, out, n_in), group)
    x = fp16_exact(rng.standard_normal((rows, n_in)))
    b = fp16_exact(rng.standard_normal(out))
    want, bound = x.astype(np.float64) @ w.w64.T, w.bound(x)
    dx, db = put(x), put(b)
    for bias in (None, db):
        announce("linear int4", rows, out, n_in, group, "bias" if bias is not None else "")
        y = Bytes(count=2 * rows * out)
        y.numel = rows * out
        d.linear_int4(dx, *w.on, group, bias, y, rows, n_in, out)
        got = y.read().view(np.float16).reshape(rows, out).astype(np.float64)
        full = want + (b if bias is not None else 0.0)
        check_half(got, full, bound + (2.0**-24 * np.abs(full) if bias is not None else 0.0))
    start = rng.standard_normal((rows, out)).astype(np.float32)
    acc = d.upload_f32(start)
    announce("accumulate", rows, out, n_in, group)
    d.linear_int4_accumulate(dx, *w.on, group, acc, rows, n_in, out)
    got = acc.to_numpy().reshape(rows, out)
    assert (np.abs(got - (start + want)) <= bound + 2.0**-23 * (np.abs(start) + np.abs(want))).all()


@pytest.mark.parametrize("rows,out,n_in,group", [
    (1, 1536, 8960, 128), (27, 1536, 8960, 128), (64, 72, 24608, 32), (1, 33, 24608, 32),
    (1, 40001, 2048, 64), (3, 151936, 896, 32), (16, 8192, 2048, 64), (2, 40001, 160, 32),
    (9, 50001, 160, 32), (30, 50001, 320, 64), (64, 60001, 384, 128), (300, 65000, 96, 32),
    (40, 16400, 2176, 128), (40, 1000, 8960, 64), (10, 20000, 4096, 64), (20, 20000, 4096, 64),
    (700, 8200, 256, 64)])
def test_linear_at_the_models_sizes(rows, out, n_in, group):
    d = mi().device
    rng = np.random.default_rng(rows + out)
    w = Int4(weight(rng, out, n_in), group)
    x = fp16_exact(rng.standard_normal((rows, n_in)))
    announce("linear int4 large", rows, out, n_in, group)
    y = d.empty(rows * out)
    d.linear_int4(put(x), *w.on, group, None, y, rows, n_in, out)
    first = y.to_numpy()
    check_half(first.reshape(rows, out), x.astype(np.float64) @ w.w64.T, w.bound(x))
    for _ in range(3):  # the sums' order does not depend on timing
        d.linear_int4(put(x), *w.on, group, None, y, rows, n_in, out)
        np.testing.assert_array_equal(y.to_numpy(), first)


def test_a_row_that_is_not_finite_stays_in_its_row():
    d = mi().device
    rng = np.random.default_rng(1)
    w = Int4(weight(rng, 48, 256), 64)
    x = fp16_exact(rng.standard_normal((5, 256)))
    clean = x.astype(np.float64) @ w.w64.T
    x[1, 70], x[3, 5] = np.nan, np.inf
    y = d.empty(5 * 48)
    announce("rows with nan and inf")
    d.linear_int4(put(x), *w.on, 64, None, y, 5, 256, 48)
    got = y.to_numpy().reshape(5, 48)
    assert np.isnan(got[1]).all() and not np.isfinite(got[3]).any()
    keep = [0, 2, 4]
    check_half(got[keep], clean[keep], w.bound(x[keep]))


@pytest.mark.parametrize("rows", [1, 4, 16])
def test_inputs_and_steps_below_fp16_s_normals(rows):
    """x of 2^-16 and steps of 2^-20: no product is taken for zero."""
    d = mi().device
    rng = np.random.default_rng(rows)
    w = Int4(fp16_exact(rng.standard_normal((20, 256)) * 2.0**-18), 64)
    x = fp16_exact(rng.standard_normal((rows, 256)) * 2.0**-16)
    acc = d.upload_f32(np.zeros(rows * 20, np.float32))
    announce("small values", rows)
    d.linear_int4_accumulate(put(x), *w.on, 64, acc, rows, 256, 20)
    want = x.astype(np.float64) @ w.w64.T
    assert np.abs(want).max() > 0
    assert (np.abs(acc.to_numpy().reshape(rows, 20) - want) <= w.bound(x)).all()


def test_views_and_a_replayed_graph():
    """A batch's rows in the middle of a buffer, captured and replayed on a stream with eager work
    between the replays."""
    m = mi()
    d = m.device
    rng = np.random.default_rng(2)
    w = Int4(weight(rng, 200, 1024), 128)
    buffer, y = d.empty(6 * 1024), d.empty(6 * 200)
    x = d.view(buffer, 1024, 3 * 1024)
    out = d.view(y, 200, 3 * 200)
    acc = d.upload_f32(np.zeros(600, np.float32))
    stream = m.Stream()
    graph = m.Graph(stream)
    launch = lambda: (d.linear_int4(x, *w.on, 128, None, out, 3, 1024, 200),  # noqa: E731
                      d.linear_int4_accumulate(x, *w.on, 128, acc, 3, 1024, 200))
    total, size = np.zeros((3, 200)), np.zeros((3, 200))
    with graph.capture():
        launch()
    for i in range(4):
        host = fp16_exact(rng.standard_normal((6, 1024)))
        m._h2d(buffer.address, host.astype(np.float16))
        announce("replay", i)
        graph.launch()
        stream.synchronize()
        want, bound = host[1:4].astype(np.float64) @ w.w64.T, w.bound(host[1:4])
        check_half(out.to_numpy().reshape(3, 200), want, bound)
        total, size = total + want, size + bound + 2.0**-23 * (np.abs(total) + 2 * np.abs(want))
        assert (np.abs(acc.to_numpy().reshape(3, 200) - total) <= size).all()
        m.synchronize()
