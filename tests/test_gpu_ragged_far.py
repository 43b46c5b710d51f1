"""Rows whose offsets pass 32 bits: views of a wide buffer, tokens 2^23 elements
apart, through every operator that takes strides; the bits of the same rows
side by side, or the oracle's."""

import numpy as np
import pytest

from conftest import announce, fp16_exact
from test_gpu_append import Batch, P
from oracle import ragged
from test_gpu_int4 import Bytes
from test_gpu_kv_pages import mi, put

pytestmark = pytest.mark.gpu

STRIDE = (1 << 23) + 8
ROWS = 520  # the last ones past 2^32 elements


class Wide:
    """Rows of a buffer of ROWS x STRIDE elements, at an offset of it."""

    def __init__(self, buffer, first, rows):
        flat = np.ascontiguousarray(rows, np.float16).reshape(len(rows), -1)
        self.address = buffer.address + 2 * first
        self.numel = (len(rows) - 1) * STRIDE + flat.shape[1]
        self.nbytes = 2 * self.numel
        for i, row in enumerate(flat):
            mi()._h2d(self.address + 2 * i * STRIDE, row)


@pytest.fixture(scope="module")
def buffer():
    return mi().device.empty(ROWS * STRIDE)


def test_packed_attention(buffer):
    d = mi().device
    rng = np.random.default_rng(0)
    for heads, kv, hd in ((6, 2, 64), (2, 1, 128)):
        x = [fp16_exact(rng.standard_normal((ROWS, h, hd))) for h in (heads, kv, kv)]
        offsets = d.DeviceIndex([0, 30, 31, 400, ROWS])
        announce("far attention", heads, kv, hd)
        near = d.empty(x[0].size)
        d.attention_packed(*(put(t) for t in x), near, offsets, None, 4, ROWS, ROWS, heads, kv, hd)
        far = d.empty(x[0].size)
        views = [Wide(buffer, first, t) for first, t in zip((0, 4096, 8192), x)]
        d.attention_packed(*views, far, offsets, None, 4, ROWS, ROWS, heads, kv, hd, STRIDE, STRIDE, STRIDE)
        np.testing.assert_array_equal(near.to_numpy(), far.to_numpy())


def test_quantised_rows(buffer):
    d = mi().device
    rng = np.random.default_rng(1)
    x = fp16_exact(rng.standard_normal((ROWS, 2064)))
    codes, scales = Bytes(count=x.size), Bytes(count=4 * ROWS)
    announce("far rows")
    d.quantise_rows_int8(Wide(buffer, 0, x), codes, scales, ROWS, 2064, STRIDE)
    want, scale = ragged.quantise_rows(x)
    np.testing.assert_array_equal(codes.read().view(np.int8).reshape(x.shape), want)
    np.testing.assert_array_equal(scales.read().view(np.float32), scale)


def test_appended_rows(buffer):
    rng = np.random.default_rng(2)
    b = Batch(rng, [ROWS - 3, 0, 3], [5, 0, 64], 4, 2, 64, 17)
    rope = mi().device.RopeTable(64, 1e4)
    rope.cover(17 * P)
    announce("far append")
    views = [Wide(buffer, first, t) for first, t in zip((0, 4096, 8192), b.x)]
    b.run(rope, strides=(STRIDE,) * 3, views=views).check(ragged.frequencies(64, 1e4, None)[0], 1.0)


def test_sampled_logits(buffer):
    d = mi().device
    rng = np.random.default_rng(3)
    x = fp16_exact(3 * rng.standard_normal((ROWS, 1000)))
    u = rng.random(ROWS).astype(np.float32)
    tokens, scratch = Bytes(count=4 * ROWS), d.empty_f32(d.sample_scratch(ROWS, 1000))
    on_u = Bytes(u.view(np.uint8))
    announce("far logits")
    d.sample(Wide(buffer, 0, x), on_u, tokens, ROWS, 1000, stride=STRIDE, scratch=scratch)
    got = tokens.read().view(np.int32)
    for i in range(ROWS):
        token, border = ragged.sample(x[i], float(u[i]))
        assert border < 1e-9 or got[i] == token
