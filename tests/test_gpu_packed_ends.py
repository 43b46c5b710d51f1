"""Packed attention whose last step has few keys left, rows far apart in a wide
buffer: the bits of the same rows side by side, and float64."""

import numpy as np
import pytest

from conftest import announce, fp16_exact
from test_gpu_int4 import Bytes
from test_gpu_kv_pages import mi, put
from test_gpu_packed import check, offsets

pytestmark = pytest.mark.gpu

FAR = (1 << 24) - 8  # elements between tokens, the most that is taken


@pytest.mark.parametrize("heads,kv,hd", [(6, 2, 64), (2, 1, 128)])
@pytest.mark.parametrize("counts", [[1], [2, 1], [17], [129], [100, 30, 1]])
def test_few_keys_left_far_apart(heads, kv, hd, counts):
    d = mi().device
    o = offsets(counts)
    rows = int(o[-1])
    rng = np.random.default_rng(rows + hd)
    x = [fp16_exact(rng.standard_normal((rows, h, hd))) for h in (heads, kv, kv)]
    # Keys and values share a buffer that ends with the last row's values.
    width = kv * hd
    buffer = d.empty((rows - 1) * FAR + 2 * width)
    views = [d.view(buffer, at, (rows - 1) * FAR + width) for at in (0, width)]
    for view, t in zip(views, x[1:]):
        for i, row in enumerate(np.ascontiguousarray(t, np.float16).reshape(rows, -1)):
            mi()._h2d(view.address + 2 * i * FAR, row)
    index = d.DeviceIndex(o)
    near, far = (Bytes(count=2 * x[0].size) for _ in range(2))
    near.numel = far.numel = x[0].size
    announce("few keys left", heads, kv, hd, counts)
    d.attention_packed(put(x[0]), put(x[1]), put(x[2]), near, index, None, len(counts), rows, rows, heads,
                       kv, hd)
    d.attention_packed(put(x[0]), *views, far, index, None, len(counts), rows, rows, heads, kv, hd, 0, FAR, FAR)
    got = [out.read().view(np.float16).reshape(x[0].shape) for out in (near, far)]
    np.testing.assert_array_equal(*got)
    check(got[0], *x, o, o, f"few keys left {counts}")


@pytest.mark.parametrize("heads,kv,hd", [(32, 8, 64), (12, 2, 128)])
def test_large_tiles_with_few_keys_left(heads, kv, hd):
    """Enough rows for the large tiles; the last step of the last sequence has one key."""
    d = mi().device
    far = 1 << 16
    o = offsets([1000, 129, 385])
    rows = int(o[-1])
    rng = np.random.default_rng(hd)
    x = [fp16_exact(rng.standard_normal((rows, h, hd))) for h in (heads, kv, kv)]
    width = kv * hd
    buffer = d.empty((rows - 1) * far + 2 * width)
    views = [d.view(buffer, at, (rows - 1) * far + width) for at in (0, width)]
    for view, t in zip(views, x[1:]):
        for i, row in enumerate(np.ascontiguousarray(t, np.float16).reshape(rows, -1)):
            mi()._h2d(view.address + 2 * i * far, row)
    index, out = d.DeviceIndex(o), Bytes(count=2 * x[0].size)
    out.numel = x[0].size
    announce("large tiles, few keys left", heads, kv, hd)
    d.attention_packed(put(x[0]), *views, out, index, None, 3, rows, rows, heads, kv, hd, 0, far, far)
    check(out.read().view(np.float16).reshape(x[0].shape), *x, o, o, "large tiles")
