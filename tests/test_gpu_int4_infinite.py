"""Rows of infinities and NaN through 4-bit weights: an output is what the sum
of x times the weights is, an infinity of its sign where the infinite terms
agree, NaN where they do not, where one meets a weight of zero or where the row
holds NaN; other rows keep their values and limits."""

import numpy as np
import pytest

from conftest import announce, fp16_exact
from test_gpu_int4 import Int4, check_half, weight
from test_gpu_kv_pages import mi, put

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,out,n_in,group", [
    (1, 33, 256, 64), (1, 16400, 96, 32), (2, 40, 8960, 128), (2, 16400, 128, 64),
    (5, 48, 256, 64), (16, 200, 2048, 128), (40, 1000, 1024, 32), (70, 40, 96, 32),
    (20, 50001, 64, 64), (70, 50001, 64, 32)])
def test_infinities_keep_their_sign(rows, out, n_in, group):
    d = mi().device
    rng = np.random.default_rng(rows + out + n_in)
    host = weight(rng, out, n_in)
    host[out // 2, :group] = 0.0  # weights of zero: a constant group's
    w = Int4(host, group)
    x = fp16_exact(rng.standard_normal((rows, n_in)))
    what = []
    for r in range(0, rows, 2):
        kind = (r // 2) % 5
        what.append((r, kind))
        at = rng.choice(n_in, 3, replace=False)
        if kind == 0:
            x[r, at[0]] = np.inf
        elif kind == 1:
            x[r, at[0]] = -np.inf
        elif kind == 2:
            x[r, at] = (np.inf, -np.inf, np.inf)
        elif kind == 3:
            x[r, at[:2]] = (np.inf, np.nan)
        else:
            x[r, rng.integers(0, group)] = np.inf  # meets the zero weights
    if rows == 1:
        x[0, 7] = np.inf
    clean = np.isfinite(x).all(1)
    want = np.empty((rows, out))
    with np.errstate(invalid="ignore"):
        want[clean] = x[clean] @ w.w64.T
        for r in np.flatnonzero(~clean):
            bad = ~np.isfinite(x[r])
            want[r] = (x[r, bad] * w.w64[:, bad]).sum(1)  # the finite terms move none of these
    assert np.isinf(want[~clean]).any()
    bound = w.bound(np.where(np.isfinite(x), x, 0.0))
    bias = fp16_exact(rng.standard_normal(out))
    dx = put(x)
    y = d.empty(rows * out)
    announce("infinite rows", rows, out, n_in, group)
    d.linear_int4(dx, *w.on, group, put(bias), y, rows, n_in, out)
    got = y.to_numpy().reshape(rows, out).astype(np.float64)
    np.testing.assert_array_equal(got[~clean], want[~clean])
    full = want[clean] + bias
    check_half(got[clean], full, bound[clean] + 2.0**-24 * np.abs(full))
    start = rng.standard_normal((rows, out)).astype(np.float32)
    acc = d.upload_f32(start)
    announce("infinite rows added", rows, out, n_in, group)
    d.linear_int4_accumulate(dx, *w.on, group, acc, rows, n_in, out)
    got = acc.to_numpy().reshape(rows, out)
    np.testing.assert_array_equal(got[~clean], want[~clean].astype(np.float32))
    full = start[clean] + want[clean]
    limit = bound[clean] + 2.0**-23 * (np.abs(start[clean]) + np.abs(want[clean]))
    assert (np.abs(got[clean] - full) <= limit).all()
