"""Every kernel form of the 4-bit projections at every group size, on numbers
whose sums are exact: x small integers, scales powers of two, zeros halves, so
that fp32 holds every partial sum (multiples of a half below 2^23 of them) in
whatever order, and the outputs are the exact sums, rounded once. A lost,
doubled or misplaced input shows in the bits. And random weights of long inputs
within the limit of the steps the sums are formed in (oracle.int4.linear_limit;
half a step of fp16 for the output, 2^-11 of the value, 2^-25 below its
normals)."""

import numpy as np
import pytest

from conftest import announce, fp16_exact
from oracle import int4
from test_gpu_int4 import Bytes, Int4, halves, weight
from test_gpu_kv_pages import mi, put

pytestmark = pytest.mark.gpu

# The form that each launches: dot products of one and two rows, by one and by four sets of
# outputs; tiles of rows, outputs and waves, s where the waves share x.
FORMS = [(1, 40, 1024), (1, 16400, 128), (2, 40, 2048), (2, 16400, 128),
         (3, 40, 2048),     # 16 x 16 by sixteen waves
         (50, 1500, 2048),  # 32 x 16 by sixteen
         (40, 2000, 384),   # 16 x 16 by eight
         (3, 20000, 3200),  # 16 x 64 by eight
         (5, 50001, 1280),  # 16 x 64 by four, s
         (20, 20000, 2048),  # 32 x 64 by eight
         (20, 50001, 640),  # 32 x 32 by eight, s
         (64, 16400, 1024),  # 64 x 32 by eight
         (64, 50001, 384),  # 64 x 32 by eight, s
         (128, 33000, 256)]  # 64 x 64 by eight, s


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows,out,n_in", FORMS)
def test_exact_sums(rows, out, n_in, group):
    d = mi().device
    if group < 128:
        n_in += group  # the last step of 128 inputs is not whole
    rng = np.random.default_rng(rows + out + n_in + group)
    codes = rng.integers(0, 16, (out, n_in), np.uint8)
    scales = np.float16(2.0) ** rng.integers(-1, 2, (out, n_in // group)).astype(np.float16)
    zeros = (rng.integers(-16, 17, scales.shape) / 2).astype(np.float16)
    x = rng.integers(-4, 5, (rows, n_in)).astype(np.float64)
    on = (Bytes(int4.packed(codes)), Bytes(halves(scales)), Bytes(halves(zeros)))
    w = (codes * np.repeat(scales.astype(np.float32), group, axis=1) +
         np.repeat(zeros.astype(np.float32), group, axis=1))
    want = x.astype(np.float32) @ w.T  # exact in fp32 too: every partial sum is held
    assert np.abs(want).max() < 60000
    bias = rng.integers(-50, 51, out).astype(np.float64)
    dx, y = put(x), Bytes(count=2 * rows * out)
    y.numel = rows * out
    announce("exact int4", rows, out, n_in, group)
    for b in (None, bias):
        d.linear_int4(dx, *on, group, None if b is None else put(b), y, rows, n_in, out)
        full = (want if b is None else want + b.astype(np.float32)).astype(np.float16)
        np.testing.assert_array_equal(y.read().view(np.float16).reshape(rows, out), full)
    start = rng.integers(-1000, 1001, (rows, out)).astype(np.float32)
    acc = d.upload_f32(start)
    announce("exact int4 added", rows, out, n_in, group)
    d.linear_int4_accumulate(dx, *on, group, acc, rows, n_in, out)
    np.testing.assert_array_equal(acc.to_numpy().reshape(rows, out), start + want)


@pytest.mark.parametrize("rows,out,n_in,group", [
    (1, 1536, 8960, 128), (2, 400, 8960, 128), (27, 1536, 8960, 128), (64, 300, 8960, 64),
    (1, 33, 24608, 32), (64, 72, 24608, 32), (50, 1500, 4096, 64), (3, 5000, 4864, 128)])
def test_long_inputs_within_the_limit_of_their_steps(rows, out, n_in, group):
    d = mi().device
    rng = np.random.default_rng(rows + out + n_in)
    w = Int4(weight(rng, out, n_in), group)
    x = fp16_exact(rng.standard_normal((rows, n_in)))
    want = x @ w.w64.T
    limit = int4.linear_limit(x, w.codes, w.scales, w.zeros, group)
    y = d.empty(rows * out)
    announce("long int4", rows, out, n_in, group)
    d.linear_int4(put(x), *w.on, group, None, y, rows, n_in, out)
    err = np.abs(y.to_numpy().reshape(rows, out) - want)
    assert (err <= limit + 2.0**-11 * np.abs(want) + 2.0**-25).all()
    acc = d.upload_f32(np.zeros(rows * out, np.float32))
    announce("long int4 added", rows, out, n_in, group)
    d.linear_int4_accumulate(put(x), *w.on, group, acc, rows, n_in, out)
    assert (np.abs(acc.to_numpy().reshape(rows, out) - want) <= limit + 2.0**-24 * np.abs(want)).all()
