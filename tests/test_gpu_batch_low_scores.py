"""Masses of a batch whose every score is far below zero, past what 2^-x holds,
with pages that are not read among those that are: their mass is zero, not the
zero sum times an overflow."""

import numpy as np
import pytest

from conftest import announce
from test_gpu_batch import UNREAD, Batch, P
from test_gpu_kv_pages import mi

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv,hd", [(14, 2, 64), (12, 2, 128)])
@pytest.mark.parametrize("length", [70, 300, 3000])
@pytest.mark.parametrize("window,sinks", [(0, 0), (200, 33)])
def test_scores_far_below_zero(length, heads, kv, hd, window, sinks):
    m = mi()
    rng = np.random.default_rng(length + hd + window)
    batch = Batch(rng, [length, 33], heads, kv, hd,
                  lambda b, p: UNREAD if b == 0 and p % 4 == 1 else 0, window, sinks)
    for b, p in zip(*np.nonzero(batch.table)):
        page = np.empty((2, P, kv, hd), np.float16)
        m._d2h(page, int(batch.table[b, p]))
        page[0, ..., 0] = 20.0
        m._h2d(int(batch.table[b, p]), page)
        batch.k[b, p * P:(p + 1) * P, :, 0] = 20.0
    batch.q[..., 0] = -200.0  # scores of -500 and -350, give or take the other channels'
    announce("batch low scores", length, heads, kv, hd, window)
    got, mass = batch.run(True, True)
    assert np.isfinite(mass).all()
    batch.check(got, mass, "low scores")
